"""64-bit definitions of the 8-bit rows, the 4-bit experts and the routing by groups
(not collected: no test_ prefix). Nothing here uses the package."""

from __future__ import annotations

import math

import numpy as np
import torch

FP4 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# e4m3 values of codes 0..126
E4M3 = np.array([(m / 8 * 2.0 ** -6) if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                 for e in range(16) for m in range(8)][:127])


def pow2(b):
    return np.where(b == 255, np.nan, np.ldexp(1.0, np.where(b == 255, 0, b.astype(np.int64)) - 127))


def block_scale(amax, largest):
    """Smallest scale byte with amax <= largest * 2^(b - 127), by search over all."""
    steps = largest * np.ldexp(1.0, np.arange(0, 255) - 127)
    return np.searchsorted(steps, amax, side="left").astype(np.int64) * (amax > 0)


def nearest(v, table):
    """Index of the table value nearest to |v|, ties to the even index."""
    m = np.abs(v)
    hi = np.clip(np.searchsorted(table, m, side="left"), 1, len(table) - 1)
    lo = hi - 1
    a, b = m - table[lo], table[hi] - m
    return np.where((a < b) | ((a == b) & (lo % 2 == 0)), lo, hi)


def mxfp8(x):
    """(code values, scale bytes, dequantised) of fp64 rows [T, H]; NaN codes for
    values that are not finite."""
    T, H = x.shape
    b = x.reshape(T, H // 32, 32)
    fin = np.isfinite(b)
    safe = np.where(fin, b, 0.0)
    s = block_scale(np.abs(safe).max(-1), 448.0)
    v = safe / np.ldexp(1.0, s - 127)[..., None]
    c = np.sign(v) * E4M3[nearest(v, E4M3)]
    c = np.where(fin, c, np.nan)
    return c.reshape(T, H), s, (c * np.ldexp(1.0, s - 127)[..., None]).reshape(T, H)


def mxfp4(w):
    """(codes [rows, cols / 2], scale bytes) of fp64 weights [rows, cols]."""
    rows, cols = w.shape
    b = w.reshape(rows, cols // 32, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    s = np.where(bad, 255, block_scale(np.abs(b).max(-1), 6.0))
    v = b / np.ldexp(1.0, np.where(bad, 127, s) - 127)[..., None]
    c = (nearest(v, FP4) | np.where(v < 0, 8, 0)).reshape(rows, cols // 2, 2).astype(np.uint8)
    return c[..., 0] | (c[..., 1] << 4), s.astype(np.uint8)


def dequant4(codes, scales):
    """fp64 of codes [..., cols / 2] and scale bytes [..., cols / 32]."""
    q = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = FP4[q & 7] * np.where(q >> 3, -1.0, 1.0)
    return v * np.repeat(pow2(scales), 32, axis=-1)


def act(name, g):
    if name == "silu":
        return g / (1.0 + np.exp(np.minimum(-g, 700.0)))
    if name == "gelu":
        return 0.5 * g * (1.0 + np.array([math.erf(t) for t in (g / math.sqrt(2.0)).ravel()])
                          .reshape(g.shape))
    return 0.5 * g * (1.0 + np.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)))


def experts(x, w1, w2, topk_w, ids, activation="silu"):
    """fp64 [T, H]: x is quantised here; w1 [E, 2I, H] and w2 [E, H, I] are values."""
    xq = mxfp8(x)[2]
    out = np.zeros((x.shape[0], w2.shape[1]))
    for e in range(w1.shape[0]):
        tok, slot = np.nonzero((ids == e) & (topk_w != 0))
        if not tok.size:
            continue
        g, u = np.split(xq[tok] @ w1[e].T, 2, axis=1)
        h = mxfp8(act(activation, g) * u)[2]
        np.add.at(out, tok, (h @ w2[e].T) * topk_w[tok, slot].astype(np.float64)[:, None])
    return out


def grouped_topk(logits, K, renormalize=True, scoring="softmax", bias=None, num_groups=1,
                 topk_groups=1, group_score="max", scale=1.0):
    """(weights fp64, ids) with every choice in 64 bits, NaN last, ties to the lower."""
    x = logits.astype(np.float64)
    T, E = x.shape
    with np.errstate(over="ignore", invalid="ignore"):
        if scoring == "sigmoid":
            s = 1.0 / (1.0 + np.exp(-x))
        else:
            e = np.exp(x - np.fmax.reduce(x, axis=1, keepdims=True))
            s = e / e.sum(1, keepdims=True)
    if bias is None and (group_score == "max" or topk_groups == num_groups):
        c = x.copy()
    else:
        c = s + (0.0 if bias is None else bias.astype(np.float64))
    S = E // num_groups
    # stable ascending sorts of -c: largest first, the lower index first, NaN last
    best = -np.sort(-c.reshape(T, num_groups, S), axis=2)
    group = best[:, :, 0]
    if group_score == "top2" and S > 1:
        two = best[:, :, 0] + best[:, :, 1]
        group = np.where(np.isnan(two), group, two)
    kept = np.zeros((T, num_groups), bool)
    np.put_along_axis(kept, np.argsort(-group, axis=1, kind="stable")[:, :topk_groups], True, 1)
    order = np.argsort(-c, axis=1, kind="stable")
    on = np.take_along_axis(np.repeat(kept, S, axis=1), order, 1)
    first = on & (np.cumsum(on, axis=1) <= K)
    ids = order[first].reshape(T, K)
    w = np.take_along_axis(s, ids, 1)
    if renormalize:
        w = w / (w.sum(1, keepdims=True) + 1e-20)
    return w * scale, ids


def to64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()
