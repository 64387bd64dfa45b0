"""The 8-bit format with a scale per block of 128, in numpy at 64 bits, and the products of
its values (not collected: no test_ prefix)."""

from __future__ import annotations

import numpy as np
import torch

BLOCK = 128
LEAST = 448.0 * 2.0 ** -126


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def blocks(n: int) -> int:
    return -(-n // BLOCK)


def rne_e4m3(q: np.ndarray) -> np.ndarray:
    """Values of the codes nearest to |q| <= 448, ties to even."""
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(q), 2.0 ** -6))) - 3)
    return np.round(q / step) * step


def _split(v: np.ndarray, axis: int) -> np.ndarray:
    pad = [(0, 0)] * v.ndim
    pad[axis] = (0, -v.shape[axis] % BLOCK)
    v = np.pad(v, pad)
    return v.reshape(*v.shape[:axis], -1, BLOCK, *v.shape[axis + 1:])


def quantize_rows(v: np.ndarray):
    """(quotients, values of the codes, scales) of [M, K]."""
    b = _split(v, 1)
    fin = np.where(np.isfinite(b), np.abs(b), 0.0)
    most = np.maximum(fin.max(-1, keepdims=True), LEAST)
    q = np.where(np.isfinite(b), b, np.nan) * 448.0 / most
    M, K = v.shape
    return (q.reshape(M, -1)[:, :K], rne_e4m3(q).reshape(M, -1)[:, :K],
            (most[..., 0] / 448.0).astype(np.float32))


def through(v: np.ndarray) -> np.ndarray:
    """[M, K] as the format holds it, scales in fp32."""
    _, c, s = quantize_rows(v)
    return c * np.repeat(s.astype(np.float64), BLOCK, 1)[:, :v.shape[1]]


def weight(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """[N, K] of the codes' values and block scales."""
    s = np.repeat(np.repeat(scales.astype(np.float64), BLOCK, 0), BLOCK, 1)
    return codes * s[:codes.shape[0], :codes.shape[1]]


def matmul(x: np.ndarray, w: np.ndarray):
    """(x @ w.T, what the products may be off by): of each step of 128 columns 2^-10 of its
    largest product (the matrix core was measured at 2^-11), and of the fp32 scaling and adding of
    the steps 2^-22 each."""
    out = x @ w.T
    off = np.zeros_like(out)
    for k in range(0, x.shape[1], BLOCK):
        a, b = np.abs(x[:, k:k + BLOCK]), np.abs(w[:, k:k + BLOCK])
        most = np.zeros_like(out)
        for j in range(a.shape[1]):
            np.maximum(most, np.outer(a[:, j], b[:, j]), out=most)
        off += 2.0 ** -10 * most + 2.0 ** -22 * (a @ b.T) * (1 + k / BLOCK)
    return out, off


def act(name: str, g: np.ndarray) -> np.ndarray:
    from scipy.special import erf

    if name == "silu":
        return g / (1.0 + np.exp(-g))
    if name == "gelu":
        return 0.5 * g * (1.0 + erf(g / np.sqrt(2.0)))
    return 0.5 * g * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (g + 0.044715 * g ** 3)))


def experts(x, w1, w2, tw, ids, name):
    """[T, H]: tokens and activations through 8 bits, all else in 64."""
    xq, out = through(x), np.zeros_like(x)
    E, I = w1.shape[0], w1.shape[1] // 2
    for e in range(E):
        t, k = np.nonzero(ids == e)
        if t.size:
            gu = xq[t] @ w1[e].T
            y = through(act(name, gu[:, :I]) * gu[:, I:]) @ w2[e].T
            np.add.at(out, t, y * tw[t, k, None].astype(np.float64))
    return out
