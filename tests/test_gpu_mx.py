"""GPU 8-bit rows and 4-bit experts against their 64-bit definitions.

Bars. Codes, scales and layouts are equal. For the experts: g and u carry a relative
error d of their typical size, so an intermediate lands on the other side of a
border of its code (whose step is at least 2^-4 of it) in a share of at most
2 d / 2^-4 of the values, and is then off by a step, at most 2^-3: in the 2-norm that
moves the result by 2^-3 * sqrt(2^5 d). The scaled MFMA keeps products to 2^-13 of
the largest, d = 2^-13: 2^-7; exact products in fp32 sums of up to 2^11 terms,
d = 2^-20 (random signs): 2^-10.5. The rounding of the result adds half a step,
2^-8 in bf16, 2^-11 in f16. Where all values are small integers nothing rounds and
the results are equal.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import _mx_ref as ref
from _helpers import banner
from reframework_amd.layers import RMSNorm
from reframework_amd.moe import Mxfp4Experts, Mxfp8Rows, fused_experts_mxfp4, quantize_mxfp8

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
REL = {torch.bfloat16: 2.0 ** -7 + 2.0 ** -8, torch.float16: 2.0 ** -10.5 + 2.0 ** -11,
       torch.float32: 2.0 ** -10.5}


def _rows_equal(q: Mxfp8Rows, x64):
    c, s, v = ref.mxfp8(x64)
    assert q.codes.shape == c.shape and q.scales.shape == s.shape
    assert np.array_equal(q.scales.view(torch.uint8).cpu().numpy(), s)
    assert np.array_equal(ref.to64(q.codes), c, equal_nan=True)
    pad = q.padded_codes.view(torch.uint8)[:, q.size:]
    assert not bool(pad.any())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,H", [(1, 32), (3, 96), (37, 128), (5, 1248), (130, 4096)])
def test_quantize_rows(T, H, dt, dev):
    banner(f"quantize_mxfp8 {dt} T={T} H={H}")
    g = torch.Generator().manual_seed(T + H)
    x = torch.randn(T, H, generator=g)
    x *= torch.exp2(torch.randint(-9, 9, (T, H // 32), generator=g).float()).repeat_interleave(32, 1)
    x = x.to(dt)
    _rows_equal(quantize_mxfp8(x.to(dev)), ref.to64(x))


@pytest.mark.parametrize("dt", DTYPES)
def test_quantize_borders_zeros_and_non_finite(dt, dev):
    banner(f"quantize_mxfp8 borders {dt}")
    x = torch.zeros(12, 64)
    codes = torch.tensor(ref.E4M3[64:96].copy(), dtype=torch.float32)
    x[1, :32] = codes                                # every code itself
    x[2, :32] = codes * 1.0625                       # midpoints of the three-bit steps
    x[2, 31] = 448.0
    x[3, 0], x[3, 33] = 448.0, -449.0                # the largest code and just over it
    x[4, :32] = torch.linspace(-1, 1, 32)
    x[4, 3], x[4, 40], x[4, 41] = float("inf"), float("nan"), -float("inf")
    x[5, 7] = torch.finfo(dt).max
    x[6, 7] = torch.finfo(dt).tiny
    x[7, :] = torch.finfo(dt).tiny * 0.5             # subnormals
    x[8, ::2] = -0.0
    x[9, 0], x[9, 1:32] = 1.0, 2.0 ** -12            # far below the block's largest
    x = x.to(dt)
    _rows_equal(quantize_mxfp8(x.to(dev)), ref.to64(x))


def test_quantize_shapes(dev):
    banner("quantize_mxfp8 shapes")
    assert len(quantize_mxfp8(torch.empty((0, 64), device=dev))) == 0
    x = torch.randn(2, 3, 160, device=dev)
    q = quantize_mxfp8(x[:, :, 32:96])
    _rows_equal(q, ref.to64(x[:, :, 32:96].reshape(6, 64)))
    assert np.array_equal(ref.to64(q.dequantize()), ref.mxfp8(ref.to64(x[:, :, 32:96].reshape(6, 64)))[2])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,H", [(1, 32), (1, 4096), (7, 1248), (37, 2048), (300, 96), (3, 8192)])
@pytest.mark.parametrize("wdt,with_bias", [(torch.float32, False), ("same", True)])
def test_norm_leaves_its_rows_in_8_bits(T, H, dt, wdt, with_bias, dev):
    """normed and residual are those of forward_add_residual bit for bit, the rows
    those of quantize_mxfp8(normed)."""
    banner(f"norm mxfp8 {dt} T={T} H={H} {wdt} bias={with_bias}")
    g = torch.Generator().manual_seed(T + H)
    norm = RMSNorm(H, 1e-5, bias=with_bias)
    wt = dt if wdt == "same" else wdt
    norm.weight.data = (torch.rand(H, generator=g) + 0.5).to(wt)
    if with_bias:
        norm.bias.data = (torch.randn(H, generator=g) * 0.1).to(wt)
    norm = norm.to(dev)
    x = (torch.randn(T, H, generator=g) * 2).to(dt).to(dev)
    r = torch.randn(T, H, generator=g).to(dt).to(dev)
    normed, q, res = norm.forward_add_residual_mxfp8(x, r)
    n2, r2 = norm.forward_add_residual(x, r)
    assert torch.equal(normed, n2) and torch.equal(res, r2)
    _rows_equal(q, ref.to64(normed))
    n3, q3 = norm.forward_mxfp8(x)
    assert torch.equal(n3, norm(x))
    _rows_equal(q3, ref.to64(n3))


def _random_codes(E, N, K, rng, lo=118, hi=123):
    c = rng.integers(0, 256, (E, N, K // 2), dtype=np.uint8)
    s = rng.integers(lo, hi, (E, N, K // 32), dtype=np.uint8)
    return c, s


def _experts(w1, w2, dev):
    t = [torch.from_numpy(a).to(dev) for a in (*w1, *w2)]
    return Mxfp4Experts.from_codes(*t)


@pytest.mark.parametrize("E,H,I", [(1, 32, 32), (3, 160, 96), (2, 256, 128), (5, 1248, 416)])
def test_layout_round_trip(E, H, I, dev):
    banner(f"Mxfp4Experts layout E={E} H={H} I={I}")
    rng = np.random.default_rng(H + I)
    w1, w2 = _random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng)
    x = _experts(w1, w2, dev)
    for name, w in (("w1", w1), ("w2", w2)):
        c, s = x.codes(name)
        assert np.array_equal(c.cpu().numpy(), w[0]) and np.array_equal(s.cpu().numpy(), w[1])
        assert np.array_equal(ref.to64(x.dequantize(name)), ref.dequant4(*w))


@pytest.mark.parametrize("dt", DTYPES)
def test_quantize_weights(dt, dev):
    banner(f"Mxfp4Experts.quantize {dt}")
    g = torch.Generator().manual_seed(5)
    E, H, I = 2, 96, 64
    w1 = (torch.randn(E, 2 * I, H, generator=g) * 0.05).to(dt)
    w2 = (torch.randn(E, H, I, generator=g) * 3).to(dt)
    w1[0, 0, :32] = 0.0
    w1[0, 1, 5], w1[1, 2, 40] = float("nan"), float("inf")
    w1[0, 3, :16] = torch.tensor(np.concatenate([ref.FP4, (ref.FP4[:-1] + ref.FP4[1:]) / 2,
                                                 [5.0]])).to(dt)  # codes and their midpoints
    w1[0, 4, 0] = torch.finfo(dt).max
    for a, b in ((w1.to(dev), w2.to(dev)), ([m.to(dev) for m in w1], [m.to(dev) for m in w2])):
        x = Mxfp4Experts.quantize(a, b)
        for name, w in (("w1", w1), ("w2", w2)):
            c, s = x.codes(name)
            for e in range(E):
                rc, rs = ref.mxfp4(ref.to64(w[e]))
                assert np.array_equal(s[e].cpu().numpy(), rs)
                assert np.array_equal(c[e].cpu().numpy(), rc)


def _routing(T, K, E, rng):
    ids = np.stack([rng.permutation(E)[:K] for _ in range(T)]).astype(np.int64)
    w = rng.random((T, K)).astype(np.float32) + 0.1
    return w / w.sum(1, keepdims=True), ids


def _rel(got, want):
    return float(np.linalg.norm(ref.to64(got) - want) / np.linalg.norm(want))


SIZES = [  # T, H, E, K, I
    (1, 32, 1, 1, 32), (1, 256, 8, 2, 416), (3, 160, 4, 3, 96), (17, 256, 4, 2, 128),
    (40, 1248, 3, 1, 416), (64, 128, 2, 2, 32), (130, 384, 5, 3, 160), (300, 160, 2, 1, 288),
    (700, 256, 3, 2, 384), (9, 1024, 256, 8, 64), (1200, 512, 2, 2, 256),
]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,H,E,K,I", SIZES)
def test_experts(T, H, E, K, I, dt, dev):
    banner(f"fused_experts_mxfp4 {dt} T={T} H={H} E={E} K={K} I={I}")
    rng = np.random.default_rng(T * 31 + H + I)
    w1, w2 = _random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng)
    x = torch.from_numpy(rng.normal(size=(T, H))).to(dt)
    tw, ids = _routing(T, K, E, rng)
    ex = _experts(w1, w2, dev)
    want = ref.experts(ref.to64(x), ref.dequant4(*w1), ref.dequant4(*w2), tw, ids)
    got = fused_experts_mxfp4(x.to(dev), ex, torch.from_numpy(tw).to(dev),
                              torch.from_numpy(ids).to(dev))
    assert got.dtype == dt and _rel(got, want) <= REL[dt]
    # rows that are in 8 bits already, and int32 ids: the same bits
    q = quantize_mxfp8(x.to(dev))
    again = fused_experts_mxfp4(q, ex, torch.from_numpy(tw).to(dev),
                                torch.from_numpy(ids.astype(np.int32)).to(dev), out_dtype=dt)
    assert torch.equal(got, again)


@pytest.mark.parametrize("T,H,E,K,I,dt", [
    (1024, 256, 2, 1, 8192, torch.bfloat16),   # 256-row tiles, more items than CUs
    (620, 160, 8, 2, 4096, torch.bfloat16),    # 64-row tiles
    (620, 160, 8, 2, 4096, torch.float16),
    (1024, 256, 2, 1, 8192, torch.float16),    # 128-row tiles
    (700, 8192, 3, 2, 96, torch.bfloat16),     # down: one step of columns, many weight tiles
])
def test_several_items_per_workgroup(T, H, E, K, I, dt, dev):
    """The loads of an item start while the one before it runs, with as few as one
    step of columns each."""
    banner(f"fused_experts_mxfp4 many items {dt} T={T} H={H} E={E} K={K} I={I}")
    rng = np.random.default_rng(T)
    w1, w2 = _random_codes(E, 2 * I, H, rng, 116, 119), _random_codes(E, H, I, rng)
    x = torch.from_numpy(rng.normal(size=(T, H))).to(dt)
    tw, ids = _routing(T, K, E, rng)
    want = ref.experts(ref.to64(x), ref.dequant4(*w1), ref.dequant4(*w2), tw, ids)
    got = fused_experts_mxfp4(x.to(dev), _experts(w1, w2, dev), torch.from_numpy(tw).to(dev),
                              torch.from_numpy(ids).to(dev))
    assert _rel(got, want) <= REL[dt]


def test_more_items_than_a_launch_of_resident_workgroups_holds(dev):
    """32 items for each of the workgroups that run at once are not enough here: the
    launch has more. The same tokens in parts, whose launches do not, give the same
    bits (a row's sums do not depend on the others)."""
    banner("fused_experts_mxfp4 items past the workgroups' lists")
    T, H, E, I = 8192, 65536, 2, 32
    g = torch.Generator(device=dev).manual_seed(1)
    w1 = torch.randn(E, 2 * I, H, generator=g, device=dev).bfloat16() * 0.01
    w2 = torch.randn(E, H, I, generator=g, device=dev).bfloat16()
    ex = Mxfp4Experts.quantize(w1, w2)
    del w1, w2
    x = torch.randn(T, H, generator=g, device=dev).bfloat16()
    ids = torch.randint(0, E, (T, 1), generator=g, device=dev)
    tw = torch.rand(T, 1, generator=g, device=dev) + 0.5
    whole = fused_experts_mxfp4(x, ex, tw, ids)
    assert bool(torch.isfinite(whole).all()) and float(whole.float().abs().max()) > 0
    for t in range(0, T, 2048):
        part = slice(t, t + 2048)
        assert torch.equal(fused_experts_mxfp4(x[part], ex, tw[part], ids[part]), whole[part])


def test_tokens_past_2_gb_run_in_parts(dev):
    """8-bit tokens of more bytes than the kernels' offsets hold."""
    banner("fused_experts_mxfp4 past 2 GB of tokens")
    T, H, E, I = 40000, 65536, 2, 32
    g = torch.Generator(device=dev).manual_seed(2)
    ex = Mxfp4Experts.quantize(torch.randn(E, 2 * I, H, generator=g, device=dev) * 0.01,
                               torch.randn(E, H, I, generator=g, device=dev))
    codes = torch.randint(0, 120, (T, H), generator=g, device=dev, dtype=torch.uint8)
    q = Mxfp8Rows(codes.view(torch.float8_e4m3fn),
                  torch.randint(110, 120, (T, H // 32), generator=g, device=dev,
                                dtype=torch.uint8).view(torch.float8_e8m0fnu), H)
    ids = torch.randint(0, E, (T, 1), generator=g, device=dev)
    tw = torch.rand(T, 1, generator=g, device=dev) + 0.5
    whole = fused_experts_mxfp4(q, ex, tw, ids)
    for t in (0, 16384, 32766, 32767, 32768, 39000):  # 32767 tokens of 64 KB fit below 2 GB
        n = min(1000, T - t)
        part = Mxfp8Rows(q.padded_codes[t:t + n], q.padded_scales[t:t + n], H)
        got = fused_experts_mxfp4(part, ex, tw[t:t + n], ids[t:t + n])
        assert torch.equal(got, whole[t:t + n])


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_activations(activation, dt, dev):
    banner(f"fused_experts_mxfp4 {activation} {dt}")
    rng = np.random.default_rng(2)
    T, H, E, K, I = 50, 256, 3, 2, 128
    w1, w2 = _random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng)
    x = torch.from_numpy(rng.normal(size=(T, H))).to(dt)
    tw, ids = _routing(T, K, E, rng)
    want = ref.experts(ref.to64(x), ref.dequant4(*w1), ref.dequant4(*w2), tw, ids, activation)
    got = fused_experts_mxfp4(x.to(dev), _experts(w1, w2, dev), torch.from_numpy(tw).to(dev),
                              torch.from_numpy(ids).to(dev), activation=activation)
    assert _rel(got, want) <= REL[dt]


@pytest.mark.parametrize("T,H,E,K,I", SIZES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_experts_in_integers_are_equal(T, H, E, K, I, dt, dev):
    """x in {-1, 0, 1}, few non-zero weights: g is 64, 0 or -64 (silu: 64, 0 or
    -64 exp(-64), below 2e-26), u a small integer, so h is 64 times one but for
    values below 1e-25, whatever the order of sums; weights of 1 and 2. A result of at
    most 2^8 steps of 64 is exact in bf16 too. Every feature and every column takes
    part. A result adds 2 K values of h, so the small ones themselves move it by less
    than 1e-20; but a sum of 64 and -1e-26 is rounded, and the matrix cores may round it
    towards zero (measured: 128 - 2^-17), so each of the at most K (I / 8 + 4) additions
    may be off by 2^-23 of its sum, and no sum is over the 8 K values of 64 that a result
    can have. A value in a wrong place moves a result by 64 or more."""
    banner(f"fused_experts_mxfp4 integers {dt} T={T} H={H} E={E} K={K} I={I}")
    rng = np.random.default_rng(T + H * 3 + I)
    x = rng.integers(-1, 2, (T, H)).astype(np.float64)
    x[:, 0] = 1.0  # scale of the first block, and a column that is always on
    w1 = np.zeros((E, 2 * I, H))
    w2 = np.zeros((E, H, I))
    for e in range(E):
        # gate row i looks at one column, times 64; up row i at two others
        w1[e, np.arange(I), (np.arange(I) * 7 + e) % H] = 64.0
        w1[e, I + np.arange(I), (np.arange(I) * 5 + 3 * e + 1) % H] += 1.0
        w1[e, I + np.arange(I), (np.arange(I) * 11 + e + 2) % H] += 1.0
        # down row j at two features
        w2[e, np.arange(H), (np.arange(H) * 3 + e) % I] += 1.0
        w2[e, np.arange(H), (np.arange(H) * 13 + 2 * e + 1) % I] -= 1.0
    q1, q2 = ([np.stack(z) for z in zip(*(ref.mxfp4(m) for m in w))] for w in (w1, w2))
    assert np.array_equal(ref.dequant4(*q1), w1) and np.array_equal(ref.dequant4(*q2), w2)
    ids = np.stack([rng.permutation(E)[:K] for _ in range(T)]).astype(np.int64)
    tw = rng.integers(1, 3, (T, K)).astype(np.float32)
    want = ref.experts(x, w1, w2, tw, ids)
    ex = _experts(q1, q2, dev)
    got = fused_experts_mxfp4(torch.from_numpy(x).to(dt).to(dev), ex,
                              torch.from_numpy(tw).to(dev), torch.from_numpy(ids).to(dev))
    whole = np.round(want / 64) * 64
    assert np.abs(want).max() <= 2.0 ** 14 and np.abs(want - whole).max() < 1e-20
    assert np.abs(ref.to64(got) - whole).max() <= K * (I / 8 + 4) * 2.0 ** -23 * 512 * K + 1e-20


def test_dropped_slots_and_repeated_experts(dev):
    """Ids outside the experts and weights of 0 add nothing, whatever row they name; an
    expert that a token names twice counts twice; a token with no slot left gets 0."""
    banner("fused_experts_mxfp4 dropped slots")
    rng = np.random.default_rng(9)
    T, H, E, K, I = 40, 256, 4, 3, 96
    w1, w2 = _random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng)
    x = torch.from_numpy(rng.normal(size=(T, H))).float()
    tw = rng.random((T, K)).astype(np.float32)
    ids = rng.integers(-2, E + 2, (T, K))
    ids[0], ids[1], ids[2] = -1, E, [2, 2, 2]
    tw[3], tw[4, 1] = 0.0, 0.0
    ids[5:30] = 1  # most rows on one expert
    want = ref.experts(ref.to64(x), ref.dequant4(*w1), ref.dequant4(*w2), tw, ids)
    ex = _experts(w1, w2, dev)
    for dt in DTYPES:
        got = fused_experts_mxfp4(x.to(dt).to(dev), ex, torch.from_numpy(tw).to(dev),
                                  torch.from_numpy(ids).to(dev))
        assert bool((got[[0, 1, 3]] == 0).all())
        if dt != torch.float32:  # x was rounded: its own oracle
            r = ref.experts(ref.to64(x.to(dt)), ref.dequant4(*w1), ref.dequant4(*w2), tw, ids)
        else:
            r = want
        assert _rel(got, r) <= REL[dt]
    all_out = fused_experts_mxfp4(x.to(dev), ex, torch.from_numpy(tw).to(dev),
                                  torch.full((T, K), -1, device=dev))
    assert bool((all_out == 0).all())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T", [5, 90, 700])
def test_non_finite_tokens_and_weights_stay_with_their_rows(T, dt, dev):
    banner(f"fused_experts_mxfp4 non-finite {dt} T={T}")
    rng = np.random.default_rng(4)
    H, E, K, I = 256, 3, 1, 160
    w1, w2 = _random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng)
    x = torch.from_numpy(rng.normal(size=(T, H))).to(dt)
    tw, ids = _routing(T, K, E, rng)
    clean = fused_experts_mxfp4(x.to(dev), _experts(w1, w2, dev), torch.from_numpy(tw).to(dev),
                                torch.from_numpy(ids).to(dev))
    x2 = x.clone()
    x2[1, 7], x2[3, 200] = float("nan"), float("inf")
    got = fused_experts_mxfp4(x2.to(dev), _experts(w1, w2, dev), torch.from_numpy(tw).to(dev),
                              torch.from_numpy(ids).to(dev))
    bad = torch.zeros(T, dtype=torch.bool, device=dev)
    bad[1] = bad[3] = True
    assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[~bad], clean[~bad])
    # a NaN block in one expert's down weights: that feature of its tokens alone
    w2[1][2, 9, 1] = 255
    got = fused_experts_mxfp4(x.to(dev), _experts(w1, w2, dev), torch.from_numpy(tw).to(dev),
                              torch.from_numpy(ids).to(dev))
    hit = torch.zeros((T, H), dtype=torch.bool, device=dev)
    hit[torch.from_numpy(ids[:, 0] == 2).to(dev), 9] = True
    assert bool(torch.isnan(got[hit]).all()) and torch.equal(got[~hit], clean[~hit])


def test_accumulate_empty_and_layouts(dev):
    banner("fused_experts_mxfp4 accumulate / layouts")
    rng = np.random.default_rng(6)
    T, H, E, K, I = 21, 160, 4, 2, 64
    w1, w2 = _random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng)
    ex = _experts(w1, w2, dev)
    xs = torch.from_numpy(rng.normal(size=(T, 2 * H))).float().to(dev)
    tw, ids = _routing(T, K, E, rng)
    tw, ids = torch.from_numpy(tw).to(dev), torch.from_numpy(ids).to(dev)
    x = xs[:, 1:H + 1]  # rows that are neither contiguous nor aligned
    base = fused_experts_mxfp4(x.contiguous(), ex, tw, ids)
    assert torch.equal(fused_experts_mxfp4(x, ex, tw, ids), base)
    flat = torch.empty(T * H + 1, device=dev)[1:].reshape(T, H)
    flat.copy_(x)  # contiguous, off by 4 bytes
    assert torch.equal(fused_experts_mxfp4(flat, ex, tw, ids), base)
    wide_w, wide_i = tw.repeat(1, 2), ids.repeat(1, 2)
    assert torch.equal(fused_experts_mxfp4(x, ex, wide_w[:, :K], wide_i[:, :K]), base)
    acc = torch.ones((T, H), device=dev)
    out = fused_experts_mxfp4(x, ex, tw, ids, out=acc, accumulate_f32=True)
    assert out is acc and torch.equal(acc, 1 + base)
    assert fused_experts_mxfp4(x[:0], ex, tw[:0], ids[:0]).shape == (0, H)
    assert torch.equal(fused_experts_mxfp4(x[:1], ex, tw[:1], ids[:1]), base[:1])


@pytest.mark.parametrize("T", [1, 40, 600])
def test_captured_and_replayed_beside_eager_calls(T, dev):
    """Two graphs with workspaces of their own, replayed on two streams with new inputs
    and eager calls in between."""
    banner(f"fused_experts_mxfp4 graphs T={T}")
    rng = np.random.default_rng(7)
    H, E, K, I = 256, 4, 2, 128
    ex = _experts(_random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng), dev)
    tw, ids = _routing(T, K, E, rng)
    tw, ids = torch.from_numpy(tw).to(dev), torch.from_numpy(ids).to(dev)
    norm = RMSNorm(H, 1e-5).to(dev)

    def step(x, r):
        normed, q, res = norm.forward_add_residual_mxfp8(x, r)
        return fused_experts_mxfp4(q, ex, tw, ids), res

    xs = [torch.randn(T, H, device=dev).bfloat16() for _ in range(4)]
    rs = [torch.randn(T, H, device=dev).bfloat16() for _ in range(4)]
    want = [step(x, r) for x, r in zip(xs, rs)]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gx, gr = torch.zeros_like(xs[0]), torch.zeros_like(rs[0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(gx, gr)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(gx, gr)
        graphs.append((g, gx, gr, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(4):
        for (g, gx, gr, _), s, j in zip(graphs, streams, (k, 3 - k)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                gx.copy_(xs[j])
                gr.copy_(rs[j])
                g.replay()
        eager = step(xs[k], rs[k])
        torch.cuda.synchronize()
        assert torch.equal(eager[0], want[k][0])
        for (g, _, _, out), j in zip(graphs, (k, 3 - k)):
            assert torch.equal(out[0], want[j][0]) and torch.equal(out[1], want[j][1])


def test_two_streams_at_once(dev):
    banner("fused_experts_mxfp4 two streams")
    rng = np.random.default_rng(8)
    H, E, K, I, T = 512, 8, 2, 256, 64
    ex = _experts(_random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng), dev)
    tw, ids = _routing(T, K, E, rng)
    tw, ids = torch.from_numpy(tw).to(dev), torch.from_numpy(ids).to(dev)
    xs = [torch.randn(T, H, device=dev).bfloat16() for _ in range(2)]
    want = [fused_experts_mxfp4(x, ex, tw, ids) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(fused_experts_mxfp4(x, ex, tw, ids))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("T", [3, 150, 900])
def test_results_in_place_of_the_tokens(T, dev):
    banner(f"fused_experts_mxfp4 in place T={T}")
    rng = np.random.default_rng(T)
    H, E, K, I = 288, 4, 2, 160
    ex = _experts(_random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng), dev)
    tw, ids = _routing(T, K, E, rng)
    tw, ids = torch.from_numpy(tw).to(dev), torch.from_numpy(ids).to(dev)
    x = torch.from_numpy(rng.normal(size=(T, H))).bfloat16().to(dev)
    want = fused_experts_mxfp4(x, ex, tw, ids)
    assert fused_experts_mxfp4(x, ex, tw, ids, out=x) is x and torch.equal(x, want)


@pytest.mark.parametrize("T,E", [(150, 2), (700, 3)])
def test_slot_results_of_every_magnitude(T, E, dev):
    """bf16 calls keep the slots' results in 16 bits with a scale per 64 columns: rows
    from 2^-100 to 2^110, columns of one block 2^20 apart, an infinity beside them.
    Each row and each column keeps the bar of the whole."""
    banner(f"fused_experts_mxfp4 magnitudes T={T}")
    rng = np.random.default_rng(T)
    H, K, I = 288, 2, 384
    (c1, s1), (c2, s2) = _random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng)
    s2 = (s2.astype(np.int64) + rng.integers(-10, 11, size=(1, H, 1))).astype(np.uint8)
    shift = rng.integers(-50, 54, size=(T, 1))
    x = torch.from_numpy(rng.normal(size=(T, H)) * np.exp2(shift)).bfloat16()
    tw, ids = _routing(T, K, E, rng)
    ex = _experts((c1, s1), (c2, s2), dev)
    want = ref.experts(ref.to64(x), ref.dequant4(c1, s1), ref.dequant4(c2, s2), tw, ids)
    args = ex, torch.from_numpy(tw).to(dev), torch.from_numpy(ids).to(dev)
    got = ref.to64(fused_experts_mxfp4(x.to(dev), *args))
    size = np.linalg.norm(want, axis=1, keepdims=True)
    assert size.max() / size.min() > 2.0 ** 150
    err, want = (got - want) / size, want / size
    for axis in (0, 1):
        assert np.all(np.linalg.norm(err, axis=axis) <= REL[torch.bfloat16] * np.linalg.norm(want, axis=axis))
    # a row of w2 with a NaN scale spoils its column and no other of its block
    s2[:, 70, 0] = 255
    bad = ref.to64(fused_experts_mxfp4(x.to(dev), _experts((c1, s1), (c2, s2), dev), *args[1:]))
    assert np.all(np.isnan(bad[:, 70]))
    keep = np.arange(H) != 70
    assert np.array_equal(bad[:, keep], got[:, keep])


@pytest.mark.parametrize("T,K", [(400, 10), (600, 10), (600, 8), (300, 3)])
def test_many_slots_per_token(T, K, dev):
    banner(f"fused_experts_mxfp4 T={T} K={K}")
    rng = np.random.default_rng(T + K)
    H, E, I = 96, 12, 64
    w1, w2 = _random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng)
    x = torch.from_numpy(rng.normal(size=(T, H))).bfloat16()
    tw, ids = _routing(T, K, E, rng)
    tw[::7, 1] = 0.0  # dropped
    want = ref.experts(ref.to64(x), ref.dequant4(*w1), ref.dequant4(*w2), tw, ids)
    ex = _experts(w1, w2, dev)
    args = x.to(dev), ex, torch.from_numpy(tw).to(dev), torch.from_numpy(ids).to(dev)
    got = fused_experts_mxfp4(*args)
    assert _rel(got, want) <= REL[torch.bfloat16]
    acc = torch.ones((T, H), device=dev)
    fused_experts_mxfp4(*args, out=acc, accumulate_f32=True)
    assert _rel(acc, want + 1) <= REL[torch.bfloat16]
    assert torch.equal(fused_experts_mxfp4(*args), got)


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("T,H,E,K,I", [(1, 4096, 8, 2, 2048), (5, 160, 4, 3, 96), (16, 2048, 64, 6, 1408),
                                       (40, 1248, 12, 3, 416)])
def test_few_tokens_per_expert_are_exact_in_bf16_too(T, H, E, K, I, activation, dev):
    """Calls that stream the weights multiply exactly whatever the result's type is: a
    bf16 result is the fp32 one rounded once."""
    banner(f"fused_experts_mxfp4 exact in bf16 T={T} H={H} E={E} K={K} I={I} {activation}")
    rng = np.random.default_rng(T + H)
    w1, w2 = _random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng)
    x = quantize_mxfp8(torch.from_numpy(rng.normal(size=(T, H))).bfloat16().to(dev))
    tw, ids = _routing(T, K, E, rng)
    args = x, _experts(w1, w2, dev), torch.from_numpy(tw).to(dev), torch.from_numpy(ids).to(dev)
    full = fused_experts_mxfp4(*args, activation=activation, out_dtype=torch.float32)
    got = fused_experts_mxfp4(*args, activation=activation, out_dtype=torch.bfloat16)
    assert torch.equal(got, full.bfloat16())


@pytest.mark.parametrize("T,E,K", [(700, 3, 2), (250, 5, 3)])
def test_bf16_slots_added_to_fp32_stay_in_fp32(T, E, K, dev):
    """All slots in one call or one after the other: the same products, each of which is
    weighed and added in 32 bits, so per slot two roundings of 2^-24 of it and of the sum
    so far; slots kept to 11 bits would be off by some 2^-13."""
    banner(f"fused_experts_mxfp4 fp32 slots T={T} E={E} K={K}")
    rng = np.random.default_rng(T)
    H, I = 288, 384
    ex = _experts(_random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng), dev)
    x = torch.from_numpy(rng.normal(size=(T, H))).bfloat16().to(dev)
    tw, ids = (torch.from_numpy(t).to(dev) for t in _routing(T, K, E, rng))
    whole = torch.zeros((T, H), device=dev)
    fused_experts_mxfp4(x, ex, tw, ids, out=whole, accumulate_f32=True)
    apart, size = torch.zeros((T, H), device=dev), torch.zeros((T, H), device=dev)
    for k in range(K):
        one = torch.zeros((T, H), device=dev)
        args = x, ex, tw[:, k:k + 1], ids[:, k:k + 1]
        fused_experts_mxfp4(*args, out=one, accumulate_f32=True)
        fused_experts_mxfp4(*args, out=apart, accumulate_f32=True)
        size += one.abs()
    assert bool(((whole - apart).abs() <= 2 * K * 2.0 ** -24 * 2 * size).all())


@pytest.mark.parametrize("T,dt", [(1, torch.bfloat16), (1, torch.float32), (30, torch.float32),
                                  (300, torch.float32), (300, torch.bfloat16)])
def test_scales_at_the_ends_of_their_range(T, dt, dev):
    """One product, of a token's block with scale byte b and a weights' block with the byte
    that brings it back, through up, beside a gate of 384. Exact products are those of the
    operands as bf16 numbers: bytes 3 to 246 of tokens and 1 to 252 of weights hold every
    code; beyond, the largest codes are infinite (the result is NaN) and the smallest
    multiples of 2^-133. The scaled MFMA (a bf16 result of many tokens) takes all as they
    are. A byte of 255 is NaN."""
    banner(f"fused_experts_mxfp4 scale bytes T={T} {dt}")
    scaled = dt == torch.bfloat16 and T > 12
    H, I = 128, 32
    cases = [(bx, min(max(254 - bx, 0), 254), c8, 2)
             for bx in (*range(0, 6), 100, 127, *range(244, 256)) for c8 in (1, 3, 9, 15, 56, 119, 126)]
    cases += [(min(max(254 - bw, 0), 246), bw, 56, c4)
              for bw in (0, 1, 2, 127, *range(250, 256)) for c4 in range(1, 8)]
    bx, bw, c8, c4 = (np.array(v) for v in zip(*cases))
    n = len(cases)  # one expert per case: its T rows are the same token
    x, xs = np.zeros((n, T, H), np.uint8), np.full((n, T, H // 32), 127, np.uint8)
    x[:, :, 0], x[:, :, 32], xs[:, :, 1] = 56, c8[:, None], bx[:, None]
    w1, s1 = np.zeros((n, 2 * I, H // 2), np.uint8), np.full((n, 2 * I, H // 32), 127, np.uint8)
    w1[:, :I, 0], s1[:, :I, 0] = 7, 127 + 6
    w1[:, I:, 16], s1[:, I:, 1] = c4[:, None], bw[:, None]
    w2, s2 = np.zeros((n, H, I // 2), np.uint8), np.full((n, H, 1), 127, np.uint8)
    w2[:, :, 0] = 2
    u8, u4 = ref.E4M3[c8] * ref.pow2(bx), ref.FP4[c4] * ref.pow2(bw)
    if not scaled:
        u8, u4 = (torch.from_numpy(v).float().bfloat16().double().numpy() for v in (u8, u4))
    with np.errstate(invalid="ignore"):
        h = np.repeat((384.0 * u8 * u4)[:, None], 32, 1)
    want = np.where(np.isfinite(h), ref.mxfp8(h)[2], np.nan)[:, 0]
    got = []
    for k in range(0, n, 200):  # experts of one call
        part = slice(k, k + 200)
        m = len(bx[part])
        q = Mxfp8Rows(torch.from_numpy(x[part].reshape(m * T, H)).to(dev).view(torch.float8_e4m3fn),
                      torch.from_numpy(xs[part].reshape(m * T, -1)).to(dev).view(torch.float8_e8m0fnu), H)
        ids = torch.arange(m, device=dev).repeat_interleave(T)[:, None]
        got.append(fused_experts_mxfp4(q, _experts((w1[part], s1[part]), (w2[part], s2[part]), dev),
                                       torch.ones((m * T, 1), device=dev), ids, out_dtype=dt))
    got = ref.to64(torch.cat(got)).reshape(n, T, H)
    assert np.isnan(want).any() and np.isfinite(want).sum() > 100
    want = torch.from_numpy(want).to(dt).double().numpy()
    assert np.array_equal(got, np.broadcast_to(want[:, None, None], got.shape), equal_nan=True)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,K,hot", [(60, 64, 4, 1), (60, 64, 4, 4), (130, 256, 6, 1), (40, 256, 8, 0)])
def test_popular_experts_of_a_call_that_streams(T, E, K, hot, dt, dev):
    """Few rows per expert on average, but the first `hot` experts are every token's: many
    16-row tiles of one expert beside experts of one row or none."""
    banner(f"fused_experts_mxfp4 popular experts T={T} E={E} K={K} hot={hot} {dt}")
    rng = np.random.default_rng(T + E)
    H, I = 288, 160
    w1, w2 = _random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng)
    x = torch.from_numpy(rng.normal(size=(T, H))).to(dt)
    tw, ids = _routing(T, K, E, rng)
    for t in range(T):
        ids[t] = [*range(hot), *(e for e in ids[t] if e >= hot), *range(hot, K)][:K]
    assert T * K // min(T * K, E) <= 12 and all(len(set(r)) == K for r in ids.tolist())
    want = ref.experts(ref.to64(x), ref.dequant4(*w1), ref.dequant4(*w2), tw, ids)
    got = fused_experts_mxfp4(x.to(dev), _experts(w1, w2, dev), torch.from_numpy(tw).to(dev),
                              torch.from_numpy(ids).to(dev))
    assert _rel(got, want) <= REL[dt]


@pytest.mark.parametrize("T", [0, 1, 90, 700])
def test_result_of_another_type_than_the_tokens(T, dev):
    banner(f"fused_experts_mxfp4 out_dtype T={T}")
    rng = np.random.default_rng(T)
    H, E, K, I = 288, 3, 2, 160
    ex = _experts(_random_codes(E, 2 * I, H, rng), _random_codes(E, H, I, rng), dev)
    x = torch.from_numpy(rng.normal(size=(T, H))).bfloat16().to(dev)
    tw = torch.rand((T, K), device=dev) + 0.1
    ids = torch.randint(0, E, (T, K), device=dev)
    for dt in (torch.float32, torch.float16):
        got = fused_experts_mxfp4(x, ex, tw, ids, out_dtype=dt)
        assert got.dtype == dt and got.shape == (T, H)
        assert torch.equal(got, fused_experts_mxfp4(quantize_mxfp8(x), ex, tw, ids, out_dtype=dt))
    acc = torch.zeros((T, H), device=dev)
    fused_experts_mxfp4(x, ex, tw, ids, out=acc, accumulate_f32=True, out_dtype=torch.float32)
    assert torch.equal(acc, fused_experts_mxfp4(x, ex, tw, ids, out_dtype=torch.float32))
    with pytest.raises((TypeError, ValueError)):
        fused_experts_mxfp4(x, ex, tw, ids, out_dtype=torch.float64)
