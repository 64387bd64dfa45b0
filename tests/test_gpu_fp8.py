"""8-bit rows and weights with a scale per block of 128 on the GPU, against 64 bits.

Codes of 16-bit values are exact: their quotients times 448 have few bits, and a tie is a
tie in fp32 too. Of fp32 values the quotient is rounded to 24 bits first, so a code may be the
other neighbour where the quotient lies within 2^-23 of a border. Products are exact where
every sum of a step has few bits (small whole numbers and scales of powers of two), so those
tests ask for equality; others go by _fp8_ref.matmul and half a step of the result's type.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import _fp8_ref as ref
from _helpers import DT, banner
from reframework_amd.fp8 import Fp8Rows, blocks, padded
from reframework_amd.layers import LayerNorm
from reframework_amd.moe import (Fp8Experts, Fp8Weight, combine_tokens, fused_experts,
                                 fused_experts_fp8, matmul_fp8, permute_tokens, quantize_fp8)

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def rounded(dt, v):
    """What rounding v to dt may be off by: half a step, of float16 below 2^-14 of 2^-24."""
    f = torch.finfo(dt)
    return np.maximum(f.eps / 2 * np.abs(v), f.tiny * f.eps / 2)


# ------------------------------------------------------------------ the format
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 129), (5, 1000), (17, 1248), (300, 72), (2, 4096), (700, 520)])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_rows(M, K, dt, dev):
    banner(f"fp8 quantize M={M} K={K} {dt}")
    g = torch.Generator(device=dev).manual_seed(K)
    x = torch.randn(M, K, generator=g, device=dev)
    x *= torch.exp(2 * torch.randn(M, 1, generator=g, device=dev))
    x = x.to(DT[dt])
    q = quantize_fp8(x)
    assert q.padded_codes.shape == (M, padded(K)) and not q.padded_codes[:, K:].float().any()
    quot, want, scales = ref.quantize_rows(ref.f64(x))
    got = ref.f64(q.codes.float())
    if dt == "f32":
        near = ref.rne_e4m3(quot * (1 + 2.0 ** -22)) != ref.rne_e4m3(quot * (1 - 2.0 ** -22))
        assert (got == want)[~near].all()
        assert (np.abs(got - quot) <= 2.0 ** -4 * np.abs(quot) * (1 + 2.0 ** -20) + 2.0 ** -10).all()
    else:
        assert np.array_equal(got, want)
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    assert np.array_equal(q.dequantize().cpu().numpy(), got.astype(np.float32) * np.repeat(scales, 128, 1)[:, :K])
    assert torch.equal(quantize_fp8(x.reshape(M, 1, K)).padded_codes.view(torch.uint8), q.padded_codes.view(torch.uint8))


@pytest.mark.parametrize("dt", ["bf16", "f32", "f16"])
def test_rows_at_the_ends(dt, dev):
    banner(f"fp8 quantize ends {dt}")
    dt = DT[dt]
    big = torch.finfo(dt).max
    x = torch.zeros(9, 256, dtype=dt, device=dev)
    x[1, :4] = torch.tensor([big, -big, big / 2, 1.0])
    x[2, 5], x[2, 6] = float("inf"), 3.0
    x[3, 7], x[3, 8] = float("nan"), -2.0
    x[4, 9] = torch.finfo(dt).tiny
    x[5, 3] = 2.0 ** -24 if dt == torch.float16 else 2.0 ** -133
    x[6] = float("-inf")
    x[7, 128:] = 7.0
    x[8, 0], x[8, 1] = big, 0.75 * big
    q = quantize_fp8(x)
    quot, want, scales = ref.quantize_rows(ref.f64(x))
    got = ref.f64(q.codes.float())
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert np.array_equal(got[ok], want[ok])
    assert np.array_equal(q.scales.cpu().numpy(), scales)


@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (130, 260), (1000, 72), (384, 1025)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_weights(N, K, dt, dev):
    banner(f"fp8 weight N={N} K={K} {dt}")
    g = torch.Generator(device=dev).manual_seed(N)
    w = (torch.randn(2, N, K, generator=g, device=dev) * 0.02).to(DT[dt])
    fw = Fp8Weight.quantize(w, transposed=True)
    got = ref.f64(fw.dequantize())
    for e in range(2):
        for i in range(0, N, 128):
            for j in range(0, K, 128):
                b = ref.f64(w[e, i:i + 128, j:j + 128])
                most = np.abs(b).max()
                s = np.float32(most / 448.0)
                want = ref.rne_e4m3(b * 448.0 / most) * np.float64(s)
                d = np.abs(got[e, i:i + 128, j:j + 128] - want)
                # the product of code and scale is rounded to fp32; an fp32 quotient may tip a tie
                tie = 0 if dt == "bf16" else 2.0 ** -3
                assert (d <= (2.0 ** -23 + tie) * np.abs(want) + 1e-30).all() and (d > 2.0 ** -23 * np.abs(want)).mean() < 1e-3
    again = Fp8Weight.from_codes(*fw.codes(), transposed=True)
    assert torch.equal(again.codes()[0].view(torch.uint8), fw.codes()[0].view(torch.uint8))
    for name in ("w", "wt"):
        assert all(torch.equal(a, b) for a, b in zip(fw._held(name), again._held(name)))
    assert fw.to(torch.bfloat16).dequantize().dtype == torch.float32
    assert np.array_equal(ref.f64(fw.dequantize()), got)


# ---------------------------------------------------------------- exact products
def whole(shape, gen, dev, most=2):
    return torch.randint(-most, most + 1, shape, generator=gen, device=dev).float()


def pow2(shape, gen, dev):
    return torch.exp2(torch.randint(-3, 4, shape, generator=gen, device=dev).float())


def whole_rows(M, K, gen, dev):
    codes = torch.zeros(M, padded(K), device=dev)
    codes[:, :K] = whole((M, K), gen, dev)
    return Fp8Rows(codes.to(E4M3), pow2((M, blocks(K)), gen, dev), K)


def spread(M, E, seed):
    """Offsets of E groups within M rows, some of them empty, some rows of none."""
    rng = np.random.default_rng(seed)
    cuts = np.sort(rng.integers(0, M + 1, E + 1))
    if E > 3:
        cuts[2] = cuts[1]
    if seed % 2 == 0:
        cuts[0], cuts[-1] = 0, M
    return np.sort(cuts).astype(np.int32)


SHAPES = [(1, 1, 1, 1), (1, 16, 128, 1), (1, 4096, 512, 3), (5, 130, 200, 4), (16, 64, 2048, 2), (17, 33, 384, 1),
          (64, 300, 1000, 7), (65, 256, 128, 1), (130, 515, 260, 5), (257, 1024, 640, 1), (300, 1000, 1248, 12),
          (1000, 272, 144, 64), (2000, 768, 256, 3), (777, 2049, 136, 2), (3000, 512, 896, 8), (40, 64, 64, 256),
          # items of the last round cut along the columns, on both tile heights
          (1500, 1040, 2100, 3), (700, 514, 4096, 2), (130, 1000, 3300, 5), (33, 2100, 4000, 1), (4000, 4200, 2048, 9),
          # tiles of 256 rows, whole and in parts, few columns and many
          (2600, 8000, 1100, 5), (1700, 16390, 136, 1), (900, 33000, 260, 4)]


@pytest.mark.parametrize("M,N,K,E", SHAPES)
def test_whole_numbers_are_exact(M, N, K, E, dev):
    banner(f"fp8 matmul exact M={M} N={N} K={K} E={E}")
    gen = torch.Generator(device=dev).manual_seed(M + N)
    x = whole_rows(M, K, gen, dev)
    wv, ws = whole((E, N, K), gen, dev), pow2((E, blocks(N), blocks(K)), gen, dev)
    weight = Fp8Weight.from_codes(wv.to(E4M3), ws, transposed=True)
    offsets = spread(M, E, M + E) if E > 1 or M % 3 == 0 else None
    xv = x.dequantize().double()
    want = torch.zeros(M, N, dtype=torch.float64, device=dev)
    wd = weight.dequantize().double()
    bounds = [0, M] if offsets is None else offsets
    for e in range(E):
        a, b = int(bounds[e]), int(bounds[e + 1])
        want[a:b] = xv[a:b] @ wd[e].t().contiguous()
    off = None if offsets is None else torch.from_numpy(offsets).to(dev)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        got = matmul_fp8(x, weight, off, out_dtype=dt)
        assert got.dtype == dt and torch.equal(got, want.float().to(dt))
    # transposed matrices, through the gradient: the result's gradient as whole numbers whose
    # blocks' largest is 448, so that its codes are themselves
    d = whole((M, N), gen, dev)
    d[:, ::128] = 448.0
    xr = torch.zeros(M, K, device=dev, requires_grad=True)
    dx = torch.autograd.grad(matmul_fp8(xr, weight, off), xr, d)[0]
    want = torch.zeros(M, K, dtype=torch.float64, device=dev)
    for e in range(E):
        a, b = int(bounds[e]), int(bounds[e + 1])
        want[a:b] = d[a:b].double() @ wd[e]
    # 448 times 2 and sums of 127 twos need 11 bits and no more
    assert torch.equal(dx, want.float())


# ------------------------------------------------------------- products in general
@pytest.mark.parametrize("M,N,K,E", [(1, 512, 1024, 2), (33, 260, 1248, 3), (333, 1000, 520, 4), (512, 640, 2048, 1)])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_products_and_their_gradient(M, N, K, E, dt, dev):
    banner(f"fp8 matmul M={M} N={N} K={K} E={E} {dt}")
    dt = DT[dt]
    g = torch.Generator(device=dev).manual_seed(M)
    x = (torch.randn(M, K, generator=g, device=dev) * torch.exp(torch.randn(K, generator=g, device=dev))).to(dt)
    dout = torch.randn(M, N, generator=g, device=dev).to(dt)
    weight = Fp8Weight.quantize(torch.randn(E, N, K, generator=g, device=dev) * 0.02, transposed=True)
    offsets = spread(M, E, 2 * M)
    x.requires_grad_()
    out = matmul_fp8(x, weight, torch.from_numpy(offsets).to(dev))
    dx = torch.autograd.grad(out, x, dout)[0]
    w = ref.f64(weight.dequantize())
    for got, v, t in ((out, x, False), (dx, dout, True)):
        rows = ref.f64(quantize_fp8(v).dequantize())
        for e in range(E):
            a, b = offsets[e], offsets[e + 1]
            want, off = ref.matmul(rows[a:b], w[e].T if t else w[e])
            # dequantize rounds code * scale to fp32, on both sides
            off += 2.0 ** -22 * (np.abs(rows[a:b]) @ np.abs(w[e] if t else w[e].T))
            assert (np.abs(ref.f64(got[a:b]) - want) <= rounded(dt, want) + 1.01 * off).all()
    again = matmul_fp8(x, weight, torch.from_numpy(offsets).long().to(dev))
    assert torch.equal(again, out)
    assert torch.equal(matmul_fp8(quantize_fp8(x), weight, torch.from_numpy(offsets).to(dev), out_dtype=dt), out)


def test_gradient_against_differences(dev):
    """x on the values that 8 bits hold: the product is linear between them."""
    banner("fp8 matmul differences")
    g = torch.Generator(device=dev).manual_seed(0)
    M, N, K = 8, 96, 160
    weight = Fp8Weight.quantize(torch.randn(N, K, generator=g, device=dev), transposed=True)
    x = torch.randn(M, K, generator=g, device=dev).requires_grad_()
    dout = quantize_fp8(torch.randn(M, N, generator=g, device=dev)).dequantize()
    dx = ref.f64(torch.autograd.grad(matmul_fp8(x, weight), x, dout)[0])
    w, d = ref.f64(weight.dequantize())[0], ref.f64(dout)
    rng = np.random.default_rng(1)
    for _ in range(4):
        a, h = rng.standard_normal((M, K)), 0.5
        x64 = ref.f64(x)
        diff = ((((x64 + h * a) @ w.T) - ((x64 - h * a) @ w.T)) * d).sum() / (2 * h)
        _, off = ref.matmul(d, w.T)
        assert abs((dx * a).sum() - diff) <= ((off + 2.0 ** -20 * (np.abs(d) @ np.abs(w))) * np.abs(a)).sum()


def test_not_a_number_stays_in_its_row_and_column(dev):
    banner("fp8 matmul NaN")
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn(70, 300, generator=g, device=dev).bfloat16()
    w = torch.randn(1, 200, 300, generator=g, device=dev)
    clean = matmul_fp8(x, Fp8Weight.quantize(w))
    x[9, 17] = float("inf")
    w[0, 150, 40] = float("nan")
    out = matmul_fp8(x, Fp8Weight.quantize(w))
    bad = torch.zeros(70, 200, dtype=torch.bool, device=dev)
    bad[9], bad[:, 150] = True, True
    assert torch.equal(torch.isnan(out), bad)
    far = torch.ones(200, dtype=torch.bool, device=dev)
    far[128:] = False  # the block of the NaN has other scales
    rows = [i for i in range(70) if i != 9]
    assert torch.equal(out[rows][:, far], clean[rows][:, far])


def test_no_rows_and_views(dev):
    banner("fp8 matmul views")
    g = torch.Generator(device=dev).manual_seed(6)
    weight = Fp8Weight.quantize(torch.randn(40, 96, generator=g, device=dev), transposed=True)
    empty = torch.empty(0, 96, device=dev, requires_grad=True)
    out = matmul_fp8(empty, weight)
    assert out.shape == (0, 40) and torch.autograd.grad(out, empty, out)[0].shape == (0, 96)
    big = torch.randn(33, 300, generator=g, device=dev).bfloat16()
    v = big[:, 5:101]
    assert torch.equal(matmul_fp8(v, weight), matmul_fp8(v.contiguous(), weight))
    offsets = torch.tensor([7, 7], dtype=torch.int32, device=dev)
    assert not matmul_fp8(v, weight, offsets).any()
    strided = torch.tensor([0, 9, 33, 9], dtype=torch.int32, device=dev)[::2]
    assert torch.equal(matmul_fp8(v, weight, strided), matmul_fp8(v, weight))
    # codes that start off 16 bytes
    codes, scales = weight.codes()
    raw = torch.empty(codes.numel() + 3, dtype=torch.uint8, device=dev)[3:].view(codes.shape)
    raw.copy_(codes.view(torch.uint8))
    odd = Fp8Weight.from_codes(raw, scales)
    assert torch.equal(matmul_fp8(v, odd), matmul_fp8(v, weight))


# ------------------------------------------------------------------- the experts
REL = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def make_experts(E, H, I, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    w1 = torch.randn(E, 2 * I, H, generator=g, device=dev) / H ** 0.5
    w2 = torch.randn(E, H, I, generator=g, device=dev) / I ** 0.5
    return Fp8Experts.quantize(w1, w2)


@pytest.mark.parametrize("T,H,I,E,K,act", [
    (1, 256, 512, 4, 2, "silu"), (1, 64, 16, 1, 1, "gelu"), (7, 400, 336, 8, 3, "gelu_tanh"),
    (16, 512, 256, 64, 6, "silu"), (100, 256, 128, 2, 1, "silu"), (260, 384, 1040, 4, 2, "gelu"),
    (1100, 256, 640, 6, 2, "silu"), (33, 16, 144, 256, 8, "silu"),
    # gate|up on tiles of 256 rows, in parts too
    (1200, 256, 9008, 4, 2, "gelu"), (1300, 2048, 6000, 2, 1, "silu"),
    # down on tiles of 256 rows (bf16: to slots of 16 bits), in parts too
    (1792, 4112, 144, 4, 2, "silu"), (1792, 4112, 2064, 4, 2, "gelu_tanh")])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_experts(T, H, I, E, K, act, dt, dev):
    """Off by half a step of the type (and 2^-12 where bf16 slots wait in f16); and an
    intermediate whose quotient lies as near to a border as the sums are exact becomes the other
    neighbour, 2^-3 away at most. In bf16 the matrix core's sums are (2^-14): a share of 2^-14 / 2^-4 of them, so 2^-3 * 2^-5 = 2^-8 in the
    norm. Sums of exact products in fp32 are to 2^-18: 2^-3 * 2^-7 = 2^-10."""
    banner(f"fp8 experts T={T} H={H} I={I} E={E} K={K} {act} {dt}")
    dt = DT[dt]
    ex = make_experts(E, H, I, dev, seed=T)
    g = torch.Generator(device=dev).manual_seed(T + 1)
    x = torch.randn(T, H, generator=g, device=dev).to(dt)
    ids = torch.argsort(torch.rand(T, E, generator=g, device=dev), -1)[:, :K]
    tw = torch.rand(T, K, generator=g, device=dev)
    ids[0, 0] = -1  # elsewhere
    if T > 2:
        tw[2, 0] = 0.0
    got = fused_experts_fp8(x, ex, tw, ids, activation=act)
    want = ref.experts(ref.f64(x), ref.f64(ex.dequantize("w1")), ref.f64(ex.dequantize("w2")),
                       ref.f64(tw), ids.cpu().numpy(), act)
    rel = np.linalg.norm(ref.f64(got) - want) / max(np.linalg.norm(want), 1e-30)
    assert got.dtype == dt and rel <= REL[dt] + 2.0 ** (-8 if dt == torch.bfloat16 else -10)
    rows = quantize_fp8(x)
    assert torch.equal(fused_experts_fp8(rows, ex, tw, ids.int(), activation=act, out_dtype=dt), got)
    other = fused_experts_fp8(x, ex, tw, ids, activation=act, out_dtype=torch.float32)
    rel = np.linalg.norm(ref.f64(other) - want) / max(np.linalg.norm(want), 1e-30)
    assert other.dtype == torch.float32 and rel <= 2.0 ** -10


def test_operators_together(dev):
    """Norm, tokens to their experts, products, activation, products and back, as a training
    program runs them, and the same experts as one call. In bf16, with the gradients of a
    16-bit layer's formulas in fp32 through the same roundings."""
    from reframework_amd.layers import LayerNorm

    banner("operators together")
    T, H, I, E, K = 200, 256, 384, 6, 2
    ex = make_experts(E, H, I, dev, seed=8)
    w1 = Fp8Weight.from_codes(*ex.codes("w1"), transposed=True)
    w2 = Fp8Weight.from_codes(*ex.codes("w2"), transposed=True)
    norm = LayerNorm(H, 1e-5).to(dev)
    g = torch.Generator(device=dev).manual_seed(9)
    x = torch.randn(T, H, generator=g, device=dev, requires_grad=True)
    res = torch.randn(T, H, generator=g, device=dev)
    ids = torch.argsort(torch.rand(T, E, generator=g, device=dev), -1)[:, :K]
    tw = torch.rand(T, K, generator=g, device=dev, requires_grad=True)
    normed, new_res = norm.forward_add_residual(x, res)
    rows, order = permute_tokens(normed, ids, E)
    gate, up = matmul_fp8(rows, w1, order.offsets).chunk(2, -1)
    y = matmul_fp8(torch.nn.functional.silu(gate) * up, w2, order.offsets)
    out = combine_tokens(y, order, tw) + new_res
    whole_call = fused_experts_fp8(normed, ex, tw, ids) + new_res
    # the same sums, but for tipped codes of the intermediate
    assert float(((out - whole_call).norm() / (whole_call - new_res).norm()).detach()) <= 2.0 ** -8
    dout = torch.randn(T, H, generator=g, device=dev)
    got = torch.autograd.grad(out, [x, tw, norm.weight, norm.bias], dout)

    # the same chain from plain operations; the products through the same roundings
    class Product(torch.autograd.Function):
        @staticmethod
        def forward(ctx, a, w):
            ctx.w = w
            return quantize_fp8(a).dequantize() @ w.t().contiguous()

        @staticmethod
        def backward(ctx, d):
            return quantize_fp8(d).dequantize() @ ctx.w, None

    n2 = torch.nn.functional.layer_norm(x + res, (H,), norm.weight, norm.bias, 1e-5)
    acc = x + res
    d1, d2 = w1.dequantize(), w2.dequantize()
    for e in range(E):
        t, k = torch.nonzero(ids == e, as_tuple=True)
        gate, up = Product.apply(n2[t], d1[e]).chunk(2, -1)
        y = Product.apply(torch.nn.functional.silu(gate) * up, d2[e])
        acc = acc.index_add(0, t, y * tw[t, k, None])
    want = torch.autograd.grad(acc, [x, tw, norm.weight, norm.bias], dout)
    for a, b in zip(got, want):
        assert float((a - b).norm() / b.norm()) <= 2.0 ** -6  # codes of three chained products tip


def test_streams_graphs_and_workspaces(dev):
    banner("fp8 graph")
    T, H, I, E, K = 64, 256, 384, 6, 2
    ex = make_experts(E, H, I, dev, seed=10)
    weight = Fp8Weight.quantize(torch.randn(E, 320, H, device=dev), transposed=True)
    x = torch.randn(T, H, device=dev).bfloat16()
    ids = torch.randint(0, E, (T, K), device=dev)
    tw = torch.rand(T, K, device=dev)
    dout = torch.randn(T * K, 320, device=dev).bfloat16()

    def step():
        out = fused_experts_fp8(x, ex, tw, ids)
        rows, order = permute_tokens(x, ids, E)
        leaf = rows.detach().requires_grad_()
        y = matmul_fp8(leaf, weight, order.offsets)
        return out, y.detach(), torch.autograd.grad(y, leaf, dout)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs have workspaces of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(4):
        gen = torch.Generator(device=dev).manual_seed(i)
        x.copy_(torch.randn(T, H, generator=gen, device=dev))
        ids.copy_(torch.randint(-1, E, (T, K), generator=gen, device=dev))
        torch.cuda.synchronize()
        for (graph, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        for _, held in graphs:
            assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_against_16_bit_experts(dev):
    """The layer that the weights came from: e4m3 keeps 4 bits, off by 2^-4 / sqrt(12) per
    product, of which three follow each other."""
    banner("fp8 experts against bf16")
    T, H, I, E, K = 48, 512, 256, 4, 2
    g = torch.Generator(device=dev).manual_seed(3)
    w1 = (torch.randn(E, 2 * I, H, generator=g, device=dev) / H ** 0.5).bfloat16()
    w2 = (torch.randn(E, H, I, generator=g, device=dev) / I ** 0.5).bfloat16()
    x = torch.randn(T, H, generator=g, device=dev).bfloat16()
    ids = torch.argsort(torch.rand(T, E, generator=g, device=dev), -1)[:, :K]
    tw = torch.rand(T, K, generator=g, device=dev)
    a = fused_experts(x, w1, w2, tw, ids).float()
    b = fused_experts_fp8(x, Fp8Experts.quantize(w1, w2), tw, ids).float()
    assert float((a - b).norm() / a.norm()) <= 0.08


def test_no_second_derivatives(dev):
    """First derivatives under create_graph are as without; a second one is refused."""
    banner("no second derivatives")
    norm = LayerNorm(256, 1e-5).to(dev)
    x = torch.randn(9, 256, device=dev, requires_grad=True)
    ids = torch.tensor([[0, 1]] * 9, device=dev)
    w = torch.rand(9, 2, device=dev, requires_grad=True)
    weight = Fp8Weight.quantize(torch.randn(2, 128, 256, device=dev), transposed=True)

    def both(v):
        rows, order = permute_tokens(v, ids, 2)
        return combine_tokens(rows, order, w)

    def product(v):
        return matmul_fp8(v, weight, torch.tensor([0, 4, 9], dtype=torch.int32, device=dev))

    for f in (norm, both, product):
        first, = torch.autograd.grad(f(x).square().sum(), [x])
        again, = torch.autograd.grad(f(x).square().sum(), [x], create_graph=True)
        assert torch.equal(first, again)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            again.sum().backward()


def test_no_derivatives_forwards(dev):
    """A tangent would be lost: refused, where nothing asks for a gradient too."""
    from torch.autograd import forward_ad

    banner("no derivatives forwards")
    norm = LayerNorm(256, 1e-5).to(dev).requires_grad_(False)
    x, t = torch.randn(9, 256, device=dev), torch.randn(9, 256, device=dev)
    ids = torch.tensor([[0, 1]] * 9, device=dev)
    weight = Fp8Weight.quantize(torch.randn(128, 256, device=dev), transposed=True)
    rows, order = permute_tokens(x, ids, 2)
    w = torch.rand(9, 2, device=dev)
    calls = [(norm, x), (lambda v: norm.forward_add_residual(x, v), x), (lambda v: permute_tokens(v, ids, 2), x),
             (lambda v: combine_tokens(v, order, w), rows), (lambda v: combine_tokens(rows, order, v), w),
             (lambda v: matmul_fp8(v, weight), x)]
    for f, v in calls:
        f(v)
        with forward_ad.dual_level():
            f(v)  # without a tangent
            dual = forward_ad.make_dual(v, torch.ones_like(v))
            with pytest.raises(NotImplementedError, match="forward mode"):
                f(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
                f(dual)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward_inplace"):
            norm.forward_inplace(forward_ad.make_dual(x.clone(), t))


def test_weights_do_not_follow_the_tensors_they_came_from(dev):
    """A loader may fill the next layer into the buffers of the last one."""
    banner("fp8 weights are copies")
    g = torch.Generator(device=dev).manual_seed(12)
    codes = torch.randn(2, 160, 256, generator=g, device=dev).to(E4M3)
    scales = torch.rand(2, 2, 2, generator=g, device=dev) + 0.5
    want = codes.float() * scales.repeat_interleave(128, 1)[:, :160].repeat_interleave(128, 2)
    weight = Fp8Weight.from_codes(codes, scales, transposed=True)
    again = Fp8Weight.from_codes(*weight.codes(), transposed=True)
    w1, w2 = torch.randn(2, 64, 256, device=dev).to(E4M3), torch.randn(2, 256, 32, device=dev).to(E4M3)
    s1, s2 = torch.rand(2, 2, 2, device=dev), torch.rand(2, 2, 1, device=dev)
    experts = Fp8Experts.from_codes(w1, s1, w2, s2)
    held = [experts.dequantize(n).clone() for n in ("w1", "w2")]
    for t in (scales, s1, s2):
        t.zero_()
    weight.codes()[1].zero_()
    for t in (codes, w1, w2):
        t.view(torch.uint8).zero_()
    assert torch.equal(weight.dequantize(), want) and torch.equal(again.dequantize(), want)
    assert all(torch.equal(experts.dequantize(n), h) for n, h in zip(("w1", "w2"), held))
    experts.codes("w1")[1].zero_(), experts.codes("w2")[1].zero_()
    assert all(torch.equal(experts.dequantize(n), h) for n, h in zip(("w1", "w2"), held))


def test_differences_of_the_product_itself(dev):
    """matmul_fp8 at x + a and x - a, both on codes: whole numbers beside a 448 in every block. Sums
    are exact then, and so is half their difference against the gradient."""
    banner("fp8 matmul, differences of the calls")
    gen = torch.Generator(device=dev).manual_seed(13)
    M, N, K, E = 90, 300, 400, 3
    weight = Fp8Weight.from_codes(whole((E, N, K), gen, dev).to(E4M3), pow2((E, blocks(N), blocks(K)), gen, dev),
                                  transposed=True)
    offsets = torch.tensor([4, 33, 33, 87], dtype=torch.int32, device=dev)
    x, d = whole((M, K), gen, dev, 8), whole((M, N), gen, dev, 8)
    x[:, ::128], d[:, ::128] = 448.0, 448.0
    leaf = x.clone().requires_grad_()
    out = matmul_fp8(leaf, weight, offsets)
    dx = torch.autograd.grad(out, leaf, d)[0].double()
    for _ in range(4):
        a = whole((M, K), gen, dev, 1)
        a[:, ::128] = 0.0  # the blocks' largest stay
        up, down = (matmul_fp8(x + s * a, weight, offsets).double() for s in (1.0, -1.0))
        assert torch.equal((up + down) / 2, out.detach().double())
        rows = ((up - down) / 2 * d.double()).sum(1)
        assert torch.equal(rows, (dx * a.double()).sum(1)) and rows[4:87].abs().min() > 0
        assert not rows[:4].any() and not rows[87:].any()
