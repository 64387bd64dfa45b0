"""8-bit products and experts on every kernel they have (tests/test_fp8_paths.py holds that the
sizes reach them), element by element.

Products of small whole numbers with scales of powers of two are exact, so equality is asked for.
An expert's products with w1 are exact too; what each element of the result may then be off by
follows from the activation's roundings, the codes those may move across a border, down's sums,
the slots' storage and the result's own rounding (_fp8_paths.experts)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import _fp8_paths as paths
from _helpers import DT, banner
from reframework_amd.fp8 import E4M3, Fp8Rows, blocks, padded
from reframework_amd.moe import Fp8Experts, Fp8Weight, fused_experts_fp8, matmul_fp8

pytestmark = pytest.mark.gpu


def cuts(M, E, seed):
    """Offsets of E groups of about M / E rows each, one of them empty, some rows of none."""
    rng = np.random.default_rng(seed)
    at = np.linspace(3, M - 2, E + 1) + rng.integers(-(M // E // 3), M // E // 3 + 1, E + 1)
    at = np.sort(np.clip(np.round(at), 0, M))
    if E > 4:
        at[3] = at[2]
    return at.astype(np.int32)


def grouped(v, w, offsets, transposed=False):
    out = torch.zeros(v.shape[0], w.shape[2 if transposed else 1], dtype=torch.float64, device=v.device)
    for e in range(w.shape[0]):
        a, b = int(offsets[e]), int(offsets[e + 1])
        out[a:b] = v[a:b] @ (w[e] if transposed else w[e].t().contiguous())
    return out


@pytest.mark.parametrize("M,N,K,E", paths.PRODUCTS)
def test_products(M, N, K, E, dev):
    banner(f"fp8 products by kernel M={M} N={N} K={K} E={E}")
    gen = torch.Generator(device=dev).manual_seed(M + K)
    codes = torch.zeros(M, padded(K), device=dev)
    codes[:, :K] = paths.whole((M, K), gen, dev)
    x = Fp8Rows(codes.to(E4M3), paths.powers((M, blocks(K)), gen, dev, -3, 3), K)
    weight = Fp8Weight.from_codes(paths.whole((E, N, K), gen, dev).to(E4M3),
                                  paths.powers((E, blocks(N), blocks(K)), gen, dev, -3, 3), transposed=True)
    offsets = cuts(M, E, M)
    off = torch.from_numpy(offsets).to(dev)
    w = weight.dequantize().double()
    want = grouped(x.dequantize().double(), w, offsets)
    for dt in DT.values():
        got = matmul_fp8(x, weight, off, out_dtype=dt)
        wrong = got != want.float().to(dt)
        assert not wrong.any(), (dt, int(wrong.sum()), torch.nonzero(wrong)[:4].tolist())
    # Gradients in each type: blocks whose largest is 448 are their own codes. 448 times 2 and the
    # sums of 127 fours are below 2^11, and a sum of steps below 2^24 times the least scale.
    d = paths.whole((M, N), gen, dev)
    d[:, ::128] = 448.0
    want = grouped(d.double(), w, offsets, transposed=True)
    for dt in DT.values():
        leaf = torch.zeros(M, K, dtype=dt, device=dev, requires_grad=True)
        dx = torch.autograd.grad(matmul_fp8(leaf, weight, off), leaf, d.to(dt))[0]
        wrong = dx != want.float().to(dt)
        assert not wrong.any(), (dt, int(wrong.sum()), torch.nonzero(wrong)[:4].tolist())


@pytest.mark.parametrize("T,H,I,E,K,act", paths.EXPERTS)
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_experts(T, H, I, E, K, act, dt, dev):
    banner(f"fp8 experts by kernel T={T} H={H} I={I} E={E} K={K} {act} {dt}")
    dt = DT[dt]
    gen = torch.Generator(device=dev).manual_seed(T + I)
    experts = Fp8Experts.from_codes(*paths.expert_codes(H, I, E, gen, dev))
    v = paths.whole((T, H), gen, dev)
    codes = torch.zeros(T, padded(H), device=dev)
    codes[:, :H] = v
    x = Fp8Rows(codes.to(E4M3), torch.ones(T, blocks(H), device=dev), H)
    ids = torch.argsort(torch.rand(T, E, generator=gen, device=dev), -1)[:, :K]
    tw = torch.rand(T, K, generator=gen, device=dev) + 0.25
    ids[1, 0], ids[T // 2, K - 1] = -1, E  # elsewhere
    tw[2, 0] = 0.0
    got = fused_experts_fp8(x, experts, tw, ids, activation=act, out_dtype=dt)
    want = paths.experts(v.double(), experts.dequantize("w1").double(), experts.dequantize("w2").double(), tw, ids,
                         act, dt, narrow=dt == torch.bfloat16 and K > 1)
    # dequantize rounds codes times scales of w2 to fp32, a share of 2^-24 of down's products
    wrong = (got.double() - want.value).abs() > want.off * (1.0 + 2.0 ** -10)
    assert got.dtype == dt and not wrong.any(), (int(wrong.sum()), torch.nonzero(wrong)[:4].tolist())
    assert torch.equal(fused_experts_fp8(x, experts, tw, ids.int(), activation=act, out_dtype=dt), got)
