"""LayerNorm, tokens by expert and back and the 8-bit products on more than 2^31 elements: places
past 32 bits. The last rows are compared with a call on those rows alone, which has none."""

from __future__ import annotations

import pytest
import torch

from _helpers import banner
from reframework_amd.fp8 import E4M3, Fp8Rows
from reframework_amd.layers import LayerNorm
from reframework_amd.moe import (Fp8Experts, Fp8Weight, combine_tokens, fused_experts_fp8, matmul_fp8,
                                 permute_tokens)

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
LAST = 40


@pytest.fixture(autouse=True)
def give_back():
    """The memory of a test here goes back to the device, not to the tests behind it."""
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def random(shape, dev, seed, dtype=BF16):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.empty(shape, dtype=dtype, device=dev).normal_(generator=g)


def off(got, want):
    """Distance relative to the size of what is wanted."""
    got, want = got.double(), want.double()
    return float((got - want).norm() / want.norm())


def test_layer_norm(dev):
    T, H = 265_000, 8192
    banner("layer_norm of more than 2^31 elements")
    norm = LayerNorm(H, 1e-5).to(dev)
    x = random((T, H), dev, 1).requires_grad_()
    dy = random((T, H), dev, 2)
    out = norm(x)
    dx, = torch.autograd.grad(out, [x], [dy])
    tail = x.detach()[-LAST:].clone().requires_grad_()
    want = norm(tail)
    # a row's result and gradient do not depend on the others
    assert torch.equal(out.detach()[-LAST:], want.detach())
    assert torch.equal(dx[-LAST:], torch.autograd.grad(want, [tail], [dy[-LAST:]])[0])


def test_tokens(dev):
    T, H, E = 265_000, 8192, 3
    banner("tokens of more than 2^31 elements")
    x = random((T, H), dev, 3).requires_grad_()
    ids = torch.full((T, 1), 2, device=dev)
    ids[:100] = 0  # the last tokens' rows are the last ones
    rows, order = permute_tokens(x, ids, E)
    assert torch.equal(rows.detach()[-LAST:], x.detach()[-LAST:])
    w = torch.full((T, 1), 0.5, device=dev, requires_grad=True)
    out = combine_tokens(rows, order, w)
    assert torch.equal(out.detach()[-LAST:], x.detach()[-LAST:] * 0.5)
    dx, dw = torch.autograd.grad(out, [x, w], [rows.detach()])
    assert torch.equal(dx[-LAST:], x.detach()[-LAST:] * 0.5)
    want = (x.detach()[-LAST:].double() ** 2).sum(1)
    # products and sums of 8192 values in fp32
    assert bool(((dw[-LAST:, 0].double() - want).abs() <= 8192 * 2.0 ** -23 * want).all())


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_products(dtype, dev):
    M, K, N, E = 265_000, 8192, 8192, 2
    banner(f"8-bit products of more than 2^31 elements to {dtype}")
    codes = torch.empty(M, K, dtype=torch.uint8, device=dev).random_(0x30, 0x40)
    x = Fp8Rows(codes.view(E4M3), torch.rand(M, K // 128, device=dev) + 0.5, K)
    w = Fp8Weight.quantize(random((E, N, K), dev, 4))
    offsets = torch.tensor([0, 1000, M], dtype=torch.int32, device=dev)
    out = matmul_fp8(x, w, offsets, out_dtype=dtype)
    tail = Fp8Rows(x.padded_codes[-LAST:], x.scales[-LAST:], K)
    want = matmul_fp8(tail, w, torch.tensor([0, 0, LAST], dtype=torch.int32, device=dev), out_dtype=dtype)
    # a step's sum is off by 2^-11 of its largest product at most, a result of 64 steps of
    # random signs by less than 2^-9 of its size; rounding adds 2^-8 on each side
    assert off(out[-LAST:], want) <= 2.0 ** -6


def test_experts(dev):
    T, H, I, E, K = 70_000, 256, 16384, 2, 2
    banner("8-bit experts whose intermediate rows pass 2^31 bytes")
    x = random((T, H), dev, 5)
    experts = Fp8Experts.quantize(random((E, 2 * I, H), dev, 6) / 16, random((E, H, I), dev, 7) / 128)
    ids = torch.tensor([[0, 1]], device=dev).expand(T, 2)
    w = torch.rand(T, K, device=dev)
    out = fused_experts_fp8(x, experts, w, ids)
    want = fused_experts_fp8(x[-LAST:], experts, w[-LAST:], ids[-LAST:])
    # the intermediate values may fall on neighbouring codes, 2^-3 of a value apart at most
    assert off(out[-LAST:], want) <= 2.0 ** -3


def test_experts_in_parts(dev):
    """Tokens of more than 2 GB in 8 bits: the call runs in two parts."""
    T, H, I, E = 262_143 + LAST, 8192, 16, 2
    banner("8-bit experts in parts")
    x = random((T, H), dev, 8)
    experts = Fp8Experts.quantize(random((E, 2 * I, H), dev, 9) / 90, random((E, H, I), dev, 10) / 4)
    ids = torch.arange(T, device=dev)[:, None] % E
    w = torch.rand(T, 1, device=dev)
    out = fused_experts_fp8(x, experts, w, ids)
    for part in (slice(0, LAST), slice(262_143 - LAST, 262_143), slice(262_143, T)):
        want = fused_experts_fp8(x[part], experts, w[part], ids[part])
        assert off(out[part], want) <= 2.0 ** -3  # as above
