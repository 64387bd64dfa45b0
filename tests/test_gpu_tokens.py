"""Tokens by expert and back on the GPU, with gradients, against 64 bits.

Moves are exact. A sum of n products in fp32 is off by at most n 2^-23 of the sum of their
magnitudes (each product and each addition is rounded), and once by half a step of its own type:
eps / 2 relative to the value, or half of the smallest number of the type where that is more
(float16 below 2^-14 has steps of 2^-24 whatever the value).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from _helpers import DT, banner
from reframework_amd.moe import TokenOrder, combine_tokens, permute_tokens, token_order

pytestmark = pytest.mark.gpu


def rounded(dt, v):
    """What rounding v to dt may be off by."""
    f = torch.finfo(dt)
    return np.maximum(f.eps / 2 * np.abs(v), f.tiny * f.eps / 2)


def f64(t):
    return t.detach().double().cpu().numpy()


def routing(T, K, E, seed, drop=0.0, skew=0.0):
    rng = np.random.default_rng(seed)
    p = np.arange(1, E + 1.0) ** -skew
    ids = np.stack([rng.choice(E, size=K, replace=False, p=p / p.sum()) for _ in range(T)])
    if drop:
        ids[rng.random((T, K)) < drop] = rng.choice([-1, E, E + 7])
    return ids.astype(np.int64), rng.random((T, K)).astype(np.float32)


def order64(ids, E):
    flat = ids.reshape(-1)
    ok = (flat >= 0) & (flat < E)
    order = np.argsort(np.where(ok, flat, E), kind="stable")[:ok.sum()]
    row = np.full(flat.size, -1)
    row[order] = np.arange(order.size)
    offsets = np.searchsorted(np.sort(flat[ok]), np.arange(E + 1))
    return offsets, row.reshape(ids.shape), order // ids.shape[1]


def data(T, R, H, dt, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(n, H, generator=g, device=dev).to(dt) for n in (T, R, R, T)]


CASES = [(1, 1, 1, 1, 0.0), (1, 8, 1, 1, 0.0), (1, 4096, 8, 2, 0.0), (5, 33, 3, 3, 0.5), (16, 2048, 64, 6, 0.0),
         (37, 257, 256, 8, 0.3), (400, 1000, 12, 3, 0.5), (130, 8200, 5, 2, 0.2), (64, 96, 4, 2, 1.0),
         (2100, 520, 16, 2, 0.1), (700, 12, 256, 9, 0.0)]


@pytest.mark.parametrize("T,H,E,K,drop", CASES)
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_there_and_back_with_gradients(T, H, E, K, drop, dt, dev):
    banner(f"tokens T={T} H={H} E={E} K={K} drop={drop} {dt}")
    dt = DT[dt]
    ids, w = routing(T, K, E, seed=T + H, drop=drop, skew=0.5)
    x, y, drows, dout = data(T, T * K, H, dt, dev, seed=H)
    x.requires_grad_(), y.requires_grad_()
    wt = torch.from_numpy(w).to(dev).requires_grad_()
    rows, order = permute_tokens(x, torch.from_numpy(ids).to(dev), E)
    offsets, row, src = order64(ids, E)
    assert np.array_equal(order.offsets.cpu().numpy(), offsets)
    assert np.array_equal(order.slot_to_row.cpu().numpy(), row)
    n = src.size
    assert np.array_equal(order.row_src.cpu().numpy()[:n], src)
    assert torch.equal(rows[:n], x.detach()[torch.from_numpy(src).to(dev)]) and not rows[n:].any()
    out = combine_tokens(y, order, wt)

    y64, on = f64(y), row >= 0
    mine = np.where(on[..., None], y64[row], 0.0)  # [T, K, H]
    terms = w.astype(np.float64)[..., None] * mine
    want, mag = terms.sum(1), np.abs(terms).sum(1)
    assert (np.abs(f64(out) - want) <= rounded(dt, want) + K * 2.0 ** -22 * mag).all()

    dx, dy, dw = torch.autograd.grad([rows, out], [x, y, wt], [drows, dout], retain_graph=True)
    parts = np.where(on[..., None], f64(drows)[row], 0.0)
    want = parts.sum(1)
    assert (np.abs(f64(dx) - want) <= rounded(dt, want) + K * 2.0 ** -22 * np.abs(parts).sum(1)).all()
    want = np.zeros_like(y64)
    want[row[on]] = (w.astype(np.float64)[..., None] * f64(dout)[:, None])[on]
    assert (np.abs(f64(dy) - want) <= rounded(dt, want) + 2.0 ** -23 * np.abs(want)).all()
    prod = f64(dout)[:, None] * mine
    assert (np.abs(f64(dw) - prod.sum(-1)) <= (H + 10) * 2.0 ** -23 * np.abs(prod).sum(-1)).all()
    # the same again, and each alone
    for inputs, one in ((x, dx), (y, dy), (wt, dw)):
        assert torch.equal(torch.autograd.grad([rows, out], inputs, [drows, dout], retain_graph=True)[0], one)
    with torch.no_grad():
        assert torch.equal(permute_tokens(x, torch.from_numpy(ids).int().to(dev), E)[0], rows)
        assert torch.equal(combine_tokens(y, order, wt), out)


def test_gradient_of_the_weights_against_differences(dev):
    """The sum is linear in weights and rows: differences of the 64-bit sum are its gradient."""
    banner("tokens differences")
    T, H, E, K = 20, 48, 5, 2
    ids, w = routing(T, K, E, seed=1, drop=0.2)
    _, y, _, dout = data(T, T * K, H, torch.float32, dev, seed=1)
    wt = torch.from_numpy(w).to(dev).requires_grad_()
    order = token_order(torch.from_numpy(ids).to(dev), E)
    y.requires_grad_()
    dy, dw = torch.autograd.grad(combine_tokens(y, order, wt), [y, wt], dout)
    _, row, _ = order64(ids, E)
    rng = np.random.default_rng(2)

    def loss(y64, w64):
        mine = np.where((row >= 0)[..., None], y64[row], 0.0)
        return ((w64[..., None] * mine).sum(1) * f64(dout)).sum()

    for _ in range(4):
        a, b, h = rng.standard_normal(y.shape), rng.standard_normal(w.shape), 1e-3
        diff = (loss(f64(y) + h * a, w.astype(np.float64)) - loss(f64(y) - h * a, w.astype(np.float64))) / (2 * h)
        assert abs((f64(dy) * a).sum() - diff) <= 1e-6 * np.abs(f64(dy) * a).sum() + 1e-9
        diff = (loss(f64(y), w + h * b) - loss(f64(y), w - h * b)) / (2 * h)
        assert abs((f64(dw) * b).sum() - diff) <= 1e-4 * np.abs(f64(dw) * b).sum() + 1e-9


def test_no_tokens_no_slots_and_strides(dev):
    banner("tokens empty and strided")
    x = torch.randn(0, 16, device=dev, requires_grad=True)
    rows, order = permute_tokens(x, torch.zeros(0, 2, dtype=torch.int64, device=dev), 4)
    out = combine_tokens(rows, order, torch.zeros(0, 2, device=dev))
    assert rows.shape == (0, 16) and out.shape == (0, 16) and not order.offsets.any()
    torch.autograd.grad(out, x, out)
    ids = torch.full((6, 2), -1, device=dev)  # every slot elsewhere
    x = torch.randn(6, 16, device=dev, requires_grad=True)
    w = torch.rand(6, 2, device=dev, requires_grad=True)
    rows, order = permute_tokens(x, ids, 4)
    out = combine_tokens(rows, order, w)
    dx, dw = torch.autograd.grad(out, [x, w], torch.ones_like(out))
    assert not rows.any() and not out.any() and not dx.any() and not dw.any()
    # strided and broadcast inputs, weights of another type
    ids = torch.randint(0, 4, (6, 2), device=dev)
    big = torch.randn(6, 40, device=dev)
    view = big[:, 3:19]
    a, order = permute_tokens(view, ids.t().contiguous().t(), 4)
    assert torch.equal(a, permute_tokens(view.contiguous(), ids, 4)[0])
    shared = torch.rand(6, 1, device=dev, dtype=torch.float64, requires_grad=True)
    out = combine_tokens(a, order, shared.expand(6, 2))
    g = torch.autograd.grad(out, shared, torch.ones_like(out))[0]
    assert g.dtype == torch.float64 and torch.allclose(
        g, combine_tokens(a, order, torch.ones(6, 2, device=dev)).double().sum(1, keepdim=True), rtol=1e-5, atol=1e-5)
    rows = torch.randn(12, 80, device=dev)[:, ::5]
    assert torch.equal(combine_tokens(rows, order, torch.ones(6, 2, device=dev)),
                       combine_tokens(rows.contiguous(), order, torch.ones(6, 2, device=dev)))


def test_infinite_rows_of_others_do_not_reach_a_token(dev):
    """Row 0, which a slot without a row is loaded in place of, holds NaN."""
    banner("tokens NaN")
    ids = torch.tensor([[0, 1], [-1, 1], [1, -1]], device=dev)
    order = token_order(ids, 2)
    rows = torch.ones(6, 24, device=dev)
    rows[0] = float("nan")
    out = combine_tokens(rows, order, torch.full((3, 2), 0.5, device=dev))
    assert bool(torch.isnan(out[0]).all()) and bool((out[1:] == 0.5).all())


def test_streams_and_graphs(dev):
    banner("tokens graph")
    T, H, E, K = 600, 264, 12, 3
    ids, w = routing(T, K, E, seed=9, drop=0.2)
    ids = torch.from_numpy(ids).to(dev)
    x, y, drows, dout = data(T, T * K, H, torch.bfloat16, dev, seed=4)
    x.requires_grad_(), y.requires_grad_()
    wt = torch.from_numpy(w).to(dev).requires_grad_()

    def step():
        rows, order = permute_tokens(x, ids, E)
        out = combine_tokens(y, order, wt)
        return (rows.detach(), order.offsets, order.slot_to_row, out.detach()) + torch.autograd.grad(
            [rows, out], [x, y, wt], [drows, dout])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        new, _ = routing(T, K, E, seed=20 + i, drop=0.1 * i)
        ids.copy_(torch.from_numpy(new))
        x.data.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_slots_of_rows_that_are_not_there(dev):
    """An order that names rows behind the last: they count as none."""
    banner("tokens rows out of range")
    T, H, E, K = 5, 40, 3, 2
    ids, w = routing(T, K, E, seed=3)
    x, y, _, dout = data(T, T * K, H, torch.float32, dev, seed=6)
    order = token_order(torch.from_numpy(ids).to(dev), E)
    bad = TokenOrder(order.offsets, order.slot_to_row.clone(), order.row_src, E)
    bad.slot_to_row[1, 0], bad.slot_to_row[4, 1] = T * K, 2 ** 31 - 1
    wt = torch.from_numpy(w).to(dev).requires_grad_()
    y.requires_grad_()
    out = combine_tokens(y, bad, wt)
    cut = wt.detach().clone()
    cut[1, 0] = cut[4, 1] = 0.0
    assert torch.equal(out.detach(), combine_tokens(y.detach(), order, cut))
    dw, = torch.autograd.grad(out, [wt], [dout])
    assert dw[1, 0] == 0 and dw[4, 1] == 0 and bool((dw != 0).sum() == T * K - 2)


def test_an_order_changed_before_the_backward_pass(dev):
    banner("tokens order changed")
    ids = torch.tensor([[0, 1], [1, 2]], device=dev)
    x = torch.randn(2, 16, device=dev, requires_grad=True)
    rows, order = permute_tokens(x, ids, 3)
    order.slot_to_row.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        rows.sum().backward()
