"""LayerNorm and its gradients on the GPU, against 64 bits.

Bounds: a result is off by half a step of its own type (eps / 2 relative to the value, or half of
the type's smallest number: float16 below 2^-14 has steps of 2^-24 whatever the value) and by what
fp32 sums of up to 16384 terms in a tree of under 80 additions a path may lose: g = 2^-17 of
the sum of magnitudes. With A = rstd * mean|r|, xhat is then off by ex = g (A + |xhat|), and
the gradients by what that and g do to their formula's terms; dw and db add the sums over T
rows, (T + 700) 2^-24 of their magnitudes. The same gradients are held against differences of
the formula in 64 bits.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from _helpers import DT, banner
from reframework_amd.layers import LayerNorm, RMSNorm
from reframework_amd.moe import FusedMoE

pytestmark = pytest.mark.gpu
EPS = 1e-5
G = 2.0 ** -17


def half(dt):
    return torch.finfo(dt).eps / 2


def rounded(dt, v):
    """What rounding v to dt may be off by."""
    f = torch.finfo(dt)
    return np.maximum(f.eps / 2 * np.abs(v), f.tiny * f.eps / 2)


def f64(t):
    return t.detach().double().cpu().numpy()


def forward64(r, w, b):
    mean = r.mean(-1, keepdims=True)
    rstd = 1.0 / np.sqrt(((r - mean) ** 2).mean(-1, keepdims=True) + EPS)
    return (r - mean) * rstd * w + b, mean, rstd


def make(T, H, dt, wdt, dev, seed=0, bias=True):
    g = torch.Generator(device=dev).manual_seed(seed)

    def n(mean, sigma, *shape, d=dt):
        return (torch.randn(*shape, generator=g, device=dev) * sigma + mean).to(d)

    norm = LayerNorm(H, EPS, bias=bias).to(dev)
    norm.weight.data = n(1.0, 0.2, H, d=wdt)
    if bias:
        norm.bias.data = n(0.0, 0.2, H, d=wdt)
    return norm, n(0.3, 1.0, T, H), n(0.5, 2.0, T, H), n(0.0, 1.0, T, H), n(0.1, 1.0, T, H)


def check_forward(out, r, w, b, dt):
    want, mean, rstd = forward64(r, w, b)
    xhat = (r - mean) * rstd
    ex = G * (rstd * np.abs(r).mean(-1, keepdims=True) + np.abs(xhat)) * np.abs(w)
    bound = rounded(dt, want) + (1 + half(dt)) * (ex + 2.0 ** -22 * (np.abs(xhat * w) + np.abs(b)))
    assert (np.abs(f64(out) - want) <= bound + 1e-30).all()


def check_backward(got, r, w, dy, dres, dt, wdt):
    dx, dw, db = (None if t is None else f64(t) for t in got)
    _, mean, rstd = forward64(r, w, 0.0)
    xhat, T = (r - mean) * rstd, r.shape[0]
    g = dy * w
    s1, s2 = g.mean(-1, keepdims=True), (g * xhat).mean(-1, keepdims=True)
    core = rstd * (g - s1 - xhat * s2)
    ex = G * (rstd * np.abs(r).mean(-1, keepdims=True) + np.abs(xhat))
    e = rstd * (G * np.abs(g).mean(-1, keepdims=True) + ex * np.abs(s2) + np.abs(xhat) * (
        G * np.abs(g * xhat).mean(-1, keepdims=True) + (np.abs(g) * ex).mean(-1, keepdims=True)))
    e += 2.0 ** -15 * (np.abs(core) + rstd * (np.abs(s1) + np.abs(xhat * s2) + np.abs(g)))
    bx = rounded(dt, core + dres) + 1.01 * e + 2.0 ** -23 * np.abs(dres)
    assert (np.abs(dx - core - dres) <= bx + 1e-30).all()
    rows = (T + 700) * 2.0 ** -24
    want = (dy * xhat).sum(0)
    bw = rounded(wdt, want) + 1.01 * ((np.abs(dy) * ex).sum(0) + rows * np.abs(dy * xhat).sum(0))
    assert (np.abs(dw - want) <= bw + 1e-30).all()
    if db is not None:
        want = dy.sum(0)
        assert (np.abs(db - want) <= rounded(wdt, want) + 1.01 * rows * np.abs(dy).sum(0) + 1e-30).all()
    return bx


SIZES = [(1, 1), (1, 4096), (3, 3), (5, 8), (2, 100), (130, 513), (777, 1000), (9, 1001), (260, 2048), (33, 4096),
         (3, 5000), (1, 8192), (1500, 72)]


@pytest.mark.parametrize("T,H", SIZES + [(4, 16384), (5, 12001)])
@pytest.mark.parametrize("dt,wdt", [("bf16", "bf16"), ("f16", "f32"), ("f32", "f32"), ("f32", "bf16")])
def test_against_64_bits(T, H, dt, wdt, dev):
    if dt == "f32" and H > 8192:
        pytest.skip("rows of fp32 are up to 8192 wide")
    banner(f"layer_norm T={T} H={H} {dt} {wdt}")
    norm, x, res, dy, dres = make(T, H, DT[dt], DT[wdt], dev, seed=T + H)
    w, b = f64(norm.weight), f64(norm.bias)
    with torch.no_grad():
        out, r = norm.forward_add_residual(x, res)
        assert torch.equal(r, x + res)
        check_forward(out, f64(r), w, b, DT[dt])
        plain = norm(r)
        assert torch.equal(plain, out)
        inplace = r.clone()
        norm.forward_inplace(inplace)
        assert torch.equal(inplace, out)
    x.requires_grad_(), res.requires_grad_()
    got = norm.forward_add_residual(x, res)
    assert torch.equal(got[0], out) and torch.equal(got[1], r)
    dx, dr, dw, db = torch.autograd.grad(got, [x, res, norm.weight, norm.bias], [dy, dres],
                                         retain_graph=True)
    assert torch.equal(dx, dr)
    check_backward((dx, dw, db), f64(r), w, f64(dy), f64(dres), DT[dt], DT[wdt])
    again = torch.autograd.grad(got, [x, norm.weight, norm.bias], [dy, dres])
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dw, db)))


def test_gradient_against_differences(dev):
    banner("layer_norm differences")
    T, H = 6, 200
    norm, x, _, dy, _ = make(T, H, torch.float32, torch.float32, dev, seed=3)
    x.requires_grad_()
    dx, dw, db = torch.autograd.grad(norm(x), [x, norm.weight, norm.bias], dy)
    r, w, b, g = f64(x), f64(norm.weight), f64(norm.bias), f64(dy)
    bx = check_backward((dx, dw, db), r, w, g, np.zeros_like(r), torch.float32, torch.float32)
    rng = np.random.default_rng(0)

    def loss(r, w, b):
        return (forward64(r, w, b)[0] * g).sum()

    h = 1e-4
    for _ in range(4):
        d, dwd, dbd = rng.standard_normal(r.shape), rng.standard_normal(H), rng.standard_normal(H)
        # central differences: off by h^2 of a third derivative, under 50 |d|^3 |dy| here
        slack = 50 * h * h * np.linalg.norm(g) * np.linalg.norm(d, axis=-1).max() ** 3
        diff = (loss(r + h * d, w, b) - loss(r - h * d, w, b)) / (2 * h)
        assert abs((f64(dx) * d).sum() - diff) <= (bx * np.abs(d)).sum() + slack
        diff = (loss(r, w + h * dwd, b) - loss(r, w - h * dwd, b)) / (2 * h)  # linear
        assert abs((f64(dw) * dwd).sum() - diff) <= 1e-5 * (np.abs(dwd) * np.abs(g).sum(0)).sum() * 4
        diff = (loss(r, w, b + h * dbd) - loss(r, w, b - h * dbd)) / (2 * h)
        assert abs((f64(db) * dbd).sum() - diff) <= 1e-5 * (np.abs(dbd) * np.abs(g).sum(0)).sum()


@pytest.mark.parametrize("H", [40, 1000])
def test_which_gradients_are_asked_for(H, dev):
    banner(f"layer_norm partial gradients H={H}")
    norm, x, res, dy, dres = make(9, H, torch.bfloat16, torch.bfloat16, dev)
    x.requires_grad_(), res.requires_grad_()
    out, r = norm.forward_add_residual(x, res)
    both = torch.autograd.grad([out, r], [x, norm.weight, norm.bias], [dy, dres], retain_graph=True)
    # only the norm goes on, then only the sum
    assert torch.equal(torch.autograd.grad(out, res, dy, retain_graph=True)[0],
                       torch.autograd.grad([out, r], res, [dy, torch.zeros_like(dres)], retain_graph=True)[0])
    only = torch.autograd.grad(r, [x, res, norm.weight, norm.bias], dres, retain_graph=True)
    assert torch.equal(only[0], dres) and torch.equal(only[1], dres)
    assert not only[2].any() and not only[3].any()
    # each alone
    assert torch.equal(torch.autograd.grad([out, r], norm.weight, [dy, dres], retain_graph=True)[0], both[1])
    assert torch.equal(torch.autograd.grad([out, r], norm.bias, [dy, dres], retain_graph=True)[0], both[2])
    norm.requires_grad_(False)
    frozen = norm.forward_add_residual(x, res)
    assert torch.equal(torch.autograd.grad(frozen, x, [dy, dres])[0], both[0])
    # a bias of another type than the weight, and none
    norm.bias.data = norm.bias.data.float()
    norm.requires_grad_(True)
    db = torch.autograd.grad(norm.forward_add_residual(x, res)[0], norm.bias, dy)[0]
    assert db.dtype == torch.float32
    bare, *_ = make(9, H, torch.bfloat16, torch.bfloat16, dev, bias=False)
    out0 = bare(x.detach())
    check_forward(out0, f64(x), f64(bare.weight), 0.0, torch.bfloat16)
    grads = torch.autograd.grad(bare(x), [x, bare.weight], dy)
    check_backward((*grads, None), f64(x), f64(bare.weight), f64(dy), 0.0 * f64(dy), torch.bfloat16,
                   torch.bfloat16)


def test_strides_shapes_and_no_rows(dev):
    banner("layer_norm strides")
    norm, x, res, dy, _ = make(24, 96, torch.float16, torch.float32, dev)
    want = norm(x).detach()
    wide = torch.zeros(24, 200, dtype=torch.float16, device=dev)
    wide[:, 3:99] = x
    assert torch.equal(norm(wide[:, 3:99]), want)
    assert torch.equal(norm(x.reshape(2, 3, 4, 96)).reshape(24, 96), want)
    odd = torch.zeros(24 * 96 + 1, dtype=torch.float16, device=dev)[1:].view(24, 96)
    odd.copy_(x)  # starts on 2 bytes
    assert torch.equal(norm(odd), want)
    t = x.t().contiguous().t()
    with torch.no_grad():
        norm.forward_inplace(t)
    assert torch.equal(t, want)
    # a broadcast input gets the sum of its rows' gradients
    one = x[:1].clone().requires_grad_()
    g = torch.autograd.grad(norm(one.expand(24, 96)), one, dy)[0]
    full = x[:1].expand(24, 96).contiguous().requires_grad_()
    rows = torch.autograd.grad(norm(full), full, dy)[0]
    s = f64(rows).sum(0, keepdims=True)
    assert (np.abs(f64(g) - s) <= 24 * half(torch.float16) * np.abs(f64(rows)).sum(0)).all()
    empty = torch.empty(0, 96, dtype=torch.float16, device=dev, requires_grad=True)
    out, r = norm.forward_add_residual(empty, empty)
    grads = torch.autograd.grad([out, r], [empty, norm.weight, norm.bias], [out, r])
    assert grads[0].shape == (0, 96) and not grads[1].any() and not grads[2].any()


def test_infinities_stay_in_their_row(dev):
    banner("layer_norm infinities")
    norm, x, _, dy, _ = make(40, 264, torch.float32, torch.float32, dev)
    clean = norm(x)
    bad = x.clone()
    bad[7, 3], bad[11, 200] = float("inf"), float("nan")
    out = norm(bad)
    keep = [i for i in range(40) if i not in (7, 11)]
    assert torch.equal(out[keep], clean[keep]) and bool(torch.isnan(out[[7, 11]]).any(-1).all())


def test_a_constant_row_and_a_far_mean(dev):
    """No difference of large sums: rows around 1000 with a deviation of 1."""
    banner("layer_norm far mean")
    norm, x, *_ = make(16, 1024, torch.float32, torch.float32, dev)
    x = x + 1000.0
    x[3] = 1000.0
    out = norm(x).detach()
    check_forward(out, f64(x), f64(norm.weight), f64(norm.bias), torch.float32)
    assert torch.equal(out[3], norm.bias.detach())


def test_streams_and_graphs(dev):
    banner("layer_norm graph")
    norm, x, res, dy, dres = make(300, 640, torch.bfloat16, torch.bfloat16, dev)
    norm.requires_grad_(False)
    leaves = [x.clone().requires_grad_(), res.clone().requires_grad_()]
    w = norm.weight.detach().clone().requires_grad_()
    norm.weight = torch.nn.Parameter(w.detach())

    def step():
        out = norm.forward_add_residual(*leaves)
        return tuple(t.detach() for t in out) + torch.autograd.grad(out, leaves + [norm.weight], [dy, dres])

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
        g = torch.Generator(device=dev).manual_seed(100 + i)
        for t in leaves:
            t.data.copy_(torch.randn(t.shape, generator=g, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_before_an_expert_layer(dev):
    """FusedMoE.forward_with_norm takes a LayerNorm: the norm's call, then the layer's."""
    banner("layer_norm before FusedMoE")
    torch.manual_seed(5)
    E, K, H, I, T = 4, 2, 256, 128, 19
    moe = FusedMoE(E, K, H, I, dtype=torch.bfloat16).to(dev)
    with torch.no_grad():
        for p in moe.parameters():
            p.normal_(std=0.05)
    norm = LayerNorm(H, 1e-5).to(dev)
    with torch.no_grad():
        norm.weight.uniform_(0.5, 1.5)
        norm.bias.normal_()
    x, res = (torch.randn(T, H, device=dev).to(torch.bfloat16) for _ in range(2))
    out, new_res = moe.forward_with_norm(x, res, norm)
    with torch.no_grad():
        normed, want_res = norm.forward_add_residual(x, res)
        want = moe(normed)
    assert torch.equal(new_res, want_res) and torch.equal(out, want)
    assert not out.requires_grad and not new_res.requires_grad


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_before_an_expert_layer_in_any_shape(dt, dev):
    """Results have the input's shape, as behind an RMSNorm, and are those of the rows."""
    banner(f"layer_norm before FusedMoE, shapes, {dt}")
    torch.manual_seed(6)
    H = 256
    moe = FusedMoE(4, 2, H, 128, dtype=torch.bfloat16).to(dev)
    with torch.no_grad():
        for p in moe.parameters():
            p.normal_(std=0.05)
    norm = LayerNorm(H, EPS).to(dev)
    for shape in ((2, 5, H), (3, 1, H), (1, 1, H), (2, 2, 3, H), (H,), (0, H), (2, 0, H)):
        x, res = (torch.randn(shape, device=dev).to(DT[dt]) for _ in range(2))
        out, new_res = moe.forward_with_norm(x, res, norm)
        assert out.shape == x.shape and new_res.shape == x.shape
        assert out.dtype == x.dtype and new_res.dtype == res.dtype
        if x.numel():
            rows = moe.forward_with_norm(x.reshape(-1, H), res.reshape(-1, H), norm)
            assert torch.equal(out.reshape(-1, H), rows[0]) and torch.equal(new_res.reshape(-1, H), rows[1])
    x = torch.randn(2, 5, H, device=dev).to(DT[dt])
    out, new_res = moe.forward_with_norm(x, x.reshape(10, H), norm)  # the residual in rows
    assert out.shape == x.shape and new_res.shape == x.shape


def test_an_overwritten_input_is_noticed(dev):
    """forward_inplace overwrites what an earlier call keeps for its gradient."""
    banner("layer_norm in place behind a recorded call")
    norm, x, *_ = make(9, 256, torch.bfloat16, torch.bfloat16, dev)
    out = norm(x)  # keeps x for the weight's gradient
    norm.forward_inplace(x)
    assert torch.equal(x, out.detach())
    with pytest.raises(RuntimeError, match="inplace"):
        out.float().sum().backward()
    rms = RMSNorm(256, EPS).to(dev)
    out = norm(x)
    rms.forward_inplace(x)
    with pytest.raises(RuntimeError, match="inplace"):
        out.float().sum().backward()
    for n in (norm, rms):
        with torch.inference_mode():
            y = torch.randn(9, 256, device=dev).bfloat16()
            want = n(y)
            n.forward_inplace(y)
            assert torch.equal(y, want)
