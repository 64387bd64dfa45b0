"""GPU routing by groups against 64-bit arithmetic.

Bars: the ids are those of exact arithmetic, ties to the lower. A weight is a score
(exp within 2 units of 2^-23, two roundings of 2^-24, for softmax a sum of positive
terms of the same errors) over a sum of scores: at most 2^-20 relative in all.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import _mx_ref as ref
from _helpers import banner
from reframework_amd import _capi
from reframework_amd.moe import grouped_topk, torch_fused_topk

pytestmark = pytest.mark.gpu
TOL = 2.0 ** -20


def _check(logits, K, dev, bias=None, **kw):
    w, ids = grouped_topk(torch.from_numpy(logits).to(dev), K,
                          bias=None if bias is None else torch.from_numpy(bias).to(dev), **kw)
    rw, rids = ref.grouped_topk(logits, K, bias=bias, **kw)
    assert w.dtype == torch.float32 and ids.dtype == torch.int64
    assert np.array_equal(ids.cpu().numpy(), rids)
    got = ref.to64(w)
    assert np.array_equal(np.isnan(got), np.isnan(rw))
    fin = ~np.isnan(rw)
    assert np.all(np.abs(got - rw)[fin] <= TOL * np.abs(rw)[fin] + 1e-30)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("T,E,K,G,KG,score", [
    (1, 1, 1, 1, 1, "max"), (5, 8, 2, 1, 1, "max"), (33, 64, 6, 8, 3, "max"),
    (19, 160, 6, 8, 3, "max"), (130, 256, 8, 8, 4, "top2"), (7, 60, 4, 12, 5, "top2"),
    (9, 96, 12, 3, 2, "top2"), (4, 256, 64, 2, 1, "max"), (6, 64, 3, 64, 5, "top2"),
    (3, 256, 5, 64, 2, "max"), (11, 255, 9, 17, 2, "top2"), (8, 34, 2, 17, 1, "top2"),
    (5, 64, 64, 1, 1, "max"), (8195, 256, 8, 8, 4, "top2"), (8193, 8, 2, 1, 1, "max"),
    (8194, 64, 6, 1, 1, "max"), (8192, 160, 6, 8, 3, "max"), (8197, 96, 8, 16, 5, "top2"),
    (8196, 60, 4, 12, 5, "top2"), (8192, 255, 7, 5, 2, "top2"), (8192, 64, 1, 2, 1, "max"),
    (8192, 64, 9, 4, 2, "max"), (8192, 255, 3, 17, 2, "top2"), (8192, 4, 4, 1, 1, "max"),
])
def test_matches_64_bit(T, E, K, G, KG, score, with_bias, scoring, dev):
    banner(f"grouped_topk T={T} E={E} K={K} G={G}/{KG} {score} {scoring} bias={with_bias}")
    rng = np.random.default_rng(E * 7 + T)
    logits = (rng.normal(size=(T, E)) * 1.5).astype(np.float32)
    bias = (rng.normal(size=E) * 0.1).astype(np.float32) if with_bias else None
    for renorm, scale in ((True, 1.0), (False, 2.5)):
        _check(logits, K, dev, bias=bias, renormalize=renorm, scoring=scoring, num_groups=G,
               topk_groups=KG, group_score=score, scale=scale)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("G,KG,score", [(1, 1, "max"), (8, 3, "max"), (8, 3, "top2")])
@pytest.mark.parametrize("T", [200, 8194])
def test_ties_and_near_ties(T, G, KG, score, scoring, dev):
    """Rounded logits (equal ones are common), a bias of few distinct values, and
    choices whose distance is below a step of 32 bits."""
    banner(f"grouped_topk ties T={T} {scoring} G={G} {score}")
    rng = np.random.default_rng(11)
    E = 64
    logits = np.round(rng.normal(size=(T, E)) * 4).astype(np.float32) / 4
    for bias in (None, np.zeros(E, np.float32), (rng.integers(0, 3, E) / 8).astype(np.float32)):
        _check(logits, 6, dev, bias=bias, scoring=scoring, num_groups=G, topk_groups=KG,
               group_score=score)
    # distances of some 1e-9: every choice is left to 64 bits
    close = (1.0 + rng.integers(0, 40, (T, E)) * 2.0 ** -23).astype(np.float32)
    _check(close, 6, dev, bias=np.full(E, 0.25, np.float32), scoring=scoring, num_groups=G,
           topk_groups=KG, group_score=score)
    # a bias that outweighs the scores: their bits are below its last one
    _check(logits, 6, dev, bias=np.full(E, 3.0e4, np.float32), scoring=scoring, num_groups=G,
           topk_groups=KG, group_score=score)
    # logits whose last bits decide, and so do equal ones
    low = (1.0 + rng.integers(0, 6, (T, E)) * 2.0 ** -23).astype(np.float32) * np.float32(-3)
    _check(low, 6, dev, scoring=scoring, num_groups=G, topk_groups=KG, group_score=score)
    # saturated scores
    _check((logits * 30).astype(np.float32), 6, dev, bias=np.zeros(E, np.float32),
           scoring="sigmoid", num_groups=G, topk_groups=KG, group_score=score)


@pytest.mark.parametrize("copies", [1, 700])
def test_nan_and_infinities_keep_ids_in_range(copies, dev):
    banner(f"grouped_topk NaN / infinities x {copies}")
    rng = np.random.default_rng(3)
    E, K = 32, 8
    logits = rng.normal(size=(12, E)).astype(np.float32)
    logits[0, :] = np.nan
    logits[1, 5] = np.nan
    logits[2, 3:9] = -np.inf
    logits[3, :] = -np.inf
    logits[4, 7] = np.inf
    logits[5, 8:] = np.nan
    logits[6, 8:] = np.finfo(np.float32).min
    logits[7, ::2] = -np.inf
    logits = np.tile(logits, (copies, 1))
    bias = (rng.normal(size=E) * 0.1).astype(np.float32)
    for b in (None, bias):
        for scoring in ("sigmoid", "softmax"):
            for G, KG, score in ((1, 1, "max"), (4, 2, "max"), (4, 2, "top2")):
                w, ids = grouped_topk(torch.from_numpy(logits).to(dev), K, scoring=scoring,
                                      bias=None if b is None else torch.from_numpy(b).to(dev),
                                      num_groups=G, topk_groups=KG, group_score=score)
                got = ids.cpu().numpy()
                assert got.min() >= 0 and got.max() < E
                assert all(len(set(r)) == K for r in got.tolist())
        rows = [r for r in range(len(logits)) if r % 12 in (1, 2, 6, 7, 8, 9, 10, 11)]
        rows = rows if copies == 1 else (rows * 2)[:8200]
        _check(logits[rows], K, dev, bias=b, scoring="sigmoid", num_groups=4, topk_groups=2)


def test_strides_types_and_empty(dev):
    banner("grouped_topk layouts")
    g = torch.Generator().manual_seed(0)
    big = torch.randn(3, 5, 128, generator=g)
    w, ids = grouped_topk(big.to(dev)[:, :, ::2], 4, num_groups=4, topk_groups=2)
    rw, rids = ref.grouped_topk(big[:, :, ::2].reshape(15, 64).numpy(), 4, num_groups=4,
                                topk_groups=2)
    assert ids.shape == (3, 5, 4) and np.array_equal(ids.cpu().numpy().reshape(15, 4), rids)
    # 16-bit logits are widened exactly
    h = torch.randn(9, 64, generator=g).bfloat16()
    w, ids = grouped_topk(h.to(dev), 4, scoring="sigmoid", num_groups=4, topk_groups=2)
    assert np.array_equal(ids.cpu().numpy(),
                          ref.grouped_topk(h.float().numpy(), 4, scoring="sigmoid", num_groups=4,
                                           topk_groups=2)[1])
    w, ids = grouped_topk(torch.empty((0, 64), device=dev), 4)
    assert w.shape == (0, 4) and ids.shape == (0, 4)
    # columns past K, and int32 ids
    lg = torch.randn(10, 64, generator=g).to(dev)
    wl = torch.full((10, 7), -1.0, device=dev)
    il = torch.full((10, 7), -5, dtype=torch.int32, device=dev)
    _capi.grouped_topk(lg, None, 4, 1, 8, 3, 0, True, 1.0, wl, il)
    w, ids = grouped_topk(lg, 4, scoring="sigmoid", num_groups=8, topk_groups=3)
    assert torch.equal(wl[:, :4], w) and torch.equal(il[:, :4].long(), ids)
    assert bool((wl[:, 4:] == -1).all()) and bool((il[:, 4:] == -5).all())


def test_plain_softmax_agrees_with_torch_fused_topk(dev):
    banner("grouped_topk == torch_fused_topk")
    lg = torch.randn(65, 64, generator=torch.Generator().manual_seed(1)).to(dev)
    w, ids = grouped_topk(lg, 6, renormalize=False)
    w2, ids2 = torch_fused_topk(lg, 6, False)
    assert torch.equal(ids, ids2)
    assert float((w - w2).abs().max()) <= 2 * TOL


@pytest.mark.parametrize("T,E", [(1, 8), (255, 160), (300, 8), (300, 24), (515, 256), (257, 64)])
@pytest.mark.parametrize("dt,H", [(torch.bfloat16, 512), (torch.float16, 264), (torch.float32, 256)])
def test_router_logits(T, E, dt, H, dev):
    """fp32 sums of H products: H * 2^-24 of their absolute sum bounds any order."""
    banner(f"router_logits T={T} E={E} H={H} {dt}")
    g = torch.Generator().manual_seed(T + E)
    x, gate = torch.randn(T, H, generator=g).to(dt), (torch.randn(E, H, generator=g) * 0.1).to(dt)
    out = torch.full((T, E), float("nan"), device=dev)
    _capi.router_logits(x.to(dev), gate.to(dev), False, out)
    r = ref.to64(x) @ ref.to64(gate).T
    bound = np.abs(ref.to64(x)) @ np.abs(ref.to64(gate)).T * H * 2.0 ** -24
    assert np.all(np.abs(ref.to64(out) - r) <= bound)
    _capi.router_logits(x.to(dev), gate.to(dev), True, out)
    rnd = out.to(dt).float()
    assert torch.equal(rnd, out)


@pytest.mark.parametrize("T", [37, 8211])
def test_starts_off_16_bytes_and_two_streams(T, dev):
    """Logits, bias and results that start on 4 bytes, in two calls at once."""
    banner(f"grouped_topk alignment T={T}")
    g = torch.Generator().manual_seed(T)
    E, K = 64, 6
    kw = dict(scoring="sigmoid", num_groups=8, topk_groups=3, group_score="top2")
    flat, bias = torch.randn(T * E + 1, generator=g).to(dev), (torch.randn(E + 1, generator=g) * 0.1).to(dev)
    pairs = [(flat[1:].view(T, E), bias[1:]), (flat[:-1].view(T, E), bias[:-1])]
    want = [ref.grouped_topk(l.cpu().numpy(), K, bias=b.cpu().numpy(), **kw) for l, b in pairs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, (l, b) in zip(streams, pairs):
            with torch.cuda.stream(s):
                got.append(grouped_topk(l, K, bias=b, **kw))
        torch.cuda.synchronize()
        for (w, ids), (rw, rids) in zip(got, want):
            assert np.array_equal(ids.cpu().numpy(), rids)
            assert np.all(np.abs(ref.to64(w) - rw) <= TOL * np.abs(rw) + 1e-30)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("b", [100.0, 1.0e4, 1.0e6])
@pytest.mark.parametrize("T", [6000, 9000])
def test_groups_whose_best_two_cancel(T, b, scoring, dev):
    """One expert of each group at +b, the others at -b: the sum of a group's best two
    keeps nothing of b, but its 32-bit terms are rounded to the bits of b."""
    banner(f"grouped_topk cancelling biases T={T} b={b} {scoring}")
    rng = np.random.default_rng(17)
    E, G = 64, 8
    bias = np.full(E, -b, np.float32)
    bias[np.arange(G) * (E // G) + rng.integers(0, E // G, G)] = b
    for _ in range(4):
        logits = (rng.normal(size=(T, E)) * 1.5).astype(np.float32)
        _check(logits, 6, dev, bias=bias, scoring=scoring, num_groups=G, topk_groups=4,
               group_score="top2")


@pytest.mark.parametrize("T", [500, 9000])
def test_a_group_of_nans_is_below_one_that_is_shut_out(T, dev):
    """A group of NaN, one of a single expert beside some with a bias of -inf (its best two
    make -inf), two of many: with one group left out it is the NaN one, and the single
    expert is the first choice."""
    banner(f"grouped_topk NaN and -inf groups T={T}")
    rng = np.random.default_rng(29)
    logits = rng.normal(size=(T, 64)).astype(np.float32)
    logits[:, :16] = np.nan
    bias = np.zeros(64, np.float32)
    bias[16:32] = -np.inf
    bias[21] = 2.0
    for score in ("max", "top2"):
        for K in (4, 8):
            _check(logits, K, dev, bias=bias, scoring="sigmoid", num_groups=4, topk_groups=3,
                   group_score=score)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("value", [-np.inf, np.finfo(np.float32).min])
@pytest.mark.parametrize("score", ["max", "top2"])
@pytest.mark.parametrize("T", [500, 9000])
def test_biases_that_shut_experts_out(T, score, value, scoring, dev):
    """Most experts shut out by the bias, so that groups keep one expert or none; a NaN
    logit ranks below them still."""
    banner(f"grouped_topk shut out T={T} {value} {score} {scoring}")
    rng = np.random.default_rng(23)
    E, G = 64, 8
    logits = (rng.normal(size=(T, E)) * 1.5).astype(np.float32)
    if scoring == "sigmoid":  # a softmax with a NaN is NaN throughout
        logits[::3, 8:16] = np.nan
        logits[1::3, 32:40:2] = np.nan
    bias = (rng.normal(size=E) * 0.1).astype(np.float32)
    bias[rng.random(E) < 0.7] = value
    bias[:8] = bias[24:32] = value
    for KG in (2, 5, 7):
        _check(logits, 6, dev, bias=bias, scoring=scoring, num_groups=G, topk_groups=KG,
               group_score=score)


@pytest.mark.parametrize("E,G,KG", [(100, 1, 1), (111, 1, 1), (128, 8, 3), (200, 5, 2), (256, 1, 1),
                                    (255, 17, 9)])
@pytest.mark.parametrize("T", [500, 7000])
def test_equal_choices_of_many_experts(T, E, G, KG, dev):
    """Experts of equal logits and equal biases tie wherever in a lane's list they are."""
    banner(f"grouped_topk equal choices T={T} E={E} G={G}")
    rng = np.random.default_rng(E)
    logits = (np.round(rng.normal(size=(T, E)) * 6) / 4).astype(np.float32)
    few = np.array([-0.3, 0.1, 0.25], np.float32)[rng.integers(0, 3, E)]
    for bias in (np.full(E, 0.25, np.float32), np.full(E, -0.3, np.float32), few):
        for scoring in ("softmax", "sigmoid"):
            _check(logits, 6, dev, bias=bias, scoring=scoring, num_groups=G, topk_groups=KG)
