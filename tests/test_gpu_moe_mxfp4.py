"""FusedMoE with routing by groups and 4-bit experts on the GPU: the operators run
together as a layer runs them, against 64 bits at every stage.

Bars: routing on the layer's own logits is exact in the ids (test_gpu_grouped_topk);
the experts' result is within what test_gpu_mx derives (2^-7 + 2^-8 in bf16,
2^-10.5 + 2^-11 in f16) of 64-bit arithmetic on the same routing, normed rows and
weights.
"""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

import _mx_ref as ref
from _helpers import banner
from reframework_amd import _capi
from reframework_amd.layers import RMSNorm
from reframework_amd.moe import FusedMoE, Mxfp4Experts, fused_experts, fused_experts_mxfp4

pytestmark = pytest.mark.gpu
REL = {torch.bfloat16: 2.0 ** -7 + 2.0 ** -8, torch.float16: 2.0 ** -10.5 + 2.0 ** -11}


def _layer(dev, dt=torch.bfloat16, E=16, K=3, H=256, I=160, seed=0, **kw):
    g = torch.Generator().manual_seed(seed)
    moe = FusedMoE(E, K, H, I, dtype=dt, **kw)
    for p in moe.parameters():
        p.data.copy_(torch.randn(p.shape, generator=g) * (0.05 if p.dim() > 1 else 0.1))
    return moe.to(dev)


GROUPS = dict(scoring="sigmoid", num_expert_groups=4, topk_groups=2, group_score="top2",
              expert_bias=True, routed_scale=2.5)


def _route64(moe, x):
    """The ids and weights of the layer's own rounded logits, in 64 bits."""
    logits = torch.empty((x.shape[0], moe.num_experts), device=x.device)
    _capi.router_logits(x, moe.gate.detach(), True, logits)
    return ref.grouped_topk(logits.cpu().numpy(), moe.top_k, moe.renormalize, moe.scoring,
                            None if moe.expert_bias is None else moe.expert_bias.detach().cpu().numpy(),
                            moe.num_expert_groups, moe.topk_groups, moe.group_score,
                            moe.routed_scale)


@pytest.mark.parametrize("T", [1, 7, 100, 300])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_grouped_layer_routes_and_sums(T, dt, dev):
    """16-bit experts: the routing is the new one, the sum the layer's own."""
    banner(f"FusedMoE grouped T={T} {dt}")
    moe = _layer(dev, dt, **GROUPS)
    x = torch.randn(T, 256, generator=torch.Generator().manual_seed(T)).to(dt).to(dev)
    w, ids = moe.route(x)
    rw, rids = _route64(moe, x)
    assert np.array_equal(ids.cpu().numpy(), rids)
    assert np.abs(ref.to64(w) - rw).max() <= 2.0 ** -20 * np.abs(rw).max()
    out = fused_experts(x, list(moe.experts_w1), list(moe.experts_w2), w, ids)
    assert torch.equal(moe(x), out)
    norm = RMSNorm(256, 1e-5).to(dev)
    res = torch.randn_like(x)
    got, new_res = moe.forward_with_norm(x, res, norm)
    normed, want_res = norm.forward_add_residual(x, res)
    assert torch.equal(new_res, want_res) and torch.equal(got, moe(normed))


@pytest.mark.parametrize("shared", [{}, {"n_shared_experts": 2}, {"shared_intermediate_size": 96}],
                         ids=["none", "folded", "apart"])
@pytest.mark.parametrize("kw", [{}, GROUPS], ids=["softmax", "groups"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 24, 260])
def test_quantised_layer(T, dt, kw, shared, dev):
    banner(f"FusedMoE 4-bit T={T} {dt} {list(kw)[:1]} {shared}")
    moe = _layer(dev, dt, **kw, **shared)
    banks = [Mxfp4Experts.quantize(list(a), list(b)) for a, b in
             ((moe.experts_w1, moe.experts_w2), (moe.shared_w1, moe.shared_w2)) if len(a)]
    w64 = [(ref.to64(b.dequantize("w1")), ref.to64(b.dequantize("w2"))) for b in banks]
    moe.quantize_experts()
    assert not len(moe.experts_w1) and not len(moe.shared_w1)
    x = torch.randn(T, 256, generator=torch.Generator().manual_seed(T + 1)).to(dt).to(dev)

    def want(rows):
        w, ids = moe.route(rows)
        x64 = ref.to64(rows)
        out = ref.experts(x64, *w64[0], ref.to64(w).astype(np.float32), ids.cpu().numpy())
        if len(w64) > 1:
            for e in range(w64[1][0].shape[0]):
                out += ref.experts(x64, w64[1][0][e:e + 1], w64[1][1][e:e + 1],
                                   np.ones((T, 1), np.float32), np.zeros((T, 1), np.int64))
        return out

    def rel(got, r):
        return np.linalg.norm(ref.to64(got) - r) / np.linalg.norm(r)

    assert rel(moe(x), want(x)) <= REL[dt]
    norm = RMSNorm(256, 1e-5).to(dev)
    res = torch.randn_like(x)
    got, new_res = moe.forward_with_norm(x, res, norm)
    normed, want_res = norm.forward_add_residual(x, res)
    assert torch.equal(new_res, want_res)
    assert rel(got, want(normed)) <= REL[dt]
    # the norm's 8-bit rows are what the layer makes of the normed ones
    assert torch.equal(got, moe(normed))


def test_state_dict_round_trip(dev):
    banner("FusedMoE 4-bit state dict")
    kw = dict(n_shared_experts=2, **GROUPS)
    moe = _layer(dev, **kw)
    moe.quantize_experts()
    sd = {k: v.clone() for k, v in moe.state_dict(prefix="l0").items()}
    assert "l0.gate.e_score_correction_bias" in sd and "l0.experts_mxfp4.w1" in sd
    assert not any(k.startswith("l0.experts.") for k in sd)
    other = _layer(dev, seed=5, **kw)
    other.load_state_dict(sd, prefix="l0")
    x = torch.randn(9, 256, device=dev).bfloat16()
    assert torch.equal(moe(x), other(x))
    other.load_state_dict(sd, prefix="l0")  # a quantised layer takes them again
    assert torch.equal(moe(x), other(x))
    plain = _layer(dev, seed=6, **kw)
    with pytest.raises(RuntimeError, match="4 bits already"):
        other.load_state_dict(plain.state_dict())
    apart = _layer(dev, shared_intermediate_size=96)
    apart.quantize_experts()
    part = {k: v for k, v in apart.state_dict().items() if not k.startswith("shared")}
    with pytest.raises(ValueError, match="only a part"):
        _layer(dev, shared_intermediate_size=96).load_state_dict(part)


def test_from_config_and_refusals(dev):
    banner("FusedMoE 4-bit refusals")
    cfg = SimpleNamespace(num_experts=16, num_experts_per_tok=3, hidden_size=256, moe_inter=160,
                          moe_activation="silu", moe_renormalize=True, dtype=torch.bfloat16,
                          scoring_func="sigmoid", n_group=4, topk_group=2, moe_expert_bias=True,
                          routed_scaling_factor=2.5)
    moe = FusedMoE.from_config(cfg)
    assert (moe.scoring, moe.num_expert_groups, moe.topk_groups, moe.group_score,
            moe.routed_scale) == ("sigmoid", 4, 2, "top2", 2.5) and moe.expert_bias is not None
    with pytest.raises(RuntimeError, match="GPU"):
        moe.quantize_experts()  # parameters on the CPU
    assert len(moe.experts_w1) == 16
    for bad in (dict(scoring="tanh"), dict(group_score="mean"), dict(num_expert_groups=3),
                dict(num_expert_groups=4, topk_groups=5)):
        with pytest.raises(ValueError):
            FusedMoE(16, 3, 256, 160, **bad)
    odd = _layer(dev, H=256, I=40)
    with pytest.raises(ValueError, match="whole blocks"):
        odd.quantize_experts()
    assert len(odd.experts_w1) == 16
    quant = _layer(dev)
    quant.quantize_experts()
    quant.quantize_experts()
    with pytest.raises(RuntimeError, match="4-bit"):
        quant.build_offload_cache(dev, 4)
    off = _layer(dev)
    off.build_offload_cache(dev, 4)
    with pytest.raises(RuntimeError, match="offloaded"):
        off.quantize_experts()
    ent = _layer(dev, **GROUPS)
    ent.entropy_adaptive_k = True
    with pytest.raises(ValueError, match="entropy"):
        ent(torch.zeros(2, 256, device=dev, dtype=torch.bfloat16))


@pytest.mark.parametrize("shared", [0, 2])
def test_two_captured_layers_calls_replayed_on_two_streams(shared, dev):
    banner(f"FusedMoE 4-bit graphs shared={shared}")
    T = 12
    moe = _layer(dev, n_shared_experts=shared, **GROUPS)
    moe.quantize_experts()
    norm = RMSNorm(256, 1e-5).to(dev)
    xs = [torch.randn(T, 256, device=dev).bfloat16() for _ in range(4)]
    rs = [torch.randn(T, 256, device=dev).bfloat16() for _ in range(4)]
    want = [moe.forward_with_norm(x, r, norm) for x, r in zip(xs, rs)]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gx, gr = torch.zeros_like(xs[0]), torch.zeros_like(rs[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = moe.forward_with_norm(gx, gr, norm)
        graphs.append((g, gx, gr, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(4):
        for (g, gx, gr, _), s, j in zip(graphs, streams, (k, 3 - k)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                gx.copy_(xs[j])
                gr.copy_(rs[j])
                g.replay()
        eager = moe.forward_with_norm(xs[k], rs[k], norm)
        torch.cuda.synchronize()
        assert torch.equal(eager[0], want[k][0])
        for (_, _, _, out), j in zip(graphs, (k, 3 - k)):
            assert torch.equal(out[0], want[j][0]) and torch.equal(out[1], want[j][1])


def test_experts_alone_as_a_dense_layer(dev):
    """One expert and weights of 1: a 4-bit feed-forward layer."""
    banner("fused_experts_mxfp4 as a dense layer")
    g = torch.Generator().manual_seed(3)
    H, I, T = 384, 736, 5
    w1, w2 = (torch.randn(s, generator=g) * 0.05 for s in ((2 * I, H), (H, I)))
    ex = Mxfp4Experts.quantize([w1.to(dev)], [w2.to(dev)])
    x = torch.randn(T, H, generator=g).bfloat16()
    one = torch.ones((T, 1))
    want = ref.experts(ref.to64(x), ref.to64(ex.dequantize("w1")), ref.to64(ex.dequantize("w2")),
                       one.numpy(), np.zeros((T, 1), np.int64))
    got = fused_experts_mxfp4(x.to(dev), ex, one.to(dev), torch.zeros((T, 1), dtype=torch.int64, device=dev))
    assert np.linalg.norm(ref.to64(got) - want) / np.linalg.norm(want) <= REL[torch.bfloat16]
