"""The bias for the choice of experts on the CPU: which configs give a layer one, and that
neither a checkpoint's bias nor a layer's is dropped without a word."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch
from safetensors.torch import save_file

from reframework_amd.checkpoint import SafetensorsIndex, load_moe_layer, load_moe_layer_offload
from reframework_amd.moe import FusedMoE

E, K, H, I = 8, 2, 16, 8


def _config(**kw):
    return SimpleNamespace(num_experts=E, num_experts_per_tok=K, hidden_size=H, moe_inter=I,
                           moe_activation="silu", moe_renormalize=True, dtype=torch.float32, **kw)


GROUPS = dict(scoring_func="sigmoid", n_group=4, topk_group=2, routed_scaling_factor=2.5)


@pytest.mark.parametrize("kw,bias,groups,score", [
    (dict(topk_method="noaux_tc", **GROUPS), True, (4, 2), "top2"),
    (dict(topk_method="noaux_tc", n_group=1, topk_group=1, scoring_func="sigmoid"), True, (1, 1), "top2"),
    (dict(topk_method="group_limited_greedy", **GROUPS), False, (4, 2), "max"),
    (dict(topk_method="greedy", **GROUPS), False, (1, 1), "max"),
    (dict(topk_method=None, **GROUPS), False, (4, 2), "max"),
    (dict(GROUPS), False, (4, 2), "max"),
    ({}, False, (1, 1), "max"),
    # this framework's own fields go first
    (dict(moe_expert_bias=True, **GROUPS), True, (4, 2), "top2"),
    (dict(topk_method="noaux_tc", moe_expert_bias=False, **GROUPS), False, (4, 2), "max"),
    (dict(topk_method="noaux_tc", moe_group_score="max", **GROUPS), True, (4, 2), "max"),
    (dict(topk_method="group_limited_greedy", moe_expert_bias=True, **GROUPS), True, (4, 2), "max"),
])
def test_what_a_config_says(kw, bias, groups, score):
    moe = FusedMoE.from_config(_config(**kw))
    assert (moe.expert_bias is not None) == bias
    assert (moe.num_expert_groups, moe.topk_groups) == groups and moe.group_score == score
    assert moe.scoring == kw.get("scoring_func", "softmax")
    assert moe.routed_scale == kw.get("routed_scaling_factor", 1.0)


def test_unknown_method():
    with pytest.raises(ValueError, match="topk_method 'other'"):
        FusedMoE.from_config(_config(topk_method="other"))


def _state(bias):
    g = torch.Generator().manual_seed(1)
    moe = FusedMoE(E, K, H, I, dtype=torch.float32, scoring="sigmoid", expert_bias=bias)
    return {k: torch.randn(v.shape, generator=g) for k, v in moe.state_dict(prefix="m").items()}


def _layer(bias):
    moe = FusedMoE(E, K, H, I, dtype=torch.float32, scoring="sigmoid", expert_bias=bias)
    for p in moe.parameters():
        p.data.fill_(0.5)
    return moe


def _untouched(moe):
    return all(bool((p == 0.5).all()) for p in moe.parameters())


@pytest.mark.parametrize("strict", [True, False])
def test_a_bias_the_layer_has_no_place_for(strict):
    moe = _layer(False)
    with pytest.raises(ValueError, match="without a bias"):
        moe.load_state_dict(_state(True), prefix="m", strict=strict)
    assert _untouched(moe)
    moe.load_state_dict(_state(False), prefix="m", strict=strict)
    assert torch.equal(moe.gate, _state(False)["m.gate.weight"])


def test_a_router_without_the_bias_of_the_layer():
    moe, sd = _layer(True), _state(False)
    with pytest.raises(ValueError, match="m.gate.weight without m.gate.e_score_correction_bias"):
        moe.load_state_dict(sd, prefix="m")
    assert _untouched(moe)
    moe.load_state_dict(sd, prefix="m", strict=False)  # keeps its own
    assert torch.equal(moe.gate, sd["m.gate.weight"]) and bool((moe.expert_bias == 0.5).all())
    moe = _layer(True)
    moe.load_state_dict({k: v for k, v in sd.items() if ".experts." in k}, prefix="m")  # no router
    assert bool((moe.gate == 0.5).all())
    moe.load_state_dict(_state(True), prefix="m")
    assert torch.equal(moe.expert_bias, _state(True)["m.gate.e_score_correction_bias"])


def _index(tmp_path, bias):
    save_file(_state(bias), str(tmp_path / "l.safetensors"))
    return SafetensorsIndex(tmp_path)


@pytest.mark.parametrize("offload", [False, True])
def test_checkpoint_with_a_bias(tmp_path, offload):
    index, moe = _index(tmp_path, True), _layer(False)
    with pytest.raises(ValueError, match="e_score_correction_bias"):
        if offload:
            load_moe_layer_offload(index, moe, "m", torch.device("cpu"), 2)
        else:
            load_moe_layer(index, moe, "m")
    assert _untouched(moe)
    moe = _layer(True)
    rep = load_moe_layer(index, moe, "m")
    assert not rep.missing and not rep.unexpected
    assert torch.equal(moe.expert_bias, _state(True)["m.gate.e_score_correction_bias"])


def test_checkpoint_without_the_bias_of_the_layer_reports_it(tmp_path):
    moe = _layer(True)
    rep = load_moe_layer(_index(tmp_path, False), moe, "m")
    assert rep.missing == ["m.gate.e_score_correction_bias"]
