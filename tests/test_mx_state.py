"""State dicts and checkpoints of layers with 4-bit experts, on the CPU (their bytes are
copied, nothing is computed): what does not fit is refused and leaves the layer as it was."""

from __future__ import annotations

import pytest
import torch
from safetensors.torch import save_file

from reframework_amd.checkpoint import SafetensorsIndex, load_moe_layer, load_moe_layer_offload
from reframework_amd.moe import FusedMoE, Mxfp4Experts

E, K, H, I = 4, 2, 64, 64
BIAS = dict(scoring="sigmoid", expert_bias=True)
APART = dict(shared_intermediate_size=96)
BANK_KEYS = ("w1", "w1_scales", "w2", "w2_scales")


def _layer(seed=0, **kw):
    g = torch.Generator().manual_seed(seed)
    moe = FusedMoE(E, K, H, I, dtype=torch.float32, **kw)
    for p in moe.parameters():
        p.data.copy_(torch.randn(p.shape, generator=g))
    return moe


def _bytes(seed, prefix="", shared=0, apart=False, bias=False):
    """State dict of a quantised layer with random contents."""
    g = torch.Generator().manual_seed(seed)
    head = prefix + "." if prefix else ""
    sd = {head + "gate.weight": torch.randn(E, H, generator=g)}
    if bias:
        sd[head + "gate.e_score_correction_bias"] = torch.randn(E, generator=g)
    banks = [("experts_mxfp4", Mxfp4Experts(E + shared, H, I))]
    if apart:
        banks.append(("shared_mxfp4", Mxfp4Experts(1, H, APART["shared_intermediate_size"])))
    for name, bank in banks:
        for key, buf in bank.named_buffers():
            sd[f"{head}{name}.{key}"] = torch.randint(0, 255, buf.shape, generator=g, dtype=torch.uint8)
    return sd


def _holds(moe, sd, prefix=""):
    mine = moe.state_dict(prefix=prefix)
    return set(mine) == set(sd) and all(torch.equal(mine[k], v) for k, v in sd.items())


def _snapshot(moe):
    return {k: v.detach().clone() for k, v in moe.state_dict().items()}


def _quantised(seed, **kw):
    moe = _layer(seed, **{k: v for k, v in kw.items() if k in ("n_shared_experts", *BIAS, *APART)})
    sd = _bytes(seed, shared=kw.get("n_shared_experts", 0), apart="shared_intermediate_size" in kw,
                bias="expert_bias" in kw)
    moe.load_state_dict(sd)
    assert _holds(moe, sd)
    return moe


@pytest.mark.parametrize("kw", [{}, BIAS, {"n_shared_experts": 2}, APART],
                         ids=["plain", "bias", "folded", "apart"])
def test_whole_state_dicts_load(kw):
    moe = _quantised(1, **kw)
    assert not len(moe.experts_w1) and not len(moe.shared_w1)
    again = _bytes(2, shared=kw.get("n_shared_experts", 0), apart=kw is APART, bias=kw is BIAS)
    moe.load_state_dict(again)  # a quantised layer takes other experts
    assert _holds(moe, again)


@pytest.mark.parametrize("missing", BANK_KEYS)
@pytest.mark.parametrize("quantised", [False, True])
def test_a_bank_without_one_of_its_tensors_is_refused(quantised, missing):
    moe = _quantised(3, **BIAS) if quantised else _layer(3, **BIAS)
    before = _snapshot(moe)
    sd = _bytes(4, bias=True)
    del sd["experts_mxfp4." + missing]
    with pytest.raises(ValueError, match="without experts_mxfp4." + missing + "$"):
        moe.load_state_dict(sd)
    assert _holds(moe, before)
    with pytest.raises(ValueError, match="without"):  # one tensor at a time
        moe.load_state_dict({"experts_mxfp4.w1": _bytes(4)["experts_mxfp4.w1"]})
    assert _holds(moe, before)


@pytest.mark.parametrize("gone", ["experts_mxfp4", "shared_mxfp4"])
@pytest.mark.parametrize("quantised", [False, True])
def test_one_of_two_banks_is_refused(quantised, gone):
    moe = _quantised(5, **APART) if quantised else _layer(5, **APART)
    before = _snapshot(moe)
    sd = {k: v for k, v in _bytes(6, apart=True).items() if not k.startswith(gone)}
    with pytest.raises(ValueError, match="only a part"):
        moe.load_state_dict(sd)
    assert _holds(moe, before)


@pytest.mark.parametrize("quantised", [False, True])
def test_a_bank_the_layer_has_no_place_for_is_refused(quantised):
    moe = _quantised(7) if quantised else _layer(7)
    before = _snapshot(moe)
    with pytest.raises(ValueError, match="no such experts"):
        moe.load_state_dict(_bytes(8, apart=True))
    assert _holds(moe, before)


@pytest.mark.parametrize("quantised", [False, True])
def test_a_tensor_of_another_shape_is_refused_before_any_copy(quantised):
    moe = _quantised(9, **APART) if quantised else _layer(9, **APART)
    before = _snapshot(moe)
    sd = _bytes(10, apart=True)
    sd["shared_mxfp4.w2_scales"] = sd["shared_mxfp4.w2_scales"][:, :-4]
    with pytest.raises(ValueError, match="does not match"):
        moe.load_state_dict(sd)
    assert _holds(moe, before)


def _checkpoint(tmp_path, sd):
    save_file(sd, str(tmp_path / "layer.safetensors"))
    return SafetensorsIndex(tmp_path)


@pytest.mark.parametrize("kw", [{}, BIAS, {"n_shared_experts": 2}, APART],
                         ids=["plain", "bias", "folded", "apart"])
@pytest.mark.parametrize("quantised", [False, True])
def test_checkpoint_of_a_quantised_layer(tmp_path, quantised, kw):
    p = "model.layers.3.mlp"
    sd = _bytes(11, p, shared=kw.get("n_shared_experts", 0), apart=kw is APART, bias=kw is BIAS)
    index = _checkpoint(tmp_path, sd)
    moe = _quantised(12, **kw) if quantised else _layer(12, **kw)
    rep = load_moe_layer(index, moe, p)
    assert sorted(rep.loaded) == sorted(sd) and not rep.missing and not rep.unexpected
    assert _holds(moe, sd, p)


def test_checkpoint_saved_from_a_layer_loads_into_another(tmp_path):
    moe = _quantised(13, **BIAS)
    index = _checkpoint(tmp_path, {k: v.detach().contiguous()
                                   for k, v in moe.state_dict(prefix="m").items()})
    other = _layer(14, **BIAS)
    load_moe_layer(index, other, "m")
    assert _holds(other, moe.state_dict())


@pytest.mark.parametrize("quantised", [False, True])
def test_checkpoint_without_a_tensor_of_a_bank(tmp_path, quantised):
    sd = _bytes(15, "m")
    del sd["m.experts_mxfp4.w1_scales"]
    moe = _quantised(16) if quantised else _layer(16)
    before = _snapshot(moe)
    with pytest.raises(ValueError, match="without m.experts_mxfp4.w1_scales"):
        load_moe_layer(_checkpoint(tmp_path, sd), moe, "m")
    assert _holds(moe, before)


def test_checkpoint_of_16_bit_experts_leaves_a_quantised_layers_experts_and_says_so(tmp_path):
    plain = _layer(17)
    index = _checkpoint(tmp_path, {k: v.detach().contiguous()
                                   for k, v in plain.state_dict(prefix="m").items()})
    moe = _quantised(18)
    before = _snapshot(moe)
    rep = load_moe_layer(index, moe, "m")
    assert rep.loaded == ["m.gate.weight"] and len(rep.unexpected) == 3 * E
    assert sorted(rep.missing) == sorted(f"m.experts_mxfp4.{k}" for k in BANK_KEYS)
    before["gate.weight"] = plain.gate.detach()
    assert _holds(moe, before)


def test_offload_of_4_bit_experts_is_refused(tmp_path):
    index = _checkpoint(tmp_path, _bytes(19, "m"))
    for moe in (_layer(20), _quantised(20)):
        before = _snapshot(moe)
        with pytest.raises(ValueError, match="not offloaded"):
            load_moe_layer_offload(index, moe, "m", torch.device("cpu"), 2)
        assert _holds(moe, before)
