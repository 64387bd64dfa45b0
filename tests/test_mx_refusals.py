"""Refusals of the 8-bit rows, the 4-bit experts and the routing by groups, on the CPU
(nothing is launched): the C entry points by status, the Python ones by exception."""

from __future__ import annotations

import ctypes

import pytest
import torch

from reframework_amd import _capi
from reframework_amd.layers import RMSNorm
from reframework_amd.moe import (Mxfp4Experts, Mxfp8Rows, fused_experts_mxfp4, grouped_topk,
                                 quantize_mxfp8)
from reframework_amd.mx import padded

P = 4096  # an aligned address that no refused call reads


def _rc(name, *args):
    lib = _capi.lib()
    rc = getattr(lib, name)(*args)
    return rc, lib.moe355_last_error().decode()


@pytest.mark.parametrize("args,code,msg", [
    ((P, -1, 64, 1, P, P, None), -1, "T=-1"),
    ((P, 4, 48, 1, P, P, None), -2, "multiple of 32"),
    ((P, 4, 0, 1, P, P, None), -2, "multiple of 32"),
    ((P, 4, 64, 9, P, P, None), -1, "dtype"),
    ((None, 4, 64, 1, P, P, None), -1, "NULL"),
    ((P, 4, 64, 1, P, None, None), -1, "NULL"),
    ((P + 2, 4, 64, 1, P, P, None), -1, "aligned"),
    ((P, 4, 64, 1, P + 8, P, None), -1, "aligned"),
    ((None, 0, 64, 1, None, None, None), 0, None),
])
def test_quantize(args, code, msg):
    rc, err = _rc("moe355_mx_quantize", *args)
    assert rc == code and (msg is None or msg in err)


@pytest.mark.parametrize("over,code,msg", [
    ({"H": 72}, -2, "8-bit rows"), ({"H": 16384 + 32}, -2, "H <= 16384"), ({"H": 0}, -1, "H=0"),
    ({"dtype": 5}, -1, "dtype"), ({"wdtype": 5}, -1, "dtype"), ({"eps": -1.0}, -1, "eps"),
    ({"eps": float("nan")}, -1, "eps"), ({"codes": None}, -1, "NULL"), ({"scales": None}, -1, "NULL"),
    ({"residual_out": None}, -1, "residual_out"), ({"weight": P + 4}, -1, "weight"),
    ({"codes": P + 8}, -1, "aligned"), ({"T": -1}, -1, "T=-1"), ({"T": 0, "x": None}, 0, None),
])
def test_norm(over, code, msg):
    a = dict(x=P, residual=P, residual_out=P, weight=P, bias=None, wdtype=0, eps=1e-5, T=4, H=64,
             dtype=1, out=P, codes=P, scales=P)
    a.update(over)
    rc, err = _rc("moe355_add_rmsnorm_mxfp8", a["x"], a["residual"], a["residual_out"], a["weight"],
                  a["bias"], a["wdtype"], a["eps"], a["T"], a["H"], a["dtype"], a["out"],
                  a["codes"], a["scales"], None)
    assert rc == code and (msg is None or msg in err)


@pytest.mark.parametrize("over,code,msg", [
    ({"T": -1}, -1, "T=-1"), ({"E": 0}, -2, "E=0"), ({"E": 257, "G": 1, "KG": 1}, -2, "E=257"),
    ({"scoring": 2}, -1, "scoring"), ({"gs": 2}, -1, "group score"), ({"G": 0}, -1, "groups"),
    ({"G": 7}, -1, "do not divide"), ({"E": 128, "G": 128}, -2, "at most 64"),
    ({"KG": 0}, -1, "topk_groups"), ({"KG": 9}, -1, "topk_groups"), ({"K": 0}, -1, "top-k"),
    ({"K": 17, "ld": 17}, -1, "experts of 2 groups"), ({"K": 65, "KG": 8, "E": 128, "ld": 65}, -2, "over 64"),
    ({"ld": 5}, -1, "stride"), ({"scale": float("inf")}, -1, "finite"),
    ({"scale": float("nan")}, -1, "finite"), ({"logits": None}, -1, "NULL"),
    ({"w": None}, -1, "NULL"), ({"ids": None}, -1, "NULL"), ({"T": 0, "logits": None}, 0, None),
])
def test_grouped_topk(over, code, msg):
    a = dict(logits=P, bias=None, T=4, E=64, K=6, scoring=1, G=8, KG=2, gs=0, renorm=1, scale=1.0,
             w=P, ids=P, i64=1, ld=6)
    a.update(over)
    rc, err = _rc("moe355_grouped_topk", *a.values(), None)
    assert rc == code and (msg is None or msg in err)


@pytest.mark.parametrize("args,code,msg", [
    ((P, P, 4, 60, 8, 1, 1, P, None), -2, "H % 8"), ((P, P, 4, 64, 300, 1, 1, P, None), -2, "E=300"),
    ((P, P, 4, 64, 8, 4, 1, P, None), -1, "dtype"), ((P, P, 4, 64, 8, 1, 1, None, None), -1, "NULL"),
    ((P + 2, P, 4, 64, 8, 1, 1, P, None), -1, "aligned"), ((P, P, -2, 64, 8, 1, 1, P, None), -1, "T=-2"),
])
def test_router_logits(args, code, msg):
    rc, err = _rc("moe355_router_logits", *args)
    assert rc == code and msg in err


@pytest.mark.parametrize("rows,cols,gate_up,code", [
    (64, 64, 1, 0), (32, 64, 0, 0), (32, 64, 1, -2), (65, 64, 1, -1), (64, 48, 0, -2),
    (48, 64, 0, -2), (0, 64, 0, -1), (64, 0, 0, -2), (1 << 22, 64, 0, -2),
])
def test_matrix_bytes_and_pack(rows, cols, gate_up, code):
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    rc, _ = _rc("moe355_mx_matrix_bytes", rows, cols, gate_up, ctypes.byref(a), ctypes.byref(b))
    assert rc == code
    if rc == 0:
        rp = 2 * padded(rows // 2) if gate_up else padded(rows)
        assert a.value == rp * padded(cols) // 2 and b.value == rp * padded(cols) // 32
        for bad, msg in (((None, P, rows, cols, gate_up, -1, P, P, None), "NULL"),
                         ((P, None, rows, cols, gate_up, -1, P, P, None), "NULL"),
                         ((P + 4, P, rows, cols, gate_up, -1, P, P, None), "aligned"),
                         ((P, None, rows, cols, gate_up, 7, P, P, None), "dtype"),
                         ((P + 1, None, rows, cols, gate_up, 1, P, P, None), "aligned")):
            rc, err = _rc("moe355_mx_pack", *bad)
            assert rc == -1 and msg in err
    else:
        assert _rc("moe355_mx_pack", P, P, rows, cols, gate_up, -1, P, P, None)[0] == code


def _experts_args(**over):
    a = dict(x=P, xs=None, w1=P, w1s=P, w2=P, w2s=P, tw=P, ids=P, i64=1, T=4, H=64, I=64, E=8, K=2,
             dtype=1, act=0, out=P, acc=0, ws=P, ws_bytes=1 << 40)
    a.update(over)
    return (*a.values(), None)


@pytest.mark.parametrize("over,code,msg", [
    ({"T": -1}, -1, "T=-1"), ({"H": 48}, -2, "multiples of 32"), ({"I": 40}, -2, "multiples of 32"),
    ({"E": 257}, -2, "E=257"), ({"K": 9}, -1, "top-k"), ({"K": 0}, -1, "top-k"),
    ({"dtype": 3}, -1, "dtype"), ({"act": 3}, -1, "activation"), ({"T": 1 << 30}, -2, "too large"),
    ({"H": 1 << 21}, -2, "2^20"), ({"w1": None}, -1, "NULL"), ({"w2s": None}, -1, "NULL"),
    ({"tw": None}, -1, "NULL"), ({"out": None}, -1, "NULL"), ({"x": P + 8}, -1, "aligned"),
    ({"xs": P + 2}, -1, "aligned"), ({"w1s": P + 4}, -1, "aligned"), ({"ws": None}, -3, "workspace"),
    ({"ws_bytes": 1000}, -3, "workspace"), ({"ws": P + 8}, -1, "aligned"),
    ({"T": 0, "x": None, "ws": None}, 0, None),
])
def test_experts(over, code, msg):
    rc, err = _rc("moe355_mx_fused_experts", *_experts_args(**over))
    assert rc == code and (msg is None or msg in err)


@pytest.mark.parametrize("T,H,I,E,K", [(0, 64, 64, 1, 1), (1, 4096, 14336, 8, 2), (4096, 2048, 1408, 64, 6),
                                       (333, 1248, 3296, 12, 3), (100000, 4096, 14336, 8, 2)])
def test_workspace_covers_every_stage(T, H, I, E, K):
    for dtype in (0, 1, 2):
        n = _capi.mx_workspace_bytes(T, H, I, E, K, dtype, torch.device("cpu"))
        R = T * K
        least = T * padded(H) * 33 // 32 + R * padded(I) * 33 // 32 + R * 8
        assert n >= least


@pytest.mark.parametrize("H,I,E,K", [(1 << 20, 1 << 20, 4, 2), (1 << 20, 1 << 17, 1, 1), (1 << 19, 1 << 20, 8, 1),
                                     (960000, 256, 256, 2)])
def test_workspace_covers_the_last_part_of_a_call_of_several(H, I, E, K):
    """Tokens past 2 GB of 8-bit codes run in parts, and the columns of a small last part
    may be cut into more planes of fp32 results than those of a full one."""
    part = 0x7FFFFFFF // padded(H)
    cpu = torch.device("cpu")
    for dtype in (0, 1, 2):
        for rest in (0, 1, 3, 17, 200, 1381, part // 3, part // 2, part - 1):
            whole = _capi.mx_workspace_bytes(part + rest, H, I, E, K, dtype, cpu)
            assert whole >= _capi.mx_workspace_bytes(part, H, I, E, K, dtype, cpu)
            assert whole >= _capi.mx_workspace_bytes(rest, H, I, E, K, dtype, cpu)


def test_more_rows_than_the_interface_counts():
    with pytest.raises(ValueError, match="rows"):
        _capi.mx_workspace_bytes(1 << 32, 64, 64, 1, 1, 1, torch.device("cpu"))
    big = torch.zeros(1, 1).expand(1 << 31, 1)
    out = torch.zeros(1, 1)
    with pytest.raises(ValueError, match="rows"):
        _capi.grouped_topk(big, None, 1, 0, 1, 1, 0, False, 1.0, out, out, stream=0)
    with pytest.raises(ValueError, match="rows"):
        _capi.mx_quantize(big, out, out, stream=0)


def _cpu_experts(E=2, H=64, I=32):
    return Mxfp4Experts(E, H, I)


def test_python_refusals():
    x = torch.zeros(3, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        quantize_mxfp8(x)
    with pytest.raises(RuntimeError, match="GPU"):
        grouped_topk(x, 2)
    with pytest.raises(RuntimeError, match="GPU"):
        fused_experts_mxfp4(x, _cpu_experts(), torch.ones(3, 1), torch.zeros(3, 1).long())
    with pytest.raises(RuntimeError, match="GPU"):
        RMSNorm(64, 1e-5).forward_mxfp8(x)
    with pytest.raises(ValueError, match="whole blocks"):
        Mxfp4Experts(2, 48, 32)
    with pytest.raises(ValueError, match="num_experts"):
        Mxfp4Experts(257, 64, 32)
    with pytest.raises(RuntimeError, match="GPU"):
        Mxfp4Experts.quantize(torch.zeros(2, 64, 64), torch.zeros(2, 64, 32))
    u8 = torch.uint8
    good = (torch.zeros(2, 64, 32, dtype=u8), torch.zeros(2, 64, 2, dtype=u8),
            torch.zeros(2, 64, 16, dtype=u8), torch.zeros(2, 64, 1, dtype=u8))
    with pytest.raises(RuntimeError, match="GPU"):
        Mxfp4Experts.from_codes(*good)
    for k, bad, msg in ((1, torch.zeros(2, 64, 3, dtype=u8), "belong together"),
                        (0, torch.zeros(64, 32, dtype=u8), "stacked"),
                        (0, torch.zeros(2, 64, 32), "bytes"),
                        (0, torch.zeros(2, 64, 24, dtype=u8), "belong together")):
        args = list(good)
        args[k] = bad
        with pytest.raises(ValueError, match=msg):
            Mxfp4Experts.from_codes(*args)
    with pytest.raises(ValueError, match="no experts"):
        Mxfp4Experts.quantize([], [])


def test_rows_check_their_tensors():
    c = torch.zeros(3, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.zeros(3, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    q = Mxfp8Rows(c, s, 96)
    assert q.codes.shape == (3, 96) and q.scales.shape == (3, 3) and len(q) == 3
    assert Mxfp8Rows(c, s, 128).codes is c
    for args, msg in (((c, s, 100), "whole blocks"), ((c, s, 160), "codes must"),
                      ((c.view(torch.uint8), s, 96), "codes must"), ((c, s[:2], 96), "scales must"),
                      ((c[:, ::2], s, 32), "codes must"), ((c, s.view(torch.uint8), 96), "scales must")):
        with pytest.raises(ValueError, match=msg):
            Mxfp8Rows(*args)


def test_dequantize_on_the_cpu():
    codes = torch.tensor([[1.5, -448.0] + [0.0] * 126]).to(torch.float8_e4m3fn)
    scales = torch.tensor([[130, 0, 127, 255]], dtype=torch.uint8).view(torch.float8_e8m0fnu)
    v = Mxfp8Rows(codes, scales, 128).dequantize()
    assert v[0, 0] == 12.0 and v[0, 1] == -3584.0 and bool(torch.isnan(v[0, 96:]).all())
    assert bool((v[0, 2:96] == 0).all())


def test_experts_move_as_a_module_and_keep_their_bytes():
    x = _cpu_experts()
    assert x.nbytes == 2 * (2 * 128 * 128 // 2 + 2 * 128 * 128 // 32 + 128 * 128 // 2 + 128 * 128 // 32)
    assert x.to(torch.float16).w1.dtype == torch.uint8
    assert set(x.state_dict()) == {"w1", "w1_scales", "w2", "w2_scales"}


def test_column_parts_are_never_empty():
    """What mx_plan does to the steps of down on 64- and 256-row tiles: parts c with at least
    4 c steps."""
    for steps in range(1, 8193):
        for c in (1, 2, 4):
            if c == 1 or steps >= 4 * c:
                assert (c - 1) * -(-steps // c) < steps


@pytest.mark.parametrize("w,ids", [
    ((2, 6), (2, 6)),      # of the transposed routing of 6 tokens of 2 slots
    ((6, 2), (2, 6)), ((2, 6), (6, 2)),
    ((6, 2), (12,)), ((12,), (6, 2)), ((12,), (12,)),
    ((3, 4), (3, 4)), ((6, 2), (3, 4)), ((6, 2), (6, 1, 2)), ((6, 2), (6, 3)),
])
def test_routing_of_another_shape_than_the_tokens(w, ids):
    """As many numbers as [6, 2] has, or as their multiples, in other places."""
    rows = Mxfp8Rows(torch.zeros(6, 128, dtype=torch.uint8).view(torch.float8_e4m3fn),
                     torch.zeros(6, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu), 64)
    with pytest.raises(ValueError, match=r"are not \[6, K\]"):
        fused_experts_mxfp4(rows, _cpu_experts(), torch.ones(w), torch.zeros(ids).long())


@pytest.mark.parametrize("T,H,I,E,K", [(0, 64, 64, 1, 1), (1, 4096, 14336, 8, 2), (4096, 2048, 1408, 64, 6),
                                       (40000, 1 << 17, 256, 16, 2)])
def test_workspace_of_any_call_and_of_a_known_one(T, H, I, E, K):
    for dtype in (0, 1, 2):
        known = [_capi.mx_workspace_bytes(T, H, I, E, K, dtype, torch.device("cpu"), acc)
                 for acc in (False, True)]
        both = ctypes.c_size_t()
        assert _rc("moe355_mx_workspace_bytes", T, H, I, E, K, dtype, ctypes.byref(both))[0] == 0
        assert both.value == max(known)
        if dtype != 1:  # only bf16 results have slots of 16 bits
            assert known[0] == known[1]
    assert _rc("moe355_mx_call_workspace_bytes", T, H, I, E, K, 1, 0, None)[0] == -1
