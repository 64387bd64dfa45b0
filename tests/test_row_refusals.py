"""Refusals of LayerNorm, of tokens by expert and back and of the 8-bit products, on the CPU
(nothing is launched): the C entry points by status, the Python ones by exception; and what the
workspaces have to hold."""

from __future__ import annotations

import ctypes

import pytest
import torch

from reframework_amd import _capi
from reframework_amd.fp8 import blocks, padded
from reframework_amd.layers import LayerNorm
from reframework_amd.moe import (Fp8Experts, Fp8Rows, Fp8Weight, TokenOrder, combine_tokens,
                                 fused_experts_fp8, matmul_fp8, permute_tokens, quantize_fp8,
                                 token_order)

P = 4096  # an aligned address that no refused call reads
E4M3 = torch.float8_e4m3fn


def _rc(name, *args):
    lib = _capi.lib()
    rc = getattr(lib, name)(*args)
    return rc, lib.moe355_last_error().decode()


def _check(name, defaults, over, code, msg):
    a = dict(defaults)
    a.update(over)
    rc, err = _rc(name, *a.values(), None)
    assert rc == code and (msg is None or msg in err), (rc, err)


NORM = dict(x=P, residual=P, residual_out=P, weight=P, bias=P, wdtype=0, eps=1e-5, T=4, H=60, dtype=1, out=P,
            mean=P, rstd=P)


@pytest.mark.parametrize("over,code,msg", [
    ({"T": -1}, -1, "T=-1"), ({"H": 0}, -1, "H=0"), ({"H": 16385}, -2, "H <= 16384"),
    ({"H": 8193, "dtype": 0}, -2, "H <= 8192"), ({"T": 1 << 24}, -2, "2^24 rows"), ({"dtype": 3}, -1, "dtype"), ({"wdtype": -1}, -1, "dtype"),
    ({"eps": -1.0}, -1, "eps"), ({"eps": float("nan")}, -1, "eps"), ({"x": None}, -1, "NULL"),
    ({"weight": None}, -1, "NULL"), ({"out": None}, -1, "NULL"), ({"residual_out": None}, -1, "residual_out"),
    ({"mean": None}, -1, "mean and rstd"), ({"rstd": None}, -1, "mean and rstd"), ({"x": P + 1}, -1, "aligned"),
    ({"weight": P + 2}, -1, "aligned"), ({"bias": P + 2}, -1, "aligned"), ({"T": 0, "x": None}, 0, None)])
def test_layer_norm(over, code, msg):
    _check("moe355_layer_norm", NORM, over, code, msg)


BWD = dict(dy=P, dres=P, r=P, weight=P, wdtype=1, mean=P, rstd=P, T=4, H=60, dtype=1, dx=P, dw=P, db=P, ws=P,
           ws_bytes=1 << 30)


@pytest.mark.parametrize("over,code,msg", [
    ({"T": 0}, -1, "no rows"), ({"T": -3}, -1, "T=-3"), ({"H": 20000}, -2, "H <="), ({"dtype": 9}, -1, "dtype"),
    ({"dy": None}, -1, "NULL"), ({"mean": None}, -1, "NULL"), ({"r": None}, -1, "NULL"),
    ({"ws": None}, -3, "workspace"), ({"ws_bytes": 100}, -3, "workspace"), ({"ws": P + 8}, -1, "aligned"),
    ({"dx": P + 1}, -1, "aligned"), ({"dw": P + 1}, -1, "aligned")])
def test_layer_norm_bwd(over, code, msg):
    _check("moe355_layer_norm_bwd", BWD, over, code, msg)


ORDER = dict(ids=P, i64=1, T=4, K=2, E=8, offsets=P, slots=P, src=P, ws=P, ws_bytes=1 << 20)


@pytest.mark.parametrize("over,code,msg", [
    ({"T": 0}, -1, "no slots"), ({"T": -1}, -1, "T=-1"), ({"K": 0}, -1, "K=0"), ({"E": 0}, -2, "E=0"),
    ({"E": 257}, -2, "E=257"), ({"T": 1 << 25, "K": 64}, -2, "too large"),
    ({"T": 1 << 26}, -2, "2^26 tokens"), ({"ids": None}, -1, "NULL"),
    ({"offsets": None}, -1, "NULL"), ({"ws": None}, -3, "workspace"), ({"ws_bytes": 8}, -3, "workspace"),
    ({"ws": P + 4}, -1, "aligned")])
def test_token_order(over, code, msg):
    _check("moe355_token_order", ORDER, over, code, msg)


@pytest.mark.parametrize("T,K,E", [(1, 1, 1), (512, 2, 8), (513, 2, 8), (4096, 8, 256), (1 << 20, 8, 3)])
def test_token_order_workspace(T, K, E):
    n = ctypes.c_size_t()
    assert _rc("moe355_token_order_workspace_bytes", T, K, E, ctypes.byref(n))[0] == 0
    R = T * K
    # counts of 256 slots each above 1024 of them, and a tile map of at most E + R / 2^20 tiles
    assert n.value >= (-(-R // 256) if R > 1024 else 1) * E * 4 + (2 + 2 * (E + R // (1 << 20))) * 4


@pytest.mark.parametrize("name,defaults,cases", [
    ("moe355_permute_rows", dict(x=P, offsets=P, slots=P, T=4, H=60, K=2, E=8, dtype=1, rows=P), [
        ({"T": -1}, -1, "T=-1"), ({"H": 0}, -1, "H=0"), ({"dtype": 4}, -1, "dtype"), ({"x": None}, -1, "NULL"),
        ({"H": 1 << 24}, -2, "2^24 wide"),
        ({"rows": None}, -1, "NULL"), ({"x": P + 1}, -1, "aligned"), ({"T": 0, "x": None}, 0, None)]),
    ("moe355_combine_rows", dict(rows=P, w=None, slots=P, T=4, H=60, K=2, dtype=1, out=P), [
        ({"K": 0}, -1, "K=0"), ({"rows": None}, -1, "NULL"), ({"out": None}, -1, "NULL"),
        ({"out": P + 1}, -1, "aligned"), ({"dtype": 7}, -1, "dtype"), ({"T": 0, "rows": None}, 0, None)]),
    ("moe355_combine_rows_bwd", dict(dout=P, rows=P, w=P, offsets=P, slots=P, T=4, H=60, K=2, E=8, dtype=1, drows=P,
                                     dw=P), [
        ({"dout": None}, -1, "NULL"), ({"rows": None}, -1, "NULL"), ({"w": None}, -1, "NULL"),
        ({"drows": P + 1}, -1, "aligned"), ({"E": 999}, -2, "E=999"), ({"T": 0}, 0, None),
        ({"drows": None, "dw": None, "dout": None}, 0, None)])])
def test_token_rows(name, defaults, cases):
    for over, code, msg in cases:
        _check(name, defaults, over, code, msg)


@pytest.mark.parametrize("name,defaults,cases", [
    ("moe355_fp8_quantize", dict(x=P, M=4, K=60, dtype=1, codes=P, scales=P), [
        ({"M": -1}, -1, "sizes"), ({"K": 0}, -1, "sizes"), ({"K": (1 << 20) + 1}, -2, "2^20"), ({"dtype": 5}, -1, "dtype"),
        ({"M": 1 << 24, "K": 2000}, -2, "2^28 blocks"),
        ({"x": None}, -1, "NULL"), ({"scales": None}, -1, "NULL"), ({"codes": P + 8}, -1, "aligned"),
        ({"x": P + 1}, -1, "aligned"), ({"M": 0, "x": None}, 0, None)]),
    ("moe355_fp8_quantize_weight", dict(w=P, N=100, K=60, dtype=0, cells=P, scales=P), [
        ({"N": 0}, -1, "N=0"), ({"K": -1}, -1, "sizes"), ({"N": 1 << 20, "K": 4096}, -2, "2 GB"), ({"w": None}, -1, "NULL"),
        ({"w": P + 2}, -1, "aligned"), ({"cells": P + 8}, -1, "aligned")]),
    ("moe355_fp8_pack", dict(codes=P, N=100, K=60, cells=P), [
        ({"N": 0}, -1, "N=0"), ({"codes": None}, -1, "NULL"), ({"cells": P + 4}, -1, "aligned"),
        ({"N": 1 << 20, "K": 1 << 20}, -2, "2 GB")]),
    ("moe355_fp8_matmul", dict(x=P, xs=P, w=P, ws=P, offsets=P, M=4, N=100, K=60, E=3, dtype=1, out=P, space=P,
                               bytes=1 << 40), [
        ({"M": -1}, -1, "M=-1"), ({"M": 1 << 30}, -2, "too large"), ({"E": 0}, -2, "E=0"), ({"E": 300}, -2, "E=300"), ({"N": 0}, -1, "N=0"),
        ({"dtype": 8}, -1, "dtype"), ({"offsets": None}, -1, "without offsets"), ({"xs": None}, -1, "NULL"),
        ({"out": None}, -1, "NULL"), ({"x": P + 8}, -1, "aligned"), ({"offsets": P + 2}, -1, "aligned"),
        ({"out": P + 4}, -1, "aligned"), ({"space": P + 8}, -1, "aligned"), ({"M": 0, "x": None}, 0, None),
        ({"M": 8192, "N": 14336, "K": 4096, "E": 8, "space": None}, -3, "workspace"),
        ({"M": 8192, "N": 14336, "K": 4096, "E": 8, "bytes": 1 << 20}, -3, "workspace")])])
def test_fp8_entry_points(name, defaults, cases):
    for over, code, msg in cases:
        _check(name, defaults, over, code, msg)


EXPERTS = dict(x=P, xs=None, w1=P, w1s=P, w2=P, w2s=P, tw=P, ids=P, i64=1, T=4, H=64, I=48, E=8, K=2, dtype=1, act=0,
               out=P, ws=P, ws_bytes=1 << 40)


@pytest.mark.parametrize("over,code,msg", [
    ({"T": -1}, -1, "T=-1"), ({"H": 40}, -2, "multiples of 16"), ({"I": 8}, -2, "multiples of 16"), ({"H": 0}, -1, "H=0"),
    ({"E": 257}, -2, "E=257"), ({"K": 9}, -1, "top-k"), ({"K": 0}, -1, "top-k"), ({"dtype": 3}, -1, "dtype"),
    ({"act": 3}, -1, "activation"), ({"T": 1 << 30}, -2, "too large"), ({"I": 1 << 20}, -2, "2^19"),
    ({"H": 1 << 16, "I": 1 << 15}, -2, "2 GB"), ({"w1": None}, -1, "NULL"), ({"tw": None}, -1, "NULL"),
    ({"x": P + 8}, -1, "aligned"), ({"xs": P + 2}, -1, "aligned"), ({"ws": None}, -3, "workspace"),
    ({"ws_bytes": 64}, -3, "workspace"), ({"ws": P + 8}, -1, "aligned"), ({"T": 0, "x": None, "ws": None}, 0, None)])
def test_fp8_experts(over, code, msg):
    _check("moe355_fp8_fused_experts", EXPERTS, over, code, msg)


@pytest.mark.parametrize("T,H,I,E,K", [(0, 64, 64, 1, 1), (1, 4096, 14336, 8, 2), (4096, 2048, 1408, 64, 6),
                                       (333, 1248, 3296, 12, 3), (100000, 4096, 14336, 8, 2), (600000, 4096, 256, 4, 1)])
def test_fp8_workspace_covers_every_stage(T, H, I, E, K):
    part = min(T, 0x7FFFFFFF // padded(H))  # tokens past 2 GB of codes run in parts
    R = part * K
    for dtype in (0, 1, 2):
        n = _capi._size(torch.device("cpu"), "moe355_fp8_workspace_bytes", T, H, I, E, K, dtype)
        assert n >= part * (padded(H) + 4 * blocks(H)) + R * (padded(I) + 4 * blocks(I)) + \
            R * H * (2 if dtype == 1 else 4) + R * 8


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("last", [1, 100, 4000, 8000, 10000, 16000])
def test_fp8_workspace_of_a_call_in_parts(last, dtype):
    """What the last part takes may be more than the first: fewer rows, but other kernels."""
    H, I, E, K = 122880, 16, 256, 2
    first = 0x7FFFFFFF // H

    def size(T):
        return _capi._size(torch.device("cpu"), "moe355_fp8_workspace_bytes", T, H, I, E, K, dtype)

    assert size(first + last) >= max(size(first), size(last))
    assert size(2 * first + last) == size(first + last)


def _weight(E=2, N=40, K=70):
    cells = torch.zeros(E, blocks(N), blocks(K), 16384, dtype=torch.uint8)
    return Fp8Weight(cells, torch.zeros(E, blocks(N), blocks(K)), N, K)


def _experts(E=2, H=64, I=32):
    def m(n, k):
        return (torch.zeros(E, n, blocks(k), 16384, dtype=torch.uint8), torch.zeros(E, n, blocks(k)))
    return Fp8Experts(m(2 * blocks(I), H), m(blocks(H), I), H, I)


def test_python_refusals():
    x = torch.zeros(3, 64)
    for f in (lambda: LayerNorm(64, 1e-5)(x), lambda: LayerNorm(64, 1e-5).forward_add_residual(x, x),
              lambda: quantize_fp8(x), lambda: matmul_fp8(x, _weight()), lambda: Fp8Weight.quantize(x),
              lambda: permute_tokens(x, torch.zeros(3, 1).long(), 4), lambda: token_order(torch.zeros(3, 1).long(), 4),
              lambda: Fp8Experts.quantize(torch.zeros(2, 64, 64), torch.zeros(2, 64, 32)),
              lambda: fused_experts_fp8(x, _experts(), torch.ones(3, 1), torch.zeros(3, 1).long())):
        with pytest.raises(RuntimeError, match="GPU"):
            f()
    c = torch.zeros(2, 40, 70).to(E4M3)
    s = torch.zeros(2, 1, 1)
    with pytest.raises(RuntimeError, match="GPU"):
        Fp8Weight.from_codes(c, s)
    for codes, scales, msg in ((c, torch.zeros(2, 1, 2), "belong together"), (c, s[0], "stacked"), (c.float(), s, "codes are"),
                               (c, s.double(), "codes are"), (c[:, :0], s, "belong together")):
        with pytest.raises(ValueError, match=msg):
            Fp8Weight.from_codes(codes, scales)
    w1, w2 = torch.zeros(2, 64, 64).to(E4M3), torch.zeros(2, 64, 32).to(E4M3)
    for a, b, msg in ((w1, w2[:, :32], "are not"), (w1[:, :48], torch.zeros(2, 64, 24).to(E4M3), "multiples of 16"),
                      (w1[0], w2, "stacked")):
        with pytest.raises(ValueError, match=msg):
            Fp8Experts.from_codes(a, s, b, s)
    with pytest.raises(RuntimeError, match="GPU"):
        Fp8Experts.from_codes(w1, torch.zeros(2, 2, 1), w2, s)


def test_products_check_their_tensors():
    rows = Fp8Rows(torch.zeros(6, 128, dtype=torch.uint8).view(E4M3), torch.zeros(6, 1), 70)
    for args, msg in (((rows, _weight(K=71)), "columns"), ((rows, _weight()), "need offsets"),
                      ((rows, _weight(), torch.zeros(2).int()), r"not \[3\]")):
        with pytest.raises(ValueError, match=msg):
            matmul_fp8(*args)
    with pytest.raises(TypeError, match="offsets"):
        matmul_fp8(rows, _weight(), torch.zeros(3))
    with pytest.raises(TypeError, match="float"):
        matmul_fp8(rows, _weight(), torch.zeros(3).int(), out_dtype=torch.float64)
    big = Fp8Rows(torch.zeros(6, 128, dtype=torch.uint8).view(E4M3), torch.zeros(6, 1), 64)
    for w, ids in (((2, 6), (2, 6)), ((6, 2), (2, 6)), ((6, 2), (12,)), ((12,), (12,)), ((6, 2), (6, 3))):
        with pytest.raises(ValueError, match=r"are not \[6, K\]"):
            fused_experts_fp8(big, _experts(), torch.ones(w), torch.zeros(ids).long())
    with pytest.raises(ValueError, match="hidden size"):
        fused_experts_fp8(rows, _experts(), torch.ones(6, 1), torch.zeros(6, 1).long())
    with pytest.raises(ValueError, match="unknown gated activation"):
        fused_experts_fp8(big, _experts(), torch.ones(6, 1), torch.zeros(6, 1).long(), activation="relu")


def test_rows_check_their_tensors():
    c, s = torch.zeros(3, 256, dtype=torch.uint8).view(E4M3), torch.zeros(3, 2)
    q = Fp8Rows(c, s, 200)
    assert q.codes.shape == (3, 200) and len(q) == 3 and q.dequantize().shape == (3, 200)
    assert Fp8Rows(c, s, 256).codes is c
    for args, msg in (((c, s, 0), "size 0"), ((c, s, 128), "codes must"), ((c, s[:2], 200), "scales must"),
                      ((c.view(torch.uint8), s, 200), "codes must"), ((c, s.double(), 200), "scales must")):
        with pytest.raises(ValueError, match=msg):
            Fp8Rows(*args)


def test_tokens_check_their_tensors():
    order = TokenOrder(torch.zeros(5).int(), torch.zeros(3, 2).int(), torch.zeros(6).int(), 4)
    with pytest.raises(RuntimeError, match="GPU"):
        combine_tokens(torch.zeros(6, 8), order, torch.zeros(3, 2))
    o, s, r = torch.zeros(5).int(), torch.zeros(3, 2).int(), torch.zeros(6).int()
    for args, msg in (((o, s, r, 5), "are not"), ((o, s.flatten(), r, 4), "are not"), ((o, s, r[:5], 4), "are not"),
                      ((o.long(), s, r, 4), "int32"), ((o, s.long(), r, 4), "int32"),
                      ((o, torch.zeros(2, 3).int().t(), r, 4), "contiguous")):
        with pytest.raises(ValueError, match=msg):
            TokenOrder(*args)


def test_codes_leave_a_module_as_they_came():
    w = _weight()
    assert w.to(torch.float16).w.dtype == torch.uint8 and set(w.state_dict()) == {"w", "w_scales"}
    assert w.dequantize().shape == (2, 40, 70) and not w.has_transposed
    e = _experts()
    assert e.dequantize("w1").shape == (2, 64, 64) and e.dequantize("w2").shape == (2, 64, 32)
    assert set(e.state_dict()) == {"w1", "w1_scales", "w2", "w2_scales"}


def test_a_cell_holds_every_code_once():
    """Place of row n and column k in a cell, as the header states it, against the layout that
    Fp8Weight.codes() reads."""
    cell = torch.arange(16384).reshape(1, 1, 1, 8, 2, 4, 16, 16).permute(0, 1, 3, 6, 2, 4, 5, 7).reshape(128, 128)
    n, k = torch.meshgrid(torch.arange(128), torch.arange(128), indexing="ij")
    at = n // 16 * 2048 + k % 128 // 64 * 1024 + (k // 16 % 4 * 16 + n % 16) * 16 + k % 16
    assert torch.equal(cell, at) and torch.equal(at.flatten().sort()[0], torch.arange(16384))


@pytest.mark.parametrize("steps", [16, 17, 31, 32, 33, 65, 112, 200])
def test_parts_of_an_item_cover_its_steps_once(steps):
    for split in (2, 4, 8, 16):
        if steps >= 4 * split:
            ends = [(p * steps // split, (p + 1) * steps // split) for p in range(split)]
            assert ends[0][0] == 0 and ends[-1][1] == steps
            assert all(a < b for a, b in ends) and all(x[1] == y[0] for x, y in zip(ends, ends[1:]))


def test_sizes_past_a_launch_are_refused():
    """A launch holds less than 2^32 threads: 256 for every four tokens, or every 16 blocks,
    begun."""
    for T in ((1 << 26) - 3, (1 << 26) - 1):
        for name, defaults in (
                ("moe355_permute_rows", dict(x=P, offsets=P, slots=P, T=T, H=1, K=1, E=1, dtype=1, rows=P)),
                ("moe355_combine_rows", dict(rows=P, w=None, slots=P, T=T, H=1, K=1, dtype=1, out=P)),
                ("moe355_combine_rows_bwd", dict(dout=P, rows=P, w=P, offsets=P, slots=P, T=T, H=1, K=1, E=1,
                                                 dtype=1, drows=P, dw=P))):
            _check(name, defaults, {}, -2, "2^26 - 4")
    quantize = dict(x=P, M=1, K=128, dtype=1, codes=P, scales=P)
    for M, K in (((1 << 28) - 15, 1), ((1 << 28) - 1, 128), (1 << 24, 2000)):
        _check("moe355_fp8_quantize", quantize, {"M": M, "K": K}, -2, "2^28 - 16")
    n = ctypes.c_size_t()  # the order itself takes three more
    assert _rc("moe355_token_order_workspace_bytes", (1 << 26) - 1, 1, 1, ctypes.byref(n))[0] == 0
