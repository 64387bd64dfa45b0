"""The error that the routing by groups allows its 32-bit choices (group_topk.hip), on the
CPU: the constants of the source against the bound of the arithmetic they stand for, and
the arithmetic itself, replayed in 32 bits in the kernels' order, against both."""

from __future__ import annotations

import os
import re

import numpy as np
import pytest

SRC = open(os.path.join(os.path.dirname(__file__), "..", "reframework_amd", "csrc",
                        "group_topk.hip")).read()
U = 2.0 ** -24
EXPERTS = 256


def _constant(name):
    env = {}
    for key, expr in re.findall(r"\b(k\w+) = ([^,;]+)[,;]", SRC):
        expr = re.sub(r"(?<=[0-9])f\b", "", expr.strip())
        expr = re.sub(r"0x1p(-?\d+)f?", r"2.0 ** (\1)", expr)
        try:
            env[key] = eval(expr, {"__builtins__": {}}, dict(env))
        except Exception:  # not a number
            continue
    return env[name]


def _mean_exponent():
    """Largest mean of |v|, weighted by exp(v), over 256 values v <= 0 of which one is 0: the
    others equal (the weighted mean is largest where its derivative vanishes for each)."""
    a = np.linspace(0.0, 40.0, 400001)
    w = (EXPERTS - 1) * np.exp(-a)
    return float((w * a / (1.0 + w)).max())


def _pair_bound(additions):
    """Of the difference of two softmax scores, relative to the token's largest."""
    per_v = 2 * U + (1.4426950408889634 / float(np.float32(1.4426950408889634)) - 1)
    per_v = abs(per_v) + 2e-8
    unit = 2 * U
    top = per_v * _mean_exponent() + unit + additions * U + U
    each = per_v * np.exp(-1.0) + unit + U
    return top + 2 * each


def _additions():
    """(a lane's experts, levels over the lanes) of the two kernels."""
    one = max(int(n) for n in re.findall(r"group_topk_kernel<(\d+)>", SRC))
    rows = 4 * max(int(n) for n in re.findall(r"group_topk_rows_kernel<(\d+)>", SRC))
    return (one, 6), (rows, 4)


def test_constants_cover_the_bound():
    (one, wave), (rows, row) = _additions()
    assert (one, rows) == (8, 16)
    assert 2 * _constant("kScoreError") >= _pair_bound(one - 1 + wave)
    assert 2 * _constant("kRowScoreError") >= _pair_bound(rows - 1 + row)
    # bias, sum of two, difference: three roundings of a choice
    assert _constant("kRounding") >= 3 * U * (1 + 2.0 ** -20)
    assert _constant("kRowRounding") >= 2.0 ** -19 + 3 * U * (1 + 2.0 ** -18)


def _scores32(l, per_lane):
    f = np.float32
    m = l.max(1, keepdims=True)
    e = np.exp2(((l - m).astype(f) * f(1.4426950408889634)).astype(f)).astype(f)
    lanes = e.reshape(len(l), -1, per_lane)
    s = np.zeros(lanes.shape[:2], f)
    for i in range(per_lane):
        s = (s + lanes[:, :, i]).astype(f)
    while s.shape[1] > 1:
        s = (s[:, ::2] + s[:, 1::2]).astype(f)
    return (e * (f(1) / s)).astype(f)


@pytest.mark.parametrize("per_lane,name", [(8, "kScoreError"), (4, "kScoreError"), (16, "kRowScoreError")])
@pytest.mark.parametrize("spread", [0.3, 1.5, 6.0])
def test_replayed_scores_lie_within_it(per_lane, name, spread):
    rng = np.random.default_rng(per_lane)
    l = (rng.normal(size=(4000, EXPERTS)) * spread).astype(np.float32)
    x = l.astype(np.float64)
    e = np.exp(x - x.max(1, keepdims=True))
    want = e / e.sum(1, keepdims=True)
    err = _scores32(l, per_lane).astype(np.float64) - want
    pair = err.max(1) - err.min(1)
    assert np.all(pair <= 2 * _constant(name) * want.max(1))
