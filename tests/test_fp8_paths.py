"""Which kernels the tests of the 8-bit products and experts reach, on the CPU: the library's own
rule (fp8_path.h, built here as plain C++) answers for the sizes of _fp8_paths.py, so that a
change of the rule that leaves a kernel without a test shows. And the bounds of _fp8_paths.py are
narrow enough to see what they are for."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest
import torch

import _fp8_paths as paths
from reframework_amd.fp8 import BLOCK, blocks

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "reframework_amd",
                    "csrc")
CUS = 256
DTYPES = {0: "f32", 1: "bf16", 2: "f16"}
MAIN = r"""
#include <cstdio>
#include "fp8_path.h"
using namespace moe355;
int main() {
  char kind;
  int a, b, c, d, e, dtype, cus;
  while (std::scanf(" %c %d %d %d %d %d %d %d", &kind, &a, &b, &c, &d, &e, &dtype, &cus) == 8) {
    if (kind == 'p') {
      const F8Path p = f8_path(a, b, f8_pad(c), d, dtype == MOE355_F32, cus);
      std::printf("%d %d\n", p.tile_rows, p.max_parts > 0);
    } else {
      const F8Experts p = f8_experts(a * e, b, c, d, e, dtype, cus);
      std::printf("%d %d %d %d %d %d %d\n", p.up.tile_rows, p.exact_up, p.up.max_parts > 0,
                  p.down.tile_rows, p.exact_down, p.down.max_parts > 0, p.narrow);
    }
  }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    gxx = os.environ.get("CXX") or shutil.which("g++")
    if not gxx:
        pytest.skip("no C++ compiler")
    tmp = tmp_path_factory.mktemp("paths")
    src, exe = tmp / "paths.cpp", tmp / "paths"
    src.write_text(MAIN)
    subprocess.run([gxx, "-std=c++17", "-I", CSRC, str(src), "-o", str(exe)], check=True)

    def run(queries):
        text = "".join(" ".join(map(str, q)) + "\n" for q in queries)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True)
        lines = out.stdout.splitlines()
        assert len(lines) == len(queries)
        return [tuple(map(int, line.split())) for line in lines]

    return run


def test_every_kernel_of_the_products(ask):
    cases = [(s, dt, grad) for s in paths.PRODUCTS for dt in DTYPES for grad in (False, True)]
    answers = ask([("p", M, K if grad else N, N if grad else K, E, 0, dt, CUS) for (M, N, K, E), dt, grad in cases])
    for grads in ({False}, {False, True}):
        reached = {(tile, DTYPES[dt]) for (_, dt, grad), (tile, _) in zip(cases, answers) if grad in grads}
        # results in fp32 have exact products, which end at 128 rows
        assert reached == {(t, dt) for t in (0, 32, 64, 128, 256) for dt in DTYPES.values()} - {(256, "f32")}
    assert {(DTYPES[dt], cut) for (_, dt, _), (tile, cut) in zip(cases, answers) if tile == 256} == \
        {(dt, cut) for dt in ("bf16", "f16") for cut in (0, 1)}


def test_every_kernel_of_the_experts(ask):
    cases = [(s, dt) for s in paths.EXPERTS for dt in DTYPES]
    answers = ask([("e", T, H, I, E, K, dt, CUS) for (T, H, I, E, K, _), dt in cases])
    up = {(tile, exact) for tile, exact, *_ in answers}
    assert up == {(0, 1), (32, 1), (64, 1), (128, 1), (128, 0), (256, 0)}
    down = {(tile, exact) for _, _, _, tile, exact, _, _ in answers}
    assert down == {(t, e) for t in (0, 32, 64, 128) for e in (0, 1)} | {(256, 0)}
    # 256 rows: whole items and cut ones, and of down slots in 16 bits and in fp32
    assert {a[2] for a in answers if a[0] == 256} == {0, 1}
    assert {(a[5], a[6]) for a in answers if a[3] == 256} >= {(1, 1), (1, 0), (0, 0)}
    for activation in ("silu", "gelu", "gelu_tanh"):
        assert any(s[5] == activation for s, _ in cases)


def _call(T, H, I, E, K, seed=0):
    gen = torch.Generator().manual_seed(seed)
    w1, s1, w2, s2 = paths.expert_codes(H, I, E, gen, "cpu")
    x = paths.whole((T, H), gen, "cpu").double()

    def dequantized(w, s, rows):
        s = s.repeat_interleave(BLOCK, 2)[..., :w.shape[2]].double()
        parts = [s[:, i * blocks(rows):(i + 1) * blocks(rows)].repeat_interleave(BLOCK, 1)[:, :rows]
                 for i in range(w.shape[1] // rows)]
        return w.double() * torch.cat(parts, 1)

    ids = torch.argsort(torch.rand(T, E, generator=gen), -1)[:, :K]
    return x, dequantized(w1, s1, I), dequantized(w2, s2, H), torch.rand(T, K, generator=gen) + 0.25, ids


@pytest.mark.parametrize("dt,narrow", [(torch.bfloat16, True), (torch.float16, False), (torch.float32, False)])
@pytest.mark.parametrize("H,I,act", [(256, 384, "silu"), (1040, 528, "gelu_tanh")])
def test_the_bounds_of_the_experts_see_a_wrong_value(H, I, act, dt, narrow):
    """Mistakes planted into the 64-bit result: the last product of a step left out of down's sums
    or of the gates', a neighbour's gates for one feature, another activation, a neighbour's
    weights."""
    x, w1, w2, tw, ids = _call(24, H, I, 4, 2)
    want = paths.experts(x, w1, w2, tw, ids, act, dt, narrow)
    size = want.value.square().mean().sqrt()
    # beside the rounding of the result the bound is a small part of its usual size
    assert float((want.off - paths.half_step(want.value, dt)).mean() / size) < 2.0 ** -5

    def seen(v, share):
        wrong = (v - want.value).abs() > want.off + paths.half_step(want.value, dt)
        return float(wrong.double().mean()) > share

    assert not seen(want.value, 0.0)
    lost = w2.clone()
    lost[..., 127] = 0.0
    assert seen(paths.experts(x, w1, lost, tw, ids, act, dt, narrow).value, 0.25)
    lost = w1.clone()
    lost[:, :I, 127] = 0.0  # of the gates
    assert seen(paths.experts(x, lost, w2, tw, ids, act, dt, narrow).value, 0.25)
    lost = w1.clone()
    lost[:, 7] = lost[:, 8]  # the gates of one feature
    assert seen(paths.experts(x, lost, w2, tw, ids, act, dt, narrow).value, 0.01)
    other = "gelu" if act != "gelu" else "silu"
    if act == "silu":
        assert seen(paths.experts(x, w1, w2, tw, ids, other, dt, narrow).value, 0.25)
    moved = tw.roll(1, 0)
    assert seen(paths.experts(x, w1, w2, moved, ids, act, dt, narrow).value, 0.5)


def test_codes_between_the_ends_of_an_interval():
    """through(): of values known exactly the codes are those of the format's own oracle."""
    import _fp8_ref as ref

    gen = torch.Generator().manual_seed(3)
    h = torch.randn(9, 300, generator=gen).double()
    got = paths.through(h, torch.zeros_like(h))
    want = torch.from_numpy(ref.through(h.numpy()))
    assert bool(((got.value - want).abs() <= got.off + 2.0 ** -24 * want.abs()).all())
    # a value on the border between two codes may become either
    h = torch.tensor([[448.0, 17.0, 16.0, 0.0]]).double()
    got = paths.through(h, torch.zeros_like(h))
    assert float(got.off[0, 1]) >= 1.0 and float(got.off[0, 2]) < 0.01 and float(got.off[0, 3]) < 0.01
