"""Sizes that reach every kernel of the 8-bit products and experts, and the experts' result with
what each of its elements may be off by (not collected: no test_ prefix).

tests/test_fp8_paths.py asks the library's own rule which kernels these sizes take; the GPU tests
run them."""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from reframework_amd.fp8 import BLOCK, blocks

# (M, N, K, E) of a product; its gradient is one of (M, K, N, E).
PRODUCTS = [
    (40, 130, 200, 8),                     # streamed
    (160, 1100, 1300, 8),                  # 32 rows, both ways
    (896, 700, 650, 64),                   # 64 rows, both ways
    (1024, 700, 2120, 128),                # 64 rows of few rows per matrix
    (400, 1100, 1300, 8),                  # 128 rows, both ways
    (1100, 1290, 2050, 9),                 # the same, nearly whole tiles
    (3000, 6500, 300, 4),                  # 256 rows
    (2600, 6500, 2100, 4)]                 # 256 rows, the last round's items cut

# (T, H, I, E, K, activation) of an expert call.
EXPERTS = [
    (9, 272, 144, 8, 2, "gelu"),           # all streamed
    (128, 2048, 384, 128, 8, "silu"),      # gate|up on 64 rows of few rows per expert
    (448, 768, 272, 64, 2, "gelu_tanh"),   # 64 rows
    (80, 1040, 528, 8, 2, "silu"),         # 32 rows
    (120, 1040, 528, 8, 2, "gelu"),        # 128 rows, exact
    (240, 1040, 528, 8, 2, "silu"),        # 128 rows, gate|up of bf16 scaled
    (1024, 256, 3296, 4, 2, "gelu"),       # gate|up on 256 rows, whole
    (1792, 4112, 2064, 4, 2, "gelu_tanh"),  # 256 rows, in parts, bf16 slots in 16 bits
    (3000, 5136, 144, 4, 1, "silu")]       # down on 256 rows, whole, to fp32 slots


class Bounded(NamedTuple):
    """Values and what each may be off by."""
    value: torch.Tensor
    off: torch.Tensor


def rne_e4m3(q: torch.Tensor) -> torch.Tensor:
    """Values of the codes nearest to 0 <= q, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(q.clamp(min=2.0 ** -6))) - 3)
    return torch.round(q / step) * step


def _blocks_of(v: torch.Tensor) -> torch.Tensor:
    """[M, K] as [M, blocks, 128], padded with zeros."""
    return torch.nn.functional.pad(v, (0, -v.shape[1] % BLOCK)).reshape(v.shape[0], -1, BLOCK)


def activate(name: str, g: torch.Tensor):
    """(act(g), what its argument of a sigmoid is), in 64 bits."""
    if name == "silu":
        return g * torch.sigmoid(g), g
    if name == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g / math.sqrt(2.0))), torch.zeros_like(g)
    z = 2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)
    return g * torch.sigmoid(z), z


def through(h: torch.Tensor, off: torch.Tensor) -> Bounded:
    """h as 8 bits hold it, h being known to ``off``: a code is one of those between the ends of
    its quotient's interval (another factor of 1 +- 2^-21 for the quotient's own roundings), its
    scale off by the largest value's share and two roundings."""
    a, o = _blocks_of(h.abs()), _blocks_of(off)
    most = a.amax(-1, keepdim=True).clamp(min=448.0 * 2.0 ** -126)
    # whichever element comes out largest, it does so within the largest `off`
    e = o.amax(-1, keepdim=True)
    code = rne_e4m3(a * 448.0 / most)
    lo = rne_e4m3((a - o).clamp(min=0.0) * 448.0 / (most + e) * (1.0 - 2.0 ** -21))
    hi = rne_e4m3((a + o) * 448.0 / (most - e).clamp(min=448.0 * 2.0 ** -126) * (1.0 + 2.0 ** -21))
    hi = hi.clamp(max=448.0)
    scale = most / 448.0
    share = e / most + 2.0 ** -23
    d = torch.maximum(hi - code, code - lo) * scale * (1.0 + share) + code * scale * share
    M, K = h.shape
    return Bounded((code * scale).reshape(M, -1)[:, :K] * torch.sign(h), d.reshape(M, -1)[:, :K])


def products_off(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """What x @ w.T may be off by on the matrix cores: of each step of 128 columns 2^-10 of its
    largest product (measured: 2^-11), which is at most the product of the largest factors, and
    2^-22 of the magnitudes per step for scaling and adding in fp32."""
    xm, wm = (_blocks_of(v.abs()).amax(-1) for v in (x, w))
    n = xm.shape[1]
    return 2.0 ** -10 * (xm @ wm.t().contiguous()) + \
        2.0 ** -22 * (n + 1) * (x.abs() @ w.abs().t().contiguous())


def half_step(v: torch.Tensor, dt: torch.dtype) -> torch.Tensor:
    f = torch.finfo(dt)
    return (v.abs() * (f.eps / 2)).clamp(min=f.tiny * f.eps / 2)


def experts(x, w1, w2, tw, ids, name: str, dt: torch.dtype, narrow: bool) -> Bounded:
    """[T, H] in 64 bits of x [T, H] as 8 bits hold it, whose products with w1 [E, 2I, H] are
    exact. Of an activation the argument is rounded a few times (a factor exp(+-|z| 2^-22) of the
    sigmoid), the rest to 2^-21 of |gate * up|. ``narrow``: slots wait in f16 with a power of two
    per 64 columns, half a step of 11 bits, or of what lies 2^28 below the largest."""
    T, K = ids.shape
    out, off = torch.zeros_like(x), torch.zeros_like(x)
    for e in range(w1.shape[0]):
        t, k = torch.nonzero(ids == e, as_tuple=True)
        if not t.numel():
            continue
        gate, up = (x[t] @ w1[e].t().contiguous()).chunk(2, -1)
        act, z = activate(name, gate)
        h = act * up
        q = through(h, (gate * up).abs() * 2.0 ** -21 + h.abs() * 2.0 ** -22 * (z.abs() + 8.0))
        y = q.value @ w2[e].t().contiguous()
        yo = products_off(q.value.abs() + q.off, w2[e]) + q.off @ w2[e].abs().t().contiguous()
        if narrow:
            yo = yo * (1.0 + 2.0 ** -10) + y.abs() * 2.0 ** -11 + 2.0 ** -38 * y.abs().amax(-1, keepdim=True)
        w = tw[t, k, None].double()
        out.index_add_(0, t, y * w)
        # and the sum of K products in fp32
        off.index_add_(0, t, w.abs() * (yo + 2.0 ** -22 * K * y.abs()))
    return Bounded(out, off * (1.0 + 2.0 ** -8) + half_step(out, dt))


def whole(shape, gen, dev, most: int = 2) -> torch.Tensor:
    return torch.randint(-most, most + 1, shape, generator=gen, device=dev).float()


def powers(shape, gen, dev, low: int, high: int) -> torch.Tensor:
    return torch.exp2(torch.randint(low, high + 1, shape, generator=gen, device=dev).float())


def expert_codes(H: int, I: int, E: int, gen, dev):
    """(w1, w1_scales, w2, w2_scales) as Fp8Experts.from_codes takes them: w1 of whole numbers up
    to 2 and scales of powers of two, w2 of any codes and scales."""
    e4m3 = torch.float8_e4m3fn
    size = round(math.log2(math.sqrt(H)))  # gates of magnitudes around 1 to 8
    w1 = whole((E, 2 * I, H), gen, dev).to(e4m3)
    s1 = powers((E, 2 * blocks(I), blocks(H)), gen, dev, -1 - size, 1 - size)
    w2 = (torch.randn(E, H, I, generator=gen, device=dev) * 64.0).to(e4m3)
    s2 = (torch.rand(E, blocks(H), blocks(I), generator=gen, device=dev) + 0.5) * (I ** -0.5 / 64.0)
    return w1, s1, w2, s2
