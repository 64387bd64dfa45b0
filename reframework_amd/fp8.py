"""Rows and weights in 8 bits (e4m3) with one fp32 scale per block of 128, and their products.

  * rows (``Fp8Rows``): a scale per 128 consecutive values of a row;
  * weights (``Fp8Weight``, ``Fp8Experts``): a scale per 128 x 128 block.

Blocks start at multiples of 128; the last of a row or matrix may be smaller. With m a
block's largest finite magnitude, at least 448 * 2^-126, its scale is m / 448 and a value's
code is value * 448 / m, rounded to nearest even; infinities and NaN become NaN. Weights
are laid out once, block by block in the order in which the kernels load them.

The reference has neither; its quantised experts are int8 with one scale per tensor, on the
host (reframework/moe/fused.py:140-197).
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from reframework_amd import _capi
from reframework_amd.grad import once_differentiable, records

BLOCK = 128
E4M3 = torch.float8_e4m3fn


def blocks(n: int) -> int:
    return -(-n // BLOCK)


def padded(n: int) -> int:
    return blocks(n) * BLOCK


def _require_gpu(t: torch.Tensor, what: str) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{what} must be on a ROCm GPU; it is on {t.device}")


class Fp8Rows:
    """[M, size] values in 8 bits: ``codes`` (float8_e4m3fn, [M, size]) times ``scales``
    (float32, [M, ceil(size / 128)]) of their blocks. The kernels read the padded codes behind
    them, whose rows hold whole blocks: what lies past ``size`` must be zeros (a NaN
    there would reach the results)."""

    __slots__ = ("padded_codes", "scales", "size")

    def __init__(self, padded_codes: torch.Tensor, scales: torch.Tensor, size: int) -> None:
        if size <= 0:
            raise ValueError(f"8-bit rows of size {size}")
        M, Kp = padded_codes.shape[0], padded(size)
        if padded_codes.dtype != E4M3 or tuple(padded_codes.shape) != (M, Kp) or \
                not padded_codes.is_contiguous():
            raise ValueError(f"codes must be contiguous float8_e4m3fn [M, {Kp}]")
        if scales.dtype != torch.float32 or tuple(scales.shape) != (M, blocks(size)) or \
                not scales.is_contiguous() or scales.device != padded_codes.device:
            raise ValueError(f"scales must be contiguous float32 [{M}, {blocks(size)}] on the "
                             "codes' device")
        self.padded_codes, self.scales, self.size = padded_codes, scales, size

    @classmethod
    def empty(cls, M: int, size: int, device: torch.device) -> "Fp8Rows":
        """Rows for a kernel to fill (the padding included)."""
        q = cls.__new__(cls)
        n = blocks(size)
        q.padded_codes = torch.empty(M, n * BLOCK, dtype=E4M3, device=device)
        q.scales = torch.empty(M, n, dtype=torch.float32, device=device)
        q.size = size
        return q

    @property
    def codes(self) -> torch.Tensor:
        c = self.padded_codes
        return c if c.shape[1] == self.size else c.narrow(1, 0, self.size)

    @property
    def device(self) -> torch.device:
        return self.padded_codes.device

    def __len__(self) -> int:
        return self.padded_codes.shape[0]

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        v = self.padded_codes.float().reshape(len(self), -1, BLOCK) * self.scales[..., None]
        return v.reshape(len(self), -1)[:, :self.size].to(dtype)


def _quantize(x: torch.Tensor) -> Fp8Rows:
    q = Fp8Rows.empty(x.shape[0], x.shape[1], x.device)
    _capi.fp8_quantize(x, q.padded_codes, q.scales)
    return q


def quantize_fp8(x: torch.Tensor) -> Fp8Rows:
    """``x`` [..., K] (float32, bfloat16 or float16 on the GPU) as 8-bit rows, one per row of
    ``x``, without gradients."""
    _require_gpu(x, "x")
    _capi.dtype_code(x.dtype)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"8-bit rows of {tuple(x.shape)}")
    return _quantize(x.detach().reshape(-1, x.shape[-1]).contiguous())


def _check_codes(codes: torch.Tensor, scales: torch.Tensor, name: str, scale_rows=None) -> None:
    if codes.dim() != 3 or scales.dim() != 3:
        raise ValueError(f"{name}: codes and scales are stacked [E, rows, ...]")
    if codes.dtype not in (E4M3, torch.uint8) or scales.dtype != torch.float32:
        raise ValueError(f"{name}: codes are float8_e4m3fn and scales float32, not {codes.dtype} / "
                         f"{scales.dtype}")
    E, N, K = codes.shape
    n = blocks(N) if scale_rows is None else scale_rows
    if 0 in codes.shape or tuple(scales.shape) != (E, n, blocks(K)) or \
            scales.device != codes.device:
        raise ValueError(f"{name}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do "
                         "not belong together")
    if E > _capi.MAX_EXPERTS:
        raise ValueError(f"{name}: {E} matrices, at most {_capi.MAX_EXPERTS}")
    _require_gpu(codes, name)


CELL = BLOCK * BLOCK


def _cells(E: int, N: int, K: int, device: torch.device) -> torch.Tensor:
    """Room for E matrices [N, K] as cells of 128 x 128 codes (include/moe355.h)."""
    return torch.empty(E, blocks(N), blocks(K), CELL, dtype=torch.uint8, device=device)


def _pack(codes: torch.Tensor) -> torch.Tensor:
    """[E, N, K] codes as cells."""
    codes = codes.detach().view(torch.uint8).contiguous()
    cells = _cells(*codes.shape, codes.device)
    for c, m in zip(codes, cells):
        _capi.fp8_pack(c, m)
    return cells


def _unpack(cells: torch.Tensor, N: int, K: int) -> torch.Tensor:
    """The bytes [E, N, K] of matrices of cells."""
    E, n, k, _ = cells.shape
    # a cell: tile of 16 rows, half of 64 columns, 16 columns, row, column
    c = cells.reshape(E, n, k, 8, 2, 4, 16, 16).permute(0, 1, 3, 6, 2, 4, 5, 7)
    return c.reshape(E, n * BLOCK, k * BLOCK)[:, :N, :K]


class _Codes(torch.nn.Module):
    """Holds codes and scales as buffers that a change of the module's dtype leaves alone (the
    scales by their bits)."""

    def _hold(self, name: str, cells: torch.Tensor, scales: torch.Tensor) -> None:
        self.register_buffer(name, cells)
        self.register_buffer(name + "_scales", scales.detach().contiguous().view(torch.int32))

    def _held(self, name: str) -> Tuple[torch.Tensor, torch.Tensor]:
        """(cells, scales) as the kernels take them."""
        b = self._buffers
        return b[name], b[name + "_scales"]

    @property
    def nbytes(self) -> int:
        return sum(b.numel() * b.element_size() for b in self._buffers.values())


def _dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp32 [E, N, K] of codes and the scales of their blocks."""
    E, N, K = codes.shape
    s = scales.repeat_interleave(BLOCK, 1)[:, :N].repeat_interleave(BLOCK, 2)[..., :K]
    return codes.float() * s


def _quantize_matrices(w: Sequence[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """(cells, scales) of [N, K] matrices."""
    N, K = w[0].shape
    cells = _cells(len(w), N, K, w[0].device)
    scales = torch.empty(len(w), blocks(N), blocks(K), dtype=torch.float32, device=w[0].device)
    for m, c, s in zip(w, cells, scales):
        _capi.fp8_quantize_weight(m.detach().contiguous(), c, s)
    return cells, scales


class Fp8Weight(_Codes):
    """One or several matrices [N, K] in 8 bits, as matmul_fp8 multiplies by them.
    ``transposed``: it also holds the matrices transposed, which gradients of the rows are
    multiplied by. The weights themselves are constants."""

    def __init__(self, cells: torch.Tensor, scales: torch.Tensor, rows: int, columns: int,
                 transposed: bool = False) -> None:
        super().__init__()
        self.num_matrices, self.rows, self.columns = cells.shape[0], rows, columns
        self._hold("w", cells, scales)
        if transposed:
            self._hold("wt", _pack(_unpack(cells, rows, columns).transpose(1, 2)),
                       scales.transpose(1, 2))

    @classmethod
    def quantize(cls, w: torch.Tensor, transposed: bool = False) -> "Fp8Weight":
        """From weights [N, K] or [E, N, K] (float32, bfloat16 or float16 on the GPU)."""
        _require_gpu(w, "w")
        _capi.dtype_code(w.dtype)
        if w.dim() not in (2, 3) or 0 in w.shape:
            raise ValueError(f"weights are [N, K] or [E, N, K], not {tuple(w.shape)}")
        m = list(w) if w.dim() == 3 else [w]
        if len(m) > _capi.MAX_EXPERTS:
            raise ValueError(f"{len(m)} matrices, at most {_capi.MAX_EXPERTS}")
        return cls(*_quantize_matrices(m), *w.shape[-2:], transposed)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor,
                   transposed: bool = False) -> "Fp8Weight":
        """From a checkpoint's codes (float8_e4m3fn, or their bytes) [N, K] or [E, N, K] and
        scales float32 [(E,) ceil(N/128), ceil(K/128)], on the GPU; both are copied."""
        if codes.dim() == 2 and scales.dim() == 2:
            codes, scales = codes[None], scales[None]
        _check_codes(codes, scales, "weights")
        return cls(_pack(codes), scales.clone(), *codes.shape[1:], transposed)

    @property
    def device(self) -> torch.device:
        return self._buffers["w"].device

    @property
    def has_transposed(self) -> bool:
        return "wt" in self._buffers

    def codes(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """(codes [E, N, K], scales) as from_codes takes them, copies."""
        cells, scales = self._held("w")
        return _unpack(cells, self.rows, self.columns).view(E4M3), scales.view(torch.float32).clone()

    def dequantize(self) -> torch.Tensor:
        """[E, N, K] in fp32."""
        return _dequantize(*self.codes())


class Fp8Experts(_Codes):
    """The expert matrices of one layer in 8 bits: w1 [E, 2I, H] (gate rows first) and w2
    [E, H, I]. H and I are multiples of 16. The blocks of w1's gate and up halves start at the
    first row of each."""

    def __init__(self, w1: Tuple[torch.Tensor, torch.Tensor], w2: Tuple[torch.Tensor, torch.Tensor],
                 hidden_size: int, intermediate_size: int) -> None:
        super().__init__()
        self.num_experts = w2[0].shape[0]
        self.hidden_size, self.intermediate_size = hidden_size, intermediate_size
        self._hold("w1", *(t.reshape(self.num_experts, -1, *t.shape[2:]) for t in w1))
        self._hold("w2", *w2)

    @staticmethod
    def _check_sizes(w1: torch.Tensor, w2: torch.Tensor) -> Tuple[int, int, int]:
        E, I2, H = w1.shape
        if I2 % 2 or tuple(w2.shape) != (E, H, I2 // 2) or w2.device != w1.device:
            raise ValueError(f"w1 {tuple(w1.shape)} on {w1.device} and w2 {tuple(w2.shape)} on "
                             f"{w2.device} are not [E, 2I, H] and [E, H, I]")
        if H % 16 or I2 % 32 or 0 in w1.shape:
            raise ValueError(f"8-bit experts need H {H} and I {I2 // 2} to be multiples of 16")
        if E > _capi.MAX_EXPERTS:
            raise ValueError(f"{E} experts, at most {_capi.MAX_EXPERTS}")
        return E, I2 // 2, H

    @classmethod
    def quantize(cls, w1: torch.Tensor, w2: torch.Tensor) -> "Fp8Experts":
        """From stacked banks [E, 2I, H] / [E, H, I] in float32, bfloat16 or float16 on the
        GPU."""
        for name, w in (("w1", w1), ("w2", w2)):
            if w.dim() != 3:
                raise ValueError(f"{name}: expected a stacked [E, rows, columns] bank, got "
                                 f"{tuple(w.shape)}")
            _require_gpu(w, name)
            _capi.dtype_code(w.dtype)
        _, I, H = cls._check_sizes(w1, w2)
        return cls(_quantize_matrices([h for m in w1 for h in (m[:I], m[I:])]),
                   _quantize_matrices(list(w2)), H, I)

    @classmethod
    def from_codes(cls, w1: torch.Tensor, w1_scales: torch.Tensor, w2: torch.Tensor,
                   w2_scales: torch.Tensor) -> "Fp8Experts":
        """From a checkpoint's codes (float8_e4m3fn, or their bytes) [E, 2I, H] and [E, H, I]
        with float32 scales [E, 2 ceil(I/128), ceil(H/128)] (gate blocks first) and
        [E, ceil(H/128), ceil(I/128)], on the GPU; all are copied."""
        if w1.dim() != 3 or w2.dim() != 3:
            raise ValueError("codes are stacked [E, rows, columns]")
        E, I, H = cls._check_sizes(w1, w2)
        _check_codes(w1, w1_scales, "w1", 2 * blocks(I))
        _check_codes(w2, w2_scales, "w2")
        halves = w1.detach().contiguous().reshape(2 * E, I, H)
        return cls((_pack(halves), w1_scales.clone().reshape(2 * E, blocks(I), -1)),
                   (_pack(w2), w2_scales.clone()), H, I)

    @property
    def device(self) -> torch.device:
        return self._buffers["w1"].device

    def codes(self, name: str) -> Tuple[torch.Tensor, torch.Tensor]:
        """``"w1"`` or ``"w2"`` as from_codes takes it: (codes, scales), copies."""
        cells, scales = self._held(name)
        H, I = self.hidden_size, self.intermediate_size
        if name == "w2":
            return _unpack(cells, H, I).view(E4M3), scales.view(torch.float32).clone()
        halves = cells.reshape(2 * self.num_experts, blocks(I), *cells.shape[2:])
        codes = _unpack(halves, I, H).reshape(self.num_experts, 2 * I, H)
        return codes.view(E4M3), scales.view(torch.float32).clone()

    def dequantize(self, name: str) -> torch.Tensor:
        """``"w1"`` [E, 2I, H] or ``"w2"`` [E, H, I] in fp32."""
        codes, scales = self.codes(name)
        if name == "w2":
            return _dequantize(codes, scales)
        I = self.intermediate_size
        return _dequantize(codes.reshape(-1, I, codes.shape[2]), scales.reshape(-1, blocks(I), scales.shape[2])
                           ).reshape(codes.shape)


def _matmul(q: Fp8Rows, w: Tuple[torch.Tensor, torch.Tensor], N: int,
            offsets: Optional[torch.Tensor], dtype: torch.dtype) -> torch.Tensor:
    cells, scales = w
    out = torch.empty(len(q), N, dtype=dtype, device=q.device)
    _capi.fp8_matmul(q.padded_codes, q.scales, cells, scales, offsets, cells.shape[0], q.size, out)
    return out


class _MatmulFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, dtype):
        ctx.columns, ctx.dtype = weight.columns, x.dtype
        ctx.save_for_backward(*weight._held("wt"), offsets)
        return _matmul(_quantize(x), weight._held("w"), weight.rows, offsets, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        cells, scales, offsets = ctx.saved_tensors
        dx = _matmul(_quantize(dout.contiguous()), (cells, scales), ctx.columns, offsets, ctx.dtype)
        return dx, None, None, None


def matmul_fp8(x: Union[torch.Tensor, Fp8Rows], weight: Fp8Weight,
               offsets: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``x`` [M, K] times the matrices of ``weight``, transposed: [M, N] in ``out_dtype``
    (the type of ``x``; bfloat16 for Fp8Rows). Rows offsets[e] .. offsets[e + 1] - 1 are
    multiplied by matrix e (``offsets`` [E + 1] ascending within [0, M], on the GPU, as
    permute_tokens gives them; rows of no matrix become zeros); without offsets all rows by the
    only one.

    ``x`` is brought to 8 bits first unless it is Fp8Rows. Steps of 128 columns are summed by
    the matrix cores, which for 16-bit results keep about 13 bits below a step's largest
    product (float32 results have exact products, summed in fp32), then scaled and added in
    fp32. Where ``x`` records gradients, its gradient is the same product of
    the result's, brought to 8 bits, with the transposed matrices, which ``weight`` has to
    hold; the rounding to 8 bits counts as the identity. Tangents are refused."""
    if isinstance(x, Fp8Rows):
        M, K, dev = len(x), x.size, x.device
        dtype = out_dtype or torch.bfloat16
    else:
        _require_gpu(x, "x")
        if x.dim() != 2:
            raise ValueError(f"x is [M, K], not {tuple(x.shape)}")
        _capi.dtype_code(x.dtype)
        (M, K), dev = x.shape, x.device
        dtype = out_dtype or x.dtype
    _capi.dtype_code(dtype)
    if K != weight.columns:
        raise ValueError(f"x has {K} columns, the matrices {weight.columns}")
    if weight.device != dev:
        raise ValueError(f"weights on {weight.device} must be on the rows' {dev}")
    E = weight.num_matrices
    if offsets is None:
        if E != 1:
            raise ValueError(f"{E} matrices need offsets")
    else:
        if offsets.device != dev or tuple(offsets.shape) != (E + 1,):
            raise ValueError(f"offsets {tuple(offsets.shape)} on {offsets.device} are not [{E + 1}] "
                             f"on {dev}")
        if offsets.dtype != torch.int32:
            if offsets.dtype != torch.int64:
                raise TypeError(f"offsets are int32 or int64, not {offsets.dtype}")
            offsets = offsets.int()
        offsets = offsets.contiguous()
    if isinstance(x, Fp8Rows):
        return _matmul(x, weight._held("w"), weight.rows, offsets, dtype)
    x = x.contiguous()
    if records(x):
        if not weight.has_transposed:
            raise RuntimeError("gradients need weights that hold the transposed matrices "
                               "(transposed=True)")
        return _MatmulFn.apply(x, weight, offsets, dtype)
    return _matmul(_quantize(x), weight._held("w"), weight.rows, offsets, dtype)


__all__ = ["Fp8Rows", "Fp8Weight", "Fp8Experts", "quantize_fp8", "matmul_fp8"]
