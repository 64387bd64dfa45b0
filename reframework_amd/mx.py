"""Rows in 8 bits and expert weights in 4 bits, with power-of-two scales.

Both formats hold one scale per 32 consecutive values of a row, a byte ``b`` that
stands for ``2^(b - 127)`` (torch.float8_e8m0fnu):

  * rows (``Mxfp8Rows``): e4m3 codes. The scale is the smallest that brings the
    block's largest finite magnitude to at most 448, so nothing is clipped;
    infinities and NaN become NaN.
  * expert weights (``Mxfp4Experts``): e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
    their negatives), two per byte with the even column in the low half. They are
    laid out once, in the order in which the kernels stream them.

The reference has neither; its quantised experts are int8 with one scale per
tensor, on the host (reframework/moe/fused.py:140-197).
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from reframework_amd import _capi

BLOCK = 32    # values per scale
STEP = 128    # columns per matrix instruction: rows are padded to whole steps
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

Bank = Union[torch.Tensor, Sequence[torch.Tensor]]


def padded(n: int) -> int:
    return -(-n // STEP) * STEP


def _require_gpu(t: torch.Tensor, what: str) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{what} must be on a ROCm GPU; it is on {t.device}")


class Mxfp8Rows:
    """[T, size] values in 8 bits: ``codes`` (float8_e4m3fn, [T, size]) times
    ``scales`` (float8_e8m0fnu, [T, size / 32]). The kernels read the padded tensors
    behind them, whose rows hold whole steps of 128 values: what lies past ``size`` must be
    zeros (a NaN there would reach the results)."""

    __slots__ = ("padded_codes", "padded_scales", "size")

    def __init__(self, padded_codes: torch.Tensor, padded_scales: torch.Tensor, size: int) -> None:
        if size <= 0 or size % BLOCK:
            raise ValueError(f"8-bit rows need a size of whole blocks of {BLOCK}, not {size}")
        T, Hp = padded_codes.shape[0], padded(size)
        if padded_codes.dtype != torch.float8_e4m3fn or tuple(padded_codes.shape) != (T, Hp) or \
                not padded_codes.is_contiguous():
            raise ValueError(f"codes must be contiguous float8_e4m3fn [T, {Hp}]")
        if padded_scales.dtype != torch.float8_e8m0fnu or \
                tuple(padded_scales.shape) != (T, Hp // BLOCK) or \
                not padded_scales.is_contiguous() or padded_scales.device != padded_codes.device:
            raise ValueError(f"scales must be contiguous float8_e8m0fnu [{T}, {Hp // BLOCK}] on the "
                             "codes' device")
        self.padded_codes, self.padded_scales, self.size = padded_codes, padded_scales, size

    @classmethod
    def empty(cls, T: int, size: int, device: torch.device) -> "Mxfp8Rows":
        """Rows for a kernel to fill (the padding included)."""
        q = cls.__new__(cls)
        Hp = padded(size)
        q.padded_codes = torch.empty(T, Hp, dtype=torch.float8_e4m3fn, device=device)
        q.padded_scales = torch.empty(T, Hp // BLOCK, dtype=torch.float8_e8m0fnu, device=device)
        q.size = size
        return q

    @property
    def codes(self) -> torch.Tensor:
        c = self.padded_codes
        return c if c.shape[1] == self.size else c.narrow(1, 0, self.size)

    @property
    def scales(self) -> torch.Tensor:
        s = self.padded_scales
        return s if s.shape[1] * BLOCK == self.size else s.narrow(1, 0, self.size // BLOCK)

    @property
    def device(self) -> torch.device:
        return self.padded_codes.device

    def __len__(self) -> int:
        return self.padded_codes.shape[0]

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values, exact in fp32 and bf16 (above their subnormals)."""
        f = _pow2(self.scales.view(torch.uint8))
        v = self.codes.float().reshape(len(self), -1, BLOCK) * f[..., None]
        return v.reshape(len(self), self.size).to(dtype)


def _pow2(b: torch.Tensor) -> torch.Tensor:
    """2^(b - 127) in fp32 of scale bytes; 255 gives NaN."""
    bits = b.int() << 23
    bits = torch.where(b == 0, torch.full_like(bits, 1 << 22), bits)
    bits = torch.where(b == 255, torch.full_like(bits, 0x7FC00000), bits)
    return bits.view(torch.float32)


def quantize_mxfp8(x: torch.Tensor) -> Mxfp8Rows:
    """``x`` [..., H] (float32, bfloat16 or float16 on the GPU, H a multiple of 32) as
    8-bit rows, one per row of ``x``."""
    _require_gpu(x, "x")
    _capi.dtype_code(x.dtype)
    H = x.shape[-1]
    if H == 0 or H % BLOCK:
        raise ValueError(f"8-bit rows need a size of whole blocks of {BLOCK}, not {H}")
    x2 = _aligned(x.detach().reshape(-1, H).contiguous())
    q = Mxfp8Rows.empty(x2.shape[0], H, x2.device)
    _capi.mx_quantize(x2, q.padded_codes, q.padded_scales)
    return q


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` where it starts on 16 bytes, else a copy that does."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


class Mxfp4Experts(torch.nn.Module):
    """The expert matrices of one layer in 4 bits: w1 [E, 2I, H] (gate rows first) and
    w2 [E, H, I], laid out for the kernels. H and I are multiples of 32; 4.25 bits per
    weight where both are multiples of 128 (the layout is padded to those)."""

    def __init__(self, num_experts: int, hidden_size: int, intermediate_size: int,
                 device: Optional[torch.device] = None) -> None:
        super().__init__()
        if not 1 <= num_experts <= _capi.MAX_EXPERTS:
            raise ValueError(f"num_experts {num_experts} outside [1, {_capi.MAX_EXPERTS}]")
        for n in (hidden_size, intermediate_size):
            if n <= 0 or n % BLOCK:
                raise ValueError(f"4-bit experts need sizes of whole blocks of {BLOCK}: "
                                 f"H {hidden_size}, I {intermediate_size}")
        self.num_experts = num_experts
        self.hidden_size = hidden_size
        self.intermediate_size = intermediate_size
        for name, rows, cols, gate_up in self._matrices():
            codes, scales = _capi.mx_matrix_bytes(rows, cols, gate_up)
            for suffix, n in (("", codes), ("_scales", scales)):
                self.register_buffer(name + suffix, torch.empty((num_experts, n), dtype=torch.uint8,
                                                                device=device))

    def _matrices(self):
        H, I = self.hidden_size, self.intermediate_size
        return (("w1", 2 * I, H, True), ("w2", H, I, False))

    @property
    def device(self) -> torch.device:
        return self._buffers["w1"].device

    @property
    def nbytes(self) -> int:
        return sum(b.numel() for b in self._buffers.values())

    def _fill(self, name: str, e: int, src: torch.Tensor, scales: Optional[torch.Tensor]) -> None:
        rows, cols, gate_up = {n: m for n, *m in self._matrices()}[name]
        _capi.mx_pack(src, scales, rows, cols, gate_up, self._buffers[name][e],
                      self._buffers[name + "_scales"][e])

    @classmethod
    def quantize(cls, w1: Bank, w2: Bank) -> "Mxfp4Experts":
        """From weights: stacked banks [E, 2I, H] / [E, H, I] or lists of per-expert
        matrices, in float32, bfloat16 or float16 on the GPU. Each block of 32 gets the
        smallest scale that keeps it within 6; a block with an infinity or NaN
        becomes NaN."""
        m1, m2 = list(w1), list(w2)
        if not m1 or len(m1) != len(m2):
            raise ValueError("w1 and w2 hold no experts or different expert counts")
        if m1[0].dim() != 2 or m1[0].shape[0] % 2:
            raise ValueError(f"w1 matrices are [2I, H], not {tuple(m1[0].shape)}")
        (I2, H), dev = m1[0].shape, m1[0].device
        for name, mats, shape in (("w1", m1, (I2, H)), ("w2", m2, (H, I2 // 2))):
            for m in mats:
                _require_gpu(m, name)
                _capi.dtype_code(m.dtype)
                if tuple(m.shape) != shape or m.device != dev:
                    raise ValueError(f"{name}: expected {shape} on {dev}, got {tuple(m.shape)} on "
                                     f"{m.device}")
        out = cls(len(m1), H, I2 // 2, device=dev)
        for e, (a, b) in enumerate(zip(m1, m2)):
            out._fill("w1", e, a.detach().contiguous(), None)
            out._fill("w2", e, b.detach().contiguous(), None)
        return out

    @classmethod
    def from_codes(cls, w1: torch.Tensor, w1_scales: torch.Tensor, w2: torch.Tensor,
                   w2_scales: torch.Tensor) -> "Mxfp4Experts":
        """From a checkpoint's codes: uint8 [E, 2I, H/2] and [E, H, I/2] with scale bytes
        [E, 2I, H/32] and [E, H, I/32], on the GPU."""
        for name, c, s in (("w1", w1, w1_scales), ("w2", w2, w2_scales)):
            if c.dim() != 3 or s.dim() != 3:
                raise ValueError(f"{name}: codes and scales are stacked [E, rows, ...]")
            if c.element_size() != 1 or s.element_size() != 1 or c.dtype == torch.bool:
                raise ValueError(f"{name}: codes and scales are bytes, not {c.dtype} / {s.dtype}")
            if tuple(s.shape) != (c.shape[0], c.shape[1], c.shape[2] * 2 // BLOCK) or \
                    c.shape[2] * 2 % BLOCK or s.device != c.device or c.device != w1.device:
                raise ValueError(f"{name}: codes {tuple(c.shape)} and scales {tuple(s.shape)} do "
                                 "not belong together")
            _require_gpu(c, name)
        E, I2, H = w1.shape[0], w1.shape[1], w1.shape[2] * 2
        if I2 % 2 or tuple(w2.shape) != (E, H, I2 // 4):
            raise ValueError(f"w1 codes {tuple(w1.shape)} and w2 codes {tuple(w2.shape)} are not "
                             "[E, 2I, H/2] and [E, H, I/2]")
        out = cls(E, H, I2 // 2, device=w1.device)
        for name, c, s in (("w1", w1, w1_scales), ("w2", w2, w2_scales)):
            c, s = c.contiguous().view(torch.uint8), s.contiguous().view(torch.uint8)
            for e in range(E):
                out._fill(name, e, _aligned(c[e]), s[e])
        return out

    def codes(self, name: str) -> Tuple[torch.Tensor, torch.Tensor]:
        """``"w1"`` or ``"w2"`` as from_codes takes it: (codes, scale bytes)."""
        rows, cols, gate_up = {n: m for n, *m in self._matrices()}[name]
        E, cols_p = self.num_experts, padded(cols)
        rows_p = 2 * padded(rows // 2) if gate_up else padded(rows)
        # codes [supergroup, step, group, block, row, 16 bytes]; scales [supergroup,
        # step, block, row, group]; rows of a supergroup are (group, row)
        c = self._buffers[name].reshape(E, rows_p // 64, cols_p // STEP, 4, 4, 16, 16)
        s = self._buffers[name + "_scales"].reshape(E, rows_p // 64, cols_p // STEP, 4, 16, 4)
        c = c.permute(0, 1, 3, 5, 2, 4, 6).reshape(E, rows_p, cols_p // 2)
        s = s.permute(0, 1, 5, 4, 2, 3).reshape(E, rows_p, cols_p // BLOCK)
        if gate_up:  # per block: (four feature runs of 4), gate / up, (feature 8 q + 4 j + i)
            c, s = (t.reshape(E, rows_p // 64, 2, 2, 4, 4, -1).permute(0, 3, 1, 4, 2, 5, 6)
                    .reshape(E, 2, rows_p // 2, -1)[:, :, :rows // 2].reshape(E, rows, -1)
                    for t in (c, s))
        return (c[:, :rows, :cols // 2].contiguous(), s[:, :rows, :cols // BLOCK].contiguous())

    def dequantize(self, name: str) -> torch.Tensor:
        """``"w1"`` [E, 2I, H] or ``"w2"`` [E, H, I] in fp32, exactly."""
        c, s = self.codes(name)
        lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=c.device)
        v = lut[torch.stack([c & 15, c >> 4], -1).int()].reshape(*s.shape, BLOCK)
        return (v * _pow2(s)[..., None]).reshape(c.shape[0], c.shape[1], -1)


__all__ = ["Mxfp8Rows", "Mxfp4Experts", "quantize_mxfp8"]
