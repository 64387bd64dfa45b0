"""RMSNorm and LayerNorm on libmoe355 (one HIP kernel per call, GPU tensors only).

Same class surface as the reference's RMSNorm (reframework/layers/norm.py:17-53):
``RMSNorm(size, eps, bias=False)`` with ``weight`` (and ``bias``) parameters,
``forward``, ``forward_inplace`` and ``forward_add_residual``. The norm is
computed in fp32 (``x / sqrt(mean(x^2) + eps) * weight (+ bias)``) and rounded
once to the input dtype; ``forward_add_residual`` first forms
``residual = x + residual`` in the input dtype and returns
``(rmsnorm(residual), residual)``. Parameters may be stored in fp32 or the
activation dtype. ``forward_mxfp8`` and ``forward_add_residual_mxfp8`` also leave
the normed rows in 8 bits (mx.Mxfp8Rows), for expert products that take them.

``LayerNorm`` has the same surface (the reference has none) and gradients: with respect to
its inputs and parameters wherever autograd records. Tangents (forward-mode derivatives) are
refused.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from reframework_amd import _capi
from reframework_amd.grad import has_tangent, once_differentiable, records
from reframework_amd.layers.base import BaseOP
from reframework_amd.mx import BLOCK, Mxfp8Rows


def _written(x: torch.Tensor) -> None:
    """Tells autograd, which does not see the kernels' writes, that ``x`` was overwritten: a recorded
    call that keeps it for its gradient then raises instead of taking the new values."""
    torch.autograd.graph.increment_version(x)


class RMSNorm(BaseOP):
    def __init__(self, size: int, eps: float, bias: bool = False) -> None:
        super().__init__()
        self.eps = eps
        self.size = size
        self.weight = nn.Parameter(torch.ones(size))
        self.bias = nn.Parameter(torch.zeros(size)) if bias else None

    def _params(self, x: torch.Tensor) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        if x.device.type != "cuda":
            raise RuntimeError(f"reframework_amd RMSNorm runs on a ROCm GPU; input is on {x.device}")
        w = self.weight.detach()
        b = None if self.bias is None else self.bias.detach()
        if w.device != x.device:
            raise RuntimeError("RMSNorm parameters must be on the input's device")
        return w.contiguous(), (None if b is None else b.to(w.dtype).contiguous())

    def _run(self, x: torch.Tensor, residual: Optional[torch.Tensor], out: torch.Tensor,
             residual_out: Optional[torch.Tensor]) -> None:
        w, b = self._params(x)
        _capi.add_rmsnorm(x.reshape(-1, self.size), None if residual is None else
                          residual.reshape(-1, self.size),
                          None if residual_out is None else residual_out.reshape(-1, self.size),
                          w, b, self.eps, out.reshape(-1, self.size))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x = x.contiguous()
        out = torch.empty_like(x)
        self._run(x, None, out, None)
        return out

    def forward_inplace(self, x: torch.Tensor) -> None:
        if not x.is_contiguous():
            x.copy_(self.forward(x))
            return
        self._run(x, None, x, None)
        _written(x)

    def forward_add_residual(self, x: torch.Tensor,
                             residual: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Fused ``residual = x + residual; x = rmsnorm(residual)``; returns
        (normed, new_residual). The inputs are not modified."""
        x = x.contiguous()
        residual = residual.to(x.dtype).contiguous()
        new_res = torch.empty_like(x)
        out = torch.empty_like(x)
        self._run(x, residual, out, new_res)
        return out, new_res

    def _run_mxfp8(self, x: torch.Tensor, residual: Optional[torch.Tensor], out: torch.Tensor,
                   residual_out: Optional[torch.Tensor]) -> Mxfp8Rows:
        H = self.size
        if x.shape[-1] != H:
            raise ValueError(f"input rows of {x.shape[-1]} do not match the norm's size {H}")
        if H % BLOCK:
            raise ValueError(f"8-bit rows need a size of whole blocks of {BLOCK}, not {H}")
        w, b = self.weight, self.bias
        dev = x.get_device()
        if not x.is_cuda or w.get_device() != dev or not w.is_contiguous() or (
                b is not None and (b.dtype != w.dtype or b.get_device() != dev or
                                   not b.is_contiguous())):
            w, b = self._params(x)
        T = x.numel() // H
        q = Mxfp8Rows.empty(T, H, x.device)
        _capi.add_rmsnorm_mxfp8(T, H, x, residual, residual_out, w, b, self.eps, out,
                                q.padded_codes, q.padded_scales)
        return q

    def forward_mxfp8(self, x: torch.Tensor) -> Tuple[torch.Tensor, Mxfp8Rows]:
        """(normed, normed in 8 bits), in one launch; the latter is
        ``quantize_mxfp8(normed)`` bit for bit, one row per row of ``x``."""
        x = x.contiguous()
        out = torch.empty_like(x)
        return out, self._run_mxfp8(x, None, out, None)

    def forward_add_residual_mxfp8(
            self, x: torch.Tensor,
            residual: torch.Tensor) -> Tuple[torch.Tensor, Mxfp8Rows, torch.Tensor]:
        """forward_add_residual that also returns the normed rows in 8 bits:
        (normed, normed in 8 bits, new_residual), in one launch."""
        x = x.contiguous()
        if residual.dtype != x.dtype:
            residual = residual.to(x.dtype)
        residual = residual.contiguous()
        if residual.shape != x.shape or residual.get_device() != x.get_device():
            raise ValueError(f"residual {tuple(residual.shape)} on {residual.device} does not match "
                             f"x {tuple(x.shape)} on {x.device}")
        new_res = torch.empty_like(x)
        out = torch.empty_like(x)
        q = self._run_mxfp8(x, residual, out, new_res)
        return out, q, new_res


class _LayerNormFn(torch.autograd.Function):
    """(normed, x + residual), or (normed,) without a residual."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        ctx.set_materialize_grads(False)
        H = x.shape[-1]
        T = x.numel() // H
        stats = torch.empty(2, T, dtype=torch.float32, device=x.device)
        out = torch.empty_like(x)
        r = x if residual is None else torch.empty_like(x)
        _capi.layer_norm(T, H, x, residual, None if residual is None else r, weight, bias, eps, out,
                         stats)
        ctx.save_for_backward(r, weight, stats)
        ctx.has_bias = bias is not None
        return out if residual is None else (out, r)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dres=None):
        r, weight, stats = ctx.saved_tensors
        H = r.shape[-1]
        T = r.numel() // H
        need_x, need_res, need_w, need_b = ctx.needs_input_grad[:4]
        if dy is None:  # only the sum went on
            return (dres if need_x else None, dres if need_res else None,
                    torch.zeros_like(weight) if need_w else None,
                    torch.zeros_like(weight) if need_b else None, None)
        dx = torch.empty_like(r) if need_x or need_res else None
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty_like(weight) if need_b else None
        if T == 0:
            return (dx if need_x else None, dx if need_res else None, None if dw is None else
                    dw.zero_(), None if db is None else db.zero_(), None)
        _capi.layer_norm_bwd(T, H, dy.contiguous(), None if dres is None else dres.contiguous(), r,
                             weight, stats, dx, dw, db)
        return (dx if need_x else None, dx if need_res else None, dw, db, None)


class LayerNorm(BaseOP):
    """``(r - mean(r)) / sqrt(var(r) + eps) * weight (+ bias)`` over the last dimension of
    ``size``, in fp32 and rounded once to the input's type (float32, bfloat16, float16; up
    to 16384 wide, 8192 in float32). Parameters may be of another of these types than the
    inputs; their gradients are summed in fp32 over all rows, in a fixed order, and rounded
    once."""

    def __init__(self, size: int, eps: float, bias: bool = True) -> None:
        super().__init__()
        self.eps = eps
        self.size = size
        self.weight = nn.Parameter(torch.ones(size))
        self.bias = nn.Parameter(torch.zeros(size)) if bias else None

    def _check(self, x: torch.Tensor) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        w, b = self.weight, self.bias
        dev = x.get_device()
        if not x.is_cuda:
            raise RuntimeError(f"reframework_amd LayerNorm runs on a ROCm GPU; input is on {x.device}")
        if x.shape[-1] != self.size:
            raise ValueError(f"input rows of {x.shape[-1]} do not match the norm's size {self.size}")
        if w.get_device() != dev or (b is not None and b.get_device() != dev):
            raise RuntimeError("LayerNorm parameters must be on the input's device")
        if not w.is_contiguous():
            w = w.contiguous()
        if b is not None:
            if b.dtype != w.dtype:
                b = b.to(w.dtype)
            if not b.is_contiguous():
                b = b.contiguous()
        return w, b

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        w, b = self._check(x)
        x = x.contiguous()
        if records(x, w, b):
            return _LayerNormFn.apply(x, None, w, b, self.eps)
        out = torch.empty_like(x)
        _capi.layer_norm(x.numel() // self.size, self.size, x, None, None, w, b, self.eps, out)
        return out

    def forward_inplace(self, x: torch.Tensor) -> None:
        """``x`` is overwritten by its norm; no gradients are recorded through this one."""
        w, b = self._check(x)
        if torch.is_grad_enabled() and x.requires_grad or has_tangent(x, w, b):
            raise RuntimeError("forward_inplace overwrites what a derivative needs; use forward")
        if not x.is_contiguous():
            with torch.no_grad():
                x.copy_(self.forward(x))
            return
        _capi.layer_norm(x.numel() // self.size, self.size, x, None, None, w, b, self.eps, x)
        _written(x)

    def forward_add_residual(self, x: torch.Tensor,
                             residual: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """``residual = x + residual; x = layernorm(residual)`` in one launch; returns
        (normed, new_residual). The inputs are not modified."""
        w, b = self._check(x)
        if residual.shape != x.shape or residual.get_device() != x.get_device():
            raise ValueError(f"residual {tuple(residual.shape)} on {residual.device} does not match "
                             f"x {tuple(x.shape)} on {x.device}")
        x = x.contiguous()
        if residual.dtype != x.dtype:
            residual = residual.to(x.dtype)
        residual = residual.contiguous()
        if records(x, residual, w, b):
            return _LayerNormFn.apply(x, residual, w, b, self.eps)
        out, r = torch.empty_like(x), torch.empty_like(x)
        _capi.layer_norm(x.numel() // self.size, self.size, x, residual, r, w, b, self.eps, out)
        return out, r


__all__ = ["RMSNorm", "LayerNorm"]
