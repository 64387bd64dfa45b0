"""Tokens in the order of their experts and back, with gradients.

The reference gathers and adds per expert in Python (``x[tok]`` and ``out.index_add_(0, tok,
y * w)``, reframework/moe/fused.py:78-86). Here the order of all slots is found at once, and
the token rows move in one launch each way:

  * ``token_order(topk_ids, num_experts)``: which row each routed slot gets.
  * ``permute_tokens(hidden_states, topk_ids, num_experts)`` -> (rows [M*K, H], order):
    experts ascending, slots ascending within one; ``order.offsets`` are the experts' ends
    as matmul_fp8 takes them. Rows behind the last slot of an expert are zeros.
  * ``combine_tokens(rows, order, topk_weights)`` -> [M, H]: the weighted sum of each
    token's rows, in fp32 and slot order.

Both are differentiable where autograd records, the latter in the weights too; sums run in a
fixed order, so equal calls give equal results. Tangents (forward-mode derivatives) are refused.
"""

from __future__ import annotations

from typing import Tuple

import torch

from reframework_amd import _capi
from reframework_amd.grad import once_differentiable, records


class TokenOrder:
    """The order of [M, K] routed slots by expert (int32, on the tokens' GPU):

      offsets      [E + 1]  rows of expert e are offsets[e] .. offsets[e + 1] - 1
      slot_to_row  [M, K]   row of a slot, -1 where its id lies outside the experts
      row_src      [M * K]  token of a row, for rows below offsets[E]
    """

    __slots__ = ("offsets", "slot_to_row", "row_src", "num_experts")

    def __init__(self, offsets: torch.Tensor, slot_to_row: torch.Tensor, row_src: torch.Tensor,
                 num_experts: int) -> None:
        if slot_to_row.dim() != 2 or tuple(offsets.shape) != (num_experts + 1,) or \
                tuple(row_src.shape) != (slot_to_row.numel(),):
            raise ValueError(f"offsets {tuple(offsets.shape)}, slot_to_row {tuple(slot_to_row.shape)} and "
                             f"row_src {tuple(row_src.shape)} are not [{num_experts + 1}], [M, K], [M*K]")
        for t in (offsets, slot_to_row, row_src):
            if t.dtype != torch.int32 or not t.is_contiguous() or t.device != slot_to_row.device:
                raise ValueError("an order is contiguous int32, on one device")
        self.offsets, self.slot_to_row, self.row_src = offsets, slot_to_row, row_src
        self.num_experts = num_experts

    @classmethod
    def _empty(cls, M: int, K: int, num_experts: int, device: torch.device) -> "TokenOrder":
        """For a kernel to fill; without slots (M 0) as it is."""
        order = cls.__new__(cls)
        new = torch.zeros if M == 0 else torch.empty
        order.offsets = new(num_experts + 1, dtype=torch.int32, device=device)
        order.slot_to_row = torch.empty(M, K, dtype=torch.int32, device=device)
        order.row_src = torch.empty(M * K, dtype=torch.int32, device=device)
        order.num_experts = num_experts
        return order

    @property
    def device(self) -> torch.device:
        return self.slot_to_row.device


def token_order(topk_ids: torch.Tensor, num_experts: int) -> TokenOrder:
    """The order of the routed slots ``topk_ids`` [M, K] by expert."""
    if topk_ids.device.type != "cuda":
        raise RuntimeError(f"topk_ids must be on a ROCm GPU; they are on {topk_ids.device}")
    if topk_ids.dim() != 2 or topk_ids.shape[1] == 0:
        raise ValueError(f"topk_ids are [M, K], not {tuple(topk_ids.shape)}")
    if not 1 <= num_experts <= _capi.MAX_EXPERTS:
        raise ValueError(f"num_experts {num_experts} outside [1, {_capi.MAX_EXPERTS}]")
    if topk_ids.is_floating_point() or topk_ids.dtype == torch.bool:
        raise TypeError(f"topk_ids are whole numbers, not {topk_ids.dtype}")
    M, K = topk_ids.shape
    ids = topk_ids if topk_ids.dtype in (torch.int32, torch.int64) else topk_ids.long()
    order = TokenOrder._empty(M, K, num_experts, topk_ids.device)
    if M:
        _capi.token_order(ids.contiguous(), M, K, num_experts, order.offsets, order.slot_to_row,
                          order.row_src)
    return order


def _permute(x: torch.Tensor, order: TokenOrder) -> torch.Tensor:
    rows = torch.empty(order.row_src.shape[0], x.shape[1], dtype=x.dtype, device=x.device)
    _capi.permute_rows(x, order.offsets, order.slot_to_row, order.num_experts, rows)
    return rows


class _PermuteFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order):
        ctx.save_for_backward(order.slot_to_row)
        return _permute(x, order)

    @staticmethod
    @once_differentiable
    def backward(ctx, drows):
        slot_to_row, = ctx.saved_tensors
        dx = torch.empty(slot_to_row.shape[0], drows.shape[1], dtype=drows.dtype,
                         device=drows.device)
        _capi.combine_rows(drows.contiguous(), None, slot_to_row, dx)
        return dx, None


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, order):
        out = torch.empty(weights.shape[0], rows.shape[1], dtype=rows.dtype, device=rows.device)
        _capi.combine_rows(rows, weights, order.slot_to_row, out)
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, weights, order.offsets,
                              order.slot_to_row)
        ctx.num_experts = order.num_experts
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        rows, weights, offsets, slot_to_row = ctx.saved_tensors
        dout = dout.contiguous()
        drows = dw = None
        if ctx.needs_input_grad[0]:
            drows = torch.empty(slot_to_row.numel(), dout.shape[1], dtype=dout.dtype,
                                device=dout.device)
        if ctx.needs_input_grad[1]:
            dw = torch.empty_like(weights)
        _capi.combine_rows_bwd(dout, rows, weights, offsets, slot_to_row, ctx.num_experts, drows,
                               dw)
        return drows, dw, None


def permute_tokens(hidden_states: torch.Tensor, topk_ids: torch.Tensor,
                   num_experts: int) -> Tuple[torch.Tensor, TokenOrder]:
    """``hidden_states`` [M, H] (float32, bfloat16, float16) as one row per routed slot
    [M*K, H], in the order of the experts, and that order."""
    x = hidden_states
    if x.device.type != "cuda":
        raise RuntimeError(f"hidden_states must be on a ROCm GPU; they are on {x.device}")
    if x.dim() != 2 or x.shape[1] == 0 or topk_ids.dim() != 2 or topk_ids.shape[0] != x.shape[0]:
        raise ValueError(f"hidden_states {tuple(x.shape)} and topk_ids {tuple(topk_ids.shape)} are "
                         "not [M, H] and [M, K]")
    if topk_ids.device != x.device:
        raise ValueError(f"topk_ids on {topk_ids.device} must be on the tokens' {x.device}")
    _capi.dtype_code(x.dtype)
    order = token_order(topk_ids, num_experts)
    x = x.contiguous()
    if records(x):
        return _PermuteFn.apply(x, order), order
    return _permute(x, order), order


def combine_tokens(rows: torch.Tensor, order: TokenOrder,
                   topk_weights: torch.Tensor) -> torch.Tensor:
    """[M, H]: per token the sum of its slots' ``rows`` [M*K, H] times ``topk_weights`` [M, K]
    (fp32; others are converted), in the rows' type. Slots without a row add nothing and get a
    gradient of 0."""
    if rows.device.type != "cuda":
        raise RuntimeError(f"rows must be on a ROCm GPU; they are on {rows.device}")
    R, (M, K) = order.row_src.shape[0], order.slot_to_row.shape
    if rows.dim() != 2 or rows.shape[0] != R or rows.shape[1] == 0:
        raise ValueError(f"rows {tuple(rows.shape)} are not [{R}, H]")
    if tuple(topk_weights.shape) != (M, K):
        raise ValueError(f"topk_weights {tuple(topk_weights.shape)} are not [{M}, {K}]")
    if rows.device != order.device or topk_weights.device != order.device:
        raise ValueError(f"rows on {rows.device} and topk_weights on {topk_weights.device} must be "
                         f"on the order's {order.device}")
    _capi.dtype_code(rows.dtype)
    rows = rows.contiguous()
    w = topk_weights if topk_weights.dtype == torch.float32 else topk_weights.float()
    w = w.contiguous()
    if records(rows, w):
        return _CombineFn.apply(rows, w, order)
    out = torch.empty(M, rows.shape[1], dtype=rows.dtype, device=rows.device)
    _capi.combine_rows(rows, w, order.slot_to_row, out)
    return out


__all__ = ["TokenOrder", "token_order", "permute_tokens", "combine_tokens"]
