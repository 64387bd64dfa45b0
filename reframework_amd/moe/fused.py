"""Routing and grouped expert compute on libmoe355 (MI355X HIP kernels).

Same call surface as the reference's module (reframework/moe/fused.py):

  * ``torch_fused_topk(gating_output, topk, renormalize)`` -> (weights fp32
    [M,K], ids int64 [M,K]): softmax over experts, the K largest, optional
    renormalisation (fused.py:32-46).
  * ``fused_experts(hidden_states, w1, w2, topk_weights, topk_ids, activation)``
    -> [M,H] in the dtype of ``hidden_states`` (fused.py:49-87).
  * ``fused_experts_masked(..., active, activation)``: only the slots where
    ``active`` is set (the GPU half of the CPU/GPU split, fused.py:90-137).
  * ``fused_experts_cpu_int8(hidden_states, w1q, w2q, scales1, scales2,
    topk_weights, topk_ids, active, activation)`` -> fp32 [M,H] on the host:
    the split's CPU half on int8 banks (fused.py:140-197), run by
    libmoe355_host.
  * ``grouped_topk(gating_output, topk, renormalize, ...)``: routing with softmax or
    sigmoid scores, a bias for the choice and groups of experts (not in the reference).
  * ``fused_experts_mxfp4(hidden_states, experts, ...)``: fused_experts on 4-bit
    weights and 8-bit rows (mx.Mxfp4Experts, mx.Mxfp8Rows; not in the reference).
  * ``fused_experts_fp8(hidden_states, experts, ...)``: fused_experts on 8-bit weights and
    rows with a scale per block of 128 (fp8.Fp8Experts, fp8.Fp8Rows; not in the reference).

The reference loops over experts in Python (gather, two torch.mm, activation,
scale, index_add_). Here one C call runs the whole thing on the current HIP
stream: a stable counting sort of the routed slots, the grouped gate|up GEMM
with the activation fused, the grouped down GEMM, and a deterministic
weighted combine. Expert banks are passed as a table of per-expert device
pointers, so ``w1``/``w2`` may be a stacked ``[E,2I,H]`` tensor or a list of
per-expert tensors (the offload cache's HBM slots) without a stacking copy.
Exact ties in top-k go to the lower expert id.
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from reframework_amd import _capi
from reframework_amd.fp8 import Fp8Experts, Fp8Rows, _quantize
from reframework_amd.layers import activation_code
from reframework_amd.mx import Mxfp4Experts, Mxfp8Rows, _aligned, quantize_mxfp8

Bank = Union[torch.Tensor, Sequence[torch.Tensor]]


def require_gpu(t: torch.Tensor, what: str = "input") -> None:
    """The MoE kernels run only on a ROCm GPU; anything else is an error."""
    if t.device.type != "cuda":
        raise RuntimeError(
            f"reframework_amd MoE kernels run on a ROCm GPU; {what} is on {t.device}"
        )


def bank_pointers(bank: Bank) -> Tuple[List[int], Tuple[int, ...]]:
    """Per-expert device pointers of a stacked bank or a list of expert tensors.

    Returns (pointers, matrix shape). Every expert matrix must be contiguous.
    """
    if isinstance(bank, torch.Tensor):
        if bank.dim() != 3:
            raise ValueError(f"expected a stacked [E, rows, cols] bank, got {tuple(bank.shape)}")
        if not bank.is_contiguous():
            raise ValueError("stacked expert bank must be contiguous")
        base = bank.data_ptr()
        step = bank.stride(0) * bank.element_size()
        return [base + e * step for e in range(bank.shape[0])], tuple(bank.shape[1:])
    mats = list(bank)
    if not mats:
        raise ValueError("empty expert bank")
    shape = tuple(mats[0].shape)
    for m in mats:
        if tuple(m.shape) != shape or not m.is_contiguous():
            raise ValueError("per-expert tensors must be contiguous and share one shape")
    return [m.data_ptr() for m in mats], shape


def _bank_dtype(bank: Bank) -> torch.dtype:
    return bank.dtype if isinstance(bank, torch.Tensor) else bank[0].dtype


def torch_fused_topk(
    gating_output: torch.Tensor,
    topk: int,
    renormalize: bool,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Softmax over all experts, keep the top-k, renormalise the kept weights."""
    require_gpu(gating_output, "gating_output")
    E = gating_output.shape[-1]
    logits = gating_output.reshape(-1, E).float().contiguous()
    T = logits.shape[0]
    w = torch.empty((T, topk), dtype=torch.float32, device=logits.device)
    ids = torch.empty((T, topk), dtype=torch.int32, device=logits.device)
    _capi.topk_from_logits(logits, topk, renormalize, w, ids)
    shape = tuple(gating_output.shape[:-1]) + (topk,)
    return w.reshape(shape), ids.long().reshape(shape)


def grouped_topk(
    gating_output: torch.Tensor,  # [..., E] router logits
    topk: int,
    renormalize: bool = True,
    scoring: str = "softmax",
    bias: Optional[torch.Tensor] = None,  # [E], for the choice alone
    num_groups: int = 1,
    topk_groups: int = 1,
    group_score: str = "max",
    scale: float = 1.0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Routing by groups: (weights fp32 [..., topk], ids int64 [..., topk]).

    Scores ``s`` are the ``"softmax"`` or ``"sigmoid"`` of the logits, ``c = s + bias``
    the choice. The ``num_groups`` runs of consecutive experts are scored by their best
    ``c`` (``"max"``) or the sum of their best two (``"top2"``); the ``topk_groups`` best
    groups stay, and of their experts the ``topk`` of largest ``c`` are chosen, in
    descending order. The weights are their ``s``, over their sum if ``renormalize``,
    times ``scale``. The ids are those of 64-bit arithmetic on the fp32 logits and bias, or
    of the logits themselves where only their order counts (no bias, groups by their best).
    Ties, also of scores that 64 bits do not tell apart, go to the lower group and the
    lower expert; a NaN ranks last. At most 64 groups and a topk of 64."""
    require_gpu(gating_output, "gating_output")
    shape = gating_output.shape
    logits = gating_output
    if logits.dim() != 2:
        logits = logits.reshape(-1, shape[-1])
    if logits.dtype != torch.float32:
        logits = logits.float()
    logits = logits.contiguous()
    T, device = logits.shape[0], logits.device
    w = torch.empty(T, topk, dtype=torch.float32, device=device)
    ids = torch.empty(T, topk, dtype=torch.int64, device=device)
    run_grouped_topk(logits, bias, renormalize, scoring, num_groups, topk_groups, group_score,
                     scale, topk, w, ids)
    if len(shape) == 2:
        return w, ids
    return w.reshape(shape[:-1] + (topk,)), ids.reshape(shape[:-1] + (topk,))


def run_grouped_topk(logits: torch.Tensor, bias: Optional[torch.Tensor], renormalize: bool,
                     scoring: str, num_groups: int, topk_groups: int, group_score: str,
                     scale: float, topk: int, w: torch.Tensor, ids: torch.Tensor) -> None:
    """grouped_topk of contiguous fp32 ``logits`` [T, E] into the first ``topk`` columns
    of ``w`` and ``ids`` [T, ld] (fp32; int32 or int64)."""
    sc, gs = _capi.SCORE_CODES.get(scoring), _capi.GROUP_SCORE_CODES.get(group_score)
    if sc is None:
        raise ValueError(f"unknown scoring {scoring!r}; known: {tuple(_capi.SCORE_CODES)}")
    if gs is None:
        raise ValueError(f"unknown group score {group_score!r}; known: "
                         f"{tuple(_capi.GROUP_SCORE_CODES)}")
    if bias is not None:
        if bias.numel() != logits.shape[1] or bias.device != logits.device:
            raise ValueError(f"bias {tuple(bias.shape)} on {bias.device} does not match "
                             f"{logits.shape[1]} experts on {logits.device}")
        if bias.dtype != torch.float32:
            bias = bias.float()
        bias = bias.contiguous()
    _capi.grouped_topk(logits, bias, topk, sc, num_groups, topk_groups, gs, renormalize, scale, w,
                       ids)


def run_experts(
    x: torch.Tensor,
    w1_ptrs: Sequence[int],
    w2_ptrs: Sequence[int],
    intermediate_size: int,
    topk_weights: torch.Tensor,
    topk_ids: torch.Tensor,
    act: int,
    out: Optional[torch.Tensor] = None,
    expert_map: Optional[Sequence[int]] = None,
    accumulate_f32: bool = False,
    path: int = -1,
) -> torch.Tensor:
    """One libmoe355 fused_experts call on the current stream.

    x [T,H] contiguous in the bank dtype; topk_weights [T,K] fp32; topk_ids
    [T,K] int32/int64; ids are local bank rows unless ``expert_map`` renames
    them. With ``accumulate_f32`` the result is added to the fp32 ``out``.
    ``path`` forces a kernel family (``_capi.PATH_*``); -1 lets the library
    choose from the shape.
    """
    T, H = x.shape
    if out is None:
        out = torch.empty((T, H), dtype=torch.float32 if accumulate_f32 else x.dtype,
                          device=x.device)
    if T == 0:
        return out
    K = topk_ids.shape[1]
    if len(w1_ptrs) < K:
        # Fewer bank rows than slots per token (a streaming chunk or a
        # truncated offload step holding fewer experts than top_k, the other
        # slots renamed to -1): the library plans for at least K experts, so
        # the tables are padded with a row no slot maps to.
        if not len(w1_ptrs):
            raise ValueError("run_experts needs at least one expert")
        w1_ptrs = list(w1_ptrs) + [w1_ptrs[-1]] * (K - len(w1_ptrs))
        w2_ptrs = list(w2_ptrs) + [w2_ptrs[-1]] * (K - len(w2_ptrs))
    stream = _capi.stream_handle(x.device)
    plan = _capi.make_plan(T, H, intermediate_size, len(w1_ptrs), topk_ids.shape[1],
                           _capi.dtype_code(x.dtype), path)
    ws = _capi.workspaces.get(x.device, stream, plan.workspace_bytes)
    _capi.fused_experts(x, w1_ptrs, w2_ptrs, intermediate_size, topk_weights, topk_ids, act, out,
                        ws, expert_map=expert_map, accumulate_f32=accumulate_f32, stream=stream,
                        plan=plan)
    return out


def fused_experts(
    hidden_states: torch.Tensor,
    w1: Bank,  # [E, 2I, H] gate|up rows (gate first), or E tensors [2I, H]
    w2: Bank,  # [E, H, I], or E tensors [H, I]
    topk_weights: torch.Tensor,  # [M, K] fp32
    topk_ids: torch.Tensor,  # [M, K] int64 (or int32)
    activation: str = "silu",
) -> torch.Tensor:
    """Run the routed experts and return the summed output ``[M, H]``."""
    act = activation_code(activation)
    require_gpu(hidden_states, "hidden_states")
    w1_ptrs, s1 = bank_pointers(w1)
    w2_ptrs, s2 = bank_pointers(w2)
    if len(w1_ptrs) != len(w2_ptrs):
        raise ValueError("w1 and w2 hold different expert counts")
    M, H = hidden_states.shape
    I = s1[0] // 2
    if s1 != (2 * I, H) or s2 != (H, I):
        raise ValueError(f"bank shapes {s1} / {s2} do not match hidden size {H}")
    dtype = _bank_dtype(w1)
    x = hidden_states.to(dtype).contiguous()
    ids = topk_ids if topk_ids.dtype in (torch.int32, torch.int64) else topk_ids.long()
    ids = ids.reshape(M, -1).contiguous()
    w = topk_weights.reshape(M, -1).float().contiguous()
    out = run_experts(x, w1_ptrs, w2_ptrs, I, w, ids, act)
    return out if out.dtype == hidden_states.dtype else out.to(hidden_states.dtype)


def fused_experts_mxfp4(
    hidden_states: Union[torch.Tensor, Mxfp8Rows],  # [M, H]
    experts: Mxfp4Experts,
    topk_weights: torch.Tensor,  # [M, K] fp32
    topk_ids: torch.Tensor,  # [M, K] int64 (or int32)
    activation: str = "silu",
    out: Optional[torch.Tensor] = None,
    accumulate_f32: bool = False,
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """fused_experts on 4-bit weights: ``[M, H]``, summed over the K slots.

    Tokens go through gate|up in 8 bits (``hidden_states`` quantised first unless they
    are Mxfp8Rows, e.g. of RMSNorm.forward_add_residual_mxfp8) and the gated activation
    through down in 8 bits. The result is of ``out_dtype``: the tokens' type, bfloat16
    for Mxfp8Rows. Products are exact, their sums and the results of the slots fp32, but
    for a bfloat16 result of more than 12 rows per expert: that takes the scaled MFMA, whose
    products keep about 14 bits below the largest they are added to, and without
    ``accumulate_f32`` the results of its slots may be rounded to 11 bits (of values down to
    2^-28 of the largest of 64 columns) before they are added (``out_dtype=torch.float32``
    keeps bfloat16 tokens from that too). Slots whose id lies outside the experts or
    whose weight is 0 add nothing.
    With ``accumulate_f32`` the result is added to the fp32 ``out``."""
    act = activation_code(activation)
    if isinstance(hidden_states, Mxfp8Rows):
        x, x_scales = hidden_states.padded_codes, hidden_states.padded_scales
        M, H = x.shape[0], hidden_states.size
        dtype = out_dtype or torch.bfloat16
    else:
        require_gpu(hidden_states, "hidden_states")
        if hidden_states.dim() != 2:
            raise ValueError(f"hidden_states are [M, H], not {tuple(hidden_states.shape)}")
        M, H = hidden_states.shape
        dtype = out_dtype or hidden_states.dtype
        if dtype == hidden_states.dtype:
            x, x_scales = _aligned(hidden_states.contiguous()), None
        else:  # the call quantises tokens of its results' type
            _capi.dtype_code(dtype)
            rows = quantize_mxfp8(hidden_states)
            x, x_scales = rows.padded_codes, rows.padded_scales
    code = _capi.dtype_code(dtype)
    dev = x.device
    if H != experts.hidden_size:
        raise ValueError(f"hidden size {H} does not match the experts' {experts.hidden_size}")
    b = experts._buffers
    w1 = b["w1"]
    if w1.device != dev or topk_weights.device != dev or topk_ids.device != dev:
        raise ValueError(f"experts on {w1.device}, weights on {topk_weights.device} and ids on "
                         f"{topk_ids.device} must be on the tokens' {dev}")
    if topk_ids.dim() != 2 or topk_ids.shape[0] != M or topk_weights.shape != topk_ids.shape:
        raise ValueError(f"topk_ids {tuple(topk_ids.shape)} and topk_weights "
                         f"{tuple(topk_weights.shape)} are not [{M}, K]")
    out_type = torch.float32 if accumulate_f32 else dtype
    if out is None:
        if accumulate_f32:
            raise ValueError("accumulate_f32 adds to an fp32 out")
        out = torch.empty(M, H, dtype=out_type, device=dev)
    elif out.dtype != out_type or tuple(out.shape) != (M, H) or out.device != dev or \
            not out.is_contiguous():
        raise ValueError(f"out must be contiguous {out_type} [{M}, {H}] on {dev}")
    if M == 0:
        return out
    ids = topk_ids if topk_ids.dtype in (torch.int32, torch.int64) else topk_ids.long()
    w = topk_weights if topk_weights.dtype == torch.float32 else topk_weights.float()
    E, I, K = experts.num_experts, experts.intermediate_size, topk_ids.shape[1]
    # From the caching allocator on the current stream, not from a buffer that calls
    # share: captured graphs then have workspaces of their own.
    ws = torch.empty(_capi.mx_workspace_bytes(M, H, I, E, K, code, dev, accumulate_f32),
                     dtype=torch.uint8, device=dev)
    _capi.mx_fused_experts(x, x_scales, M, H, I, E, K, w1, b["w1_scales"], b["w2"],
                           b["w2_scales"], w.contiguous(), ids.contiguous(), code, act, out,
                           accumulate_f32, ws)
    return out


def fused_experts_fp8(
    hidden_states: Union[torch.Tensor, Fp8Rows],  # [M, H]
    experts: Fp8Experts,
    topk_weights: torch.Tensor,  # [M, K] fp32
    topk_ids: torch.Tensor,  # [M, K] int64 (or int32)
    activation: str = "silu",
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """fused_experts on 8-bit weights: ``[M, H]``, summed over the K slots.

    Tokens go through gate|up in 8 bits (``hidden_states`` quantised first unless they are
    Fp8Rows) and the gated activation, not rounded in between, through down in 8 bits. The result
    is of ``out_dtype``: the tokens' type, bfloat16 for Fp8Rows. Sums are those of matmul_fp8, with
    exact products in gate|up for float16 results and calls of few tokens too; the slots' results
    are added in fp32 and rounded once, but those of large bfloat16 calls wait for that in 16 bits
    (f16 with a power of two per 64 columns). Slots whose id lies outside the experts or whose
    weight is 0 add nothing. No gradients are recorded."""
    act = activation_code(activation)
    if isinstance(hidden_states, Fp8Rows):
        x, x_scales = hidden_states.padded_codes, hidden_states.scales
        M, H = x.shape[0], hidden_states.size
        dtype = out_dtype or torch.bfloat16
        _capi.dtype_code(dtype)
    else:
        require_gpu(hidden_states, "hidden_states")
        if hidden_states.dim() != 2:
            raise ValueError(f"hidden_states are [M, H], not {tuple(hidden_states.shape)}")
        M, H = hidden_states.shape
        _capi.dtype_code(hidden_states.dtype)
        dtype = out_dtype or hidden_states.dtype
        _capi.dtype_code(dtype)
        x, x_scales = hidden_states.detach().contiguous(), None
        if H != experts.hidden_size:
            raise ValueError(f"hidden size {H} does not match the experts' {experts.hidden_size}")
        if dtype == hidden_states.dtype:
            x = _aligned(x)
        else:  # the call quantises tokens of its results' type
            rows = _quantize(x)
            x, x_scales = rows.padded_codes, rows.scales
    dev = x.device
    if H != experts.hidden_size:
        raise ValueError(f"hidden size {H} does not match the experts' {experts.hidden_size}")
    if experts.device != dev or topk_weights.device != dev or topk_ids.device != dev:
        raise ValueError(f"experts on {experts.device}, weights on {topk_weights.device} and ids on "
                         f"{topk_ids.device} must be on the tokens' {dev}")
    if topk_ids.dim() != 2 or topk_ids.shape[0] != M or topk_weights.shape != topk_ids.shape:
        raise ValueError(f"topk_ids {tuple(topk_ids.shape)} and topk_weights "
                         f"{tuple(topk_weights.shape)} are not [{M}, K]")
    out = torch.empty(M, H, dtype=dtype, device=dev)
    if M == 0:
        return out
    ids = topk_ids if topk_ids.dtype in (torch.int32, torch.int64) else topk_ids.long()
    w = topk_weights.detach()
    w = w if w.dtype == torch.float32 else w.float()
    _capi.fp8_fused_experts(x, x_scales, M, H, experts.intermediate_size, experts.num_experts,
                            topk_ids.shape[1], *experts._held("w1"), *experts._held("w2"),
                            w.contiguous(), ids.contiguous(), act, out)
    return out


def fused_experts_masked(
    hidden_states: torch.Tensor,
    w1: Bank,  # [E, 2I, H], or E tensors [2I, H]: the experts this device holds
    w2: Bank,  # [E, H, I], or E tensors [H, I]
    topk_weights: torch.Tensor,  # [M, K] fp32
    topk_ids: torch.Tensor,  # [M, K], local rows of w1/w2
    active: torch.Tensor,  # [M, K] bool: the slots computed here
    activation: str = "silu",
) -> torch.Tensor:
    """fused_experts over the slots where ``active`` is set; the others add
    nothing (fused_experts_masked, reframework/moe/fused.py:90-137). The
    inactive slots are renamed to -1, which the permute drops, so the masked
    call is the same single library call. Each slot's output goes to its own
    token; the reference's ``arange(M).repeat(K)`` gives flat slot t*K+k the
    token (t*K+k) % M instead, which differs from it whenever K > 1 and a
    slot other than each token's first is active."""
    require_gpu(hidden_states, "hidden_states")
    M = hidden_states.shape[0]
    ids = topk_ids.reshape(M, -1)
    on = active.reshape(M, -1).to(device=ids.device, dtype=torch.bool)
    if on.shape != ids.shape:
        raise ValueError(f"active {tuple(active.shape)} does not match topk_ids {tuple(topk_ids.shape)}")
    ids = torch.where(on, ids, torch.full_like(ids, -1))
    return fused_experts(hidden_states, w1, w2, topk_weights, ids, activation)


def _group_active_slots(ids: np.ndarray, weights: np.ndarray, on: np.ndarray, E: int):
    """(experts used ascending, slot offsets, slot tokens, slot weights) of the
    active slots of [M, K] routing: per expert, its slots in ascending (t, k)
    order, each on its own token t."""
    K = ids.shape[1]
    flat = np.where(on, ids, -1).reshape(-1)
    chosen = flat[on.reshape(-1)]
    if chosen.size and (chosen.min() < 0 or chosen.max() >= E):
        raise ValueError(f"an active slot routes outside the {E} experts of the int8 bank")
    order = np.argsort(flat, kind="stable")
    order = order[flat[order] >= 0]
    used, counts = np.unique(flat[order], return_counts=True)
    offs = np.zeros(len(used) + 1, np.int32)
    np.cumsum(counts, out=offs[1:])
    toks = (order // K).astype(np.int32)
    sw = weights.reshape(-1)[order].astype(np.float32)
    return used, offs, toks, sw


def fused_experts_cpu_int8(
    hidden_states: torch.Tensor,  # [M, H], any device
    w1q: torch.Tensor,  # [E, 2I, H] int8 codes (symmetric, per-tensor scale)
    w2q: torch.Tensor,  # [E, H, I] int8
    scales1: torch.Tensor,  # [E] fp32
    scales2: torch.Tensor,  # [E] fp32
    topk_weights: torch.Tensor,  # [M, K] fp32
    topk_ids: torch.Tensor,  # [M, K], local rows of w1q/w2q
    active: torch.Tensor,  # [M, K] bool: the slots computed on the host
    activation: str = "silu",
    n_threads: int = 0,
) -> torch.Tensor:
    """The CPU half of the split on int8 banks (fused_experts_cpu_int8,
    reframework/moe/fused.py:140-197): an fp32 [M, H] host tensor, the sum
    over the active slots of weight * expert(x). Per expert its token rows
    (fp32) are quantized as one block, gate|up is the exact integer product
    dequantized by the two scales, act(g) * u runs in fp32, the intermediate
    is quantized the same way and the second product dequantized likewise,
    all in libmoe355_host (bit for bit the oracle's restatement of the
    reference's steps). Each slot's output goes to its own token, not the
    reference's (t*K+k) % M. Active slots must route inside the bank, where
    the reference's indexing would fail. ``n_threads`` 0 uses every OpenMP
    thread."""
    act = activation_code(activation)
    x = hidden_states.detach().to("cpu", torch.float32).contiguous()
    M, H = x.shape
    out = torch.zeros((M, H), dtype=torch.float32)
    if w1q.dim() != 3 or w2q.dim() != 3 or w1q.dtype != torch.int8 or w2q.dtype != torch.int8:
        raise ValueError("w1q / w2q must be int8 [E, 2I, H] / [E, H, I] banks")
    E, I = w1q.shape[0], w2q.shape[2]
    if tuple(w1q.shape) != (E, 2 * I, H) or tuple(w2q.shape) != (E, H, I):
        raise ValueError(f"int8 bank shapes {tuple(w1q.shape)} / {tuple(w2q.shape)} do not "
                         f"match hidden size {H}")
    ids = topk_ids.detach().cpu().long().reshape(M, -1).numpy()
    K = ids.shape[1]
    wts = topk_weights.detach().cpu().float().reshape(M, K).numpy()
    on = active.detach().cpu().reshape(M, K).numpy().astype(bool)
    used, offs, toks, sw = _group_active_slots(ids, wts, on, E)
    if not len(used):
        return out
    q1, q2 = w1q.detach().cpu().contiguous(), w2q.detach().cpu().contiguous()
    b1 = [q1[int(e)] for e in used]
    b2 = [q2[int(e)] for e in used]
    s1 = scales1.detach().cpu().float().reshape(-1)
    s2 = scales2.detach().cpu().float().reshape(-1)
    _capi.host_experts_int8(x, b1, b2, [float(s1[int(e)]) for e in used],
                            [float(s2[int(e)]) for e in used],
                            [_capi.host_int8_row_sums(b, n_threads) for b in b1],
                            [_capi.host_int8_row_sums(b, n_threads) for b in b2],
                            offs, toks, sw, act, out, n_threads)
    return out


__all__ = ["torch_fused_topk", "grouped_topk", "fused_experts", "fused_experts_mxfp4",
           "fused_experts_fp8", "fused_experts_masked", "fused_experts_cpu_int8", "run_experts", "run_grouped_topk",
           "bank_pointers", "require_gpu"]
