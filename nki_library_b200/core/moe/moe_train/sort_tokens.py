"""Token rows sorted by expert, and the experts' rows back at their tokens with the routing affinities applied."""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from .... import _lib
from .launch import launch, needs_grad, pitch_of, same_device, unit_rows

MAX_EXPERTS = 1024


class SortedTokens(NamedTuple):
    """The order of the T * K (token, choice) pairs by (expert, token, choice), all int32 on the device.

    Expert e owns rows ``expert_offsets[e]`` to ``expert_offsets[e + 1]``; pair (t, k) sits in row ``row_of_pair[t, k]``, or
    in none (-1) if its expert id lies outside ``[0, num_experts)``; row r holds pair ``pair_of_row[r]`` = t * K + k, or none
    (-1) behind the last expert.
    """
    expert_offsets: torch.Tensor
    row_of_pair: torch.Tensor
    pair_of_row: torch.Tensor
    num_experts: int


def moe_sort_plan(expert_index: torch.Tensor, num_experts: int) -> SortedTokens:
    """Sort the pairs of ``expert_index [T, K]`` (int32, uint32 or int64).  Ids outside ``[0, num_experts)``, such as the -1
    of a dropped pair, get no row; equal ids of one token get a row each."""
    _lib.require_cuda(expert_index)
    A = _lib.kernel_assert
    A(expert_index.dim() == 2, "expert_index must be [T, K]")
    A(expert_index.dtype in (torch.int32, torch.uint32, torch.int64), "expert_index must be int32, uint32 or int64")
    A(1 <= num_experts <= MAX_EXPERTS, f"num_experts ({num_experts}) must be between 1 and {MAX_EXPERTS}")
    T, K = expert_index.shape
    E, pairs = int(num_experts), T * K
    A(pairs < 2 ** 31, f"T * K ({pairs}) must be below 2^31")
    device = expert_index.device
    if pairs == 0:
        return SortedTokens(torch.zeros(E + 1, dtype=torch.int32, device=device),
                            torch.empty((T, K), dtype=torch.int32, device=device),
                            torch.empty(0, dtype=torch.int32, device=device), E)
    index = expert_index.contiguous()
    offsets = torch.empty(E + 1, dtype=torch.int32, device=device)
    row_of_pair = torch.empty((T, K), dtype=torch.int32, device=device)
    pair_of_row = torch.empty(pairs, dtype=torch.int32, device=device)
    size = _lib.load_library().b200moe_sort_workspace_bytes(pairs, E)
    ws = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    launch(device, "b200moe_sort_pairs", index.data_ptr(), index.element_size(), T, K, E, offsets.data_ptr(),
           row_of_pair.data_ptr(), pair_of_row.data_ptr(), _lib.ptr(ws), size)
    return SortedTokens(offsets, row_of_pair, pair_of_row, E)


def _check_plan(plan: SortedTokens) -> Tuple[int, int]:
    A = _lib.kernel_assert
    A(isinstance(plan, SortedTokens), "plan must be the SortedTokens of moe_sort_plan or moe_sort_tokens")
    A(plan.row_of_pair.dim() == 2 and plan.row_of_pair.dtype == torch.int32 and plan.row_of_pair.is_contiguous() and
      plan.expert_offsets.dtype == torch.int32 and plan.expert_offsets.is_contiguous() and
      plan.expert_offsets.numel() == plan.num_experts + 1, "plan must be as moe_sort_plan made it")
    return plan.row_of_pair.shape


def _check_rows(t: torch.Tensor, name: str) -> None:
    _lib.kernel_assert(t.dim() == 2 and t.dtype in (torch.bfloat16, torch.float32), f"{name} must be 2-D, bfloat16 or float32")


def _sort_rows(hidden: torch.Tensor, plan: SortedTokens) -> torch.Tensor:
    T, K = plan.row_of_pair.shape
    H = hidden.shape[1]
    rows = torch.empty((T * K, H), dtype=hidden.dtype, device=hidden.device)
    if rows.numel():
        hidden = unit_rows(hidden)
        launch(hidden.device, "b200moe_sort_rows", hidden.data_ptr(), _lib.dtype_code(hidden), pitch_of(hidden), T, K, H,
               plan.num_experts, plan.row_of_pair.data_ptr(), plan.expert_offsets.data_ptr(), rows.data_ptr())
    return rows


def _unsort_rows(rows: torch.Tensor, affinities: Optional[torch.Tensor], plan: SortedTokens) -> torch.Tensor:
    T, K = plan.row_of_pair.shape
    H = rows.shape[1]
    if T * K * H == 0:
        return torch.zeros((T, H), dtype=rows.dtype, device=rows.device)
    out = torch.empty((T, H), dtype=rows.dtype, device=rows.device)
    rows = unit_rows(rows)
    if affinities is not None:
        affinities = affinities.contiguous()
    launch(rows.device, "b200moe_unsort_rows", rows.data_ptr(), _lib.dtype_code(rows), pitch_of(rows), T, K, H,
           plan.row_of_pair.data_ptr(), _lib.ptr(affinities), _lib.F32 if affinities is None else _lib.dtype_code(affinities),
           out.data_ptr())
    return out


class _SortRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, plan):
        ctx.plan = plan
        return _sort_rows(hidden, plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_rows):
        return _unsort_rows(d_rows, None, ctx.plan), None


class _UnsortRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, affinities, plan):
        # the rows are needed for the affinities' gradient only
        ctx.save_for_backward(rows if affinities is not None and affinities.requires_grad else None, affinities)
        ctx.plan = plan
        return _unsort_rows(rows, affinities, plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        rows, affinities = ctx.saved_tensors
        plan = ctx.plan
        T, K = plan.row_of_pair.shape
        H = d_out.shape[1]
        want_rows, want_aff = ctx.needs_input_grad[:2]
        d_rows = torch.empty((T * K, H), dtype=d_out.dtype, device=d_out.device) if want_rows else None
        d_aff = torch.empty((T, K), dtype=affinities.dtype, device=d_out.device) if want_aff else None
        if T * K * H == 0:
            return d_rows, None if d_aff is None else d_aff.zero_(), None
        d_out = unit_rows(d_out)
        if want_aff:
            rows = unit_rows(rows)
        if affinities is not None:
            affinities = affinities.contiguous()
        launch(d_out.device, "b200moe_unsort_rows_backward", d_out.data_ptr(), pitch_of(d_out),
               rows.data_ptr() if want_aff else None, pitch_of(rows) if want_aff else H, _lib.dtype_code(d_out), T, K, H,
               plan.num_experts, plan.row_of_pair.data_ptr(), plan.expert_offsets.data_ptr(), _lib.ptr(affinities),
               _lib.F32 if affinities is None else _lib.dtype_code(affinities), _lib.ptr(d_rows), _lib.ptr(d_aff))
        return d_rows, d_aff, None


def moe_sort_tokens(hidden: torch.Tensor, expert_index: torch.Tensor,
                    num_experts: int) -> Tuple[torch.Tensor, SortedTokens]:
    """Rows of ``hidden [T, H]`` (bf16 or fp32) sorted by expert: ``(rows [T * K, H], plan)``.

    Every pair of ``expert_index [T, K]`` gets a copy of its token's row, ordered by (expert, token, choice); rows behind the
    last expert's (there are as many as pairs without an expert) are zero.  Differentiable: a token's gradient is the sum of
    its rows', taken in fp32 in the order of its choices and rounded once.  ``plan`` (:class:`SortedTokens`) goes to
    :func:`expert_linear` (its ``expert_offsets``) and :func:`moe_unsort_tokens`.
    """
    same_device(hidden, expert_index)
    _check_rows(hidden, "hidden")
    _lib.kernel_assert(expert_index.dim() == 2 and expert_index.shape[0] == hidden.shape[0],
                       "expert_index must be [T, K] with hidden's T")
    plan = moe_sort_plan(expert_index, num_experts)
    return (_SortRows.apply(hidden, plan) if needs_grad(hidden) else _sort_rows(hidden, plan)), plan


def moe_unsort_tokens(rows: torch.Tensor, affinities: Optional[torch.Tensor], plan: SortedTokens) -> torch.Tensor:
    """``out[t] = sum over k of affinities[t, k] * rows[row of (t, k)]``: the experts' ``rows [T * K, H]`` (bf16 or fp32)
    back at their tokens, ``[T, H]`` in the rows' type.

    ``affinities [T, K]`` fp32 or bf16 (what ``router_topk(..., return_eager_affi=True)`` returns last), or None for a plain
    sum.  Products and sums are fp32, in the order of the choices, rounded once; a token without rows comes out zero.
    Differentiable in ``rows`` (rows behind the last expert get zero) and ``affinities`` (zero for a pair without a row).
    """
    same_device(rows, affinities, plan.row_of_pair)
    T, K = _check_plan(plan)
    _check_rows(rows, "rows")
    _lib.kernel_assert(rows.shape[0] == T * K, f"rows must hold T * K ({T * K}) rows, got {rows.shape[0]}")
    if affinities is not None:
        _lib.kernel_assert(tuple(affinities.shape) == (T, K) and affinities.dtype in (torch.float32, torch.bfloat16),
                           f"affinities must be [T, K] = [{T}, {K}], float32 or bfloat16")
    if needs_grad(rows, affinities):
        return _UnsortRows.apply(rows, affinities, plan)
    return _unsort_rows(rows, affinities, plan)
