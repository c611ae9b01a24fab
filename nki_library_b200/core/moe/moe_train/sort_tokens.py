"""Token rows sorted by expert, and the experts' rows back at their tokens with the routing affinities applied."""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from .... import _lib
from .launch import launch, needs_grad, once, pitch_of, refuse, same_device, unit_rows

MAX_EXPERTS = 1024
_ID_TYPES = (torch.int32, torch.uint32, torch.int64)
_MOST_COLUMNS = 2 ** 30
_ONE_LAUNCH = 2048  # pairs that the sort takes without a workspace


class SortedTokens(NamedTuple):
    """The order of the T * K (token, choice) pairs by (expert, token, choice), int32 on the device.

    Expert e owns rows ``expert_offsets[e]`` to ``expert_offsets[e + 1]``; pair (t, k) sits in row ``row_of_pair[t, k]``, or
    in none (-1) if its expert id lies outside ``[0, num_experts)``.
    """
    expert_offsets: torch.Tensor
    row_of_pair: torch.Tensor
    num_experts: int


def _sort(expert_index: torch.Tensor, num_experts: int, hidden: Optional[torch.Tensor]):
    """``(rows, plan)``; rows None without ``hidden``."""
    if not expert_index.is_cuda:
        _lib.require_cuda(expert_index)
    if expert_index.dim() != 2:
        refuse("expert_index must be [T, K]")
    if expert_index.dtype not in _ID_TYPES:
        refuse("expert_index must be int32, uint32 or int64")
    E = int(num_experts)
    if not 1 <= E <= MAX_EXPERTS:
        refuse(f"num_experts ({num_experts}) must be between 1 and {MAX_EXPERTS}")
    T, K = expert_index.shape
    pairs = T * K
    if pairs >= 2 ** 31:
        refuse(f"T * K ({pairs}) must be below 2^31")
    device = expert_index.device
    row_of_pair = torch.empty((T, K), dtype=torch.int32, device=device)
    H = 0
    rows = None
    if hidden is not None:
        H = hidden.shape[1]
        rows = torch.empty((pairs, H), dtype=hidden.dtype, device=device)
    if pairs == 0:
        return rows, SortedTokens(torch.zeros(E + 1, dtype=torch.int32, device=device), row_of_pair, E)
    index = expert_index.contiguous()
    offsets = torch.empty(E + 1, dtype=torch.int32, device=device)
    size, ws = 0, None
    if pairs > _ONE_LAUNCH:
        size = _lib.load_library().b200moe_sort_workspace_bytes(pairs, E)
        ws = torch.empty(size, dtype=torch.uint8, device=device)
    if H:
        hidden = unit_rows(hidden)
        launch(device, "b200moe_sort_tokens", hidden.data_ptr(), _lib.dtype_code(hidden), pitch_of(hidden), index.data_ptr(),
               index.element_size(), T, K, H, E, offsets.data_ptr(), row_of_pair.data_ptr(), rows.data_ptr(), _lib.ptr(ws), size)
    else:
        launch(device, "b200moe_sort_pairs", index.data_ptr(), index.element_size(), T, K, E, offsets.data_ptr(),
               row_of_pair.data_ptr(), _lib.ptr(ws), size)
    return rows, SortedTokens(offsets, row_of_pair, E)


def moe_sort_plan(expert_index: torch.Tensor, num_experts: int) -> SortedTokens:
    """Sort the pairs of ``expert_index [T, K]`` (int32, uint32 or int64).  Ids outside ``[0, num_experts)``, such as the -1
    of a dropped pair, get no row; equal ids of one token get a row each."""
    return _sort(expert_index, num_experts, None)[1]


def _check_plan(plan: SortedTokens) -> Tuple[int, int]:
    if not isinstance(plan, SortedTokens):
        refuse("plan must be the SortedTokens of moe_sort_plan or moe_sort_tokens")
    row, offsets = plan.row_of_pair, plan.expert_offsets
    if not (row.dim() == 2 and row.dtype == torch.int32 and row.is_contiguous() and offsets.dtype == torch.int32 and
            offsets.is_contiguous() and offsets.numel() == plan.num_experts + 1):
        refuse("plan must be as moe_sort_plan made it")
    return row.shape


def _check_rows(t: torch.Tensor, name: str) -> None:
    if t.dim() != 2 or t.dtype not in (torch.bfloat16, torch.float32):
        refuse(f"{name} must be 2-D, bfloat16 or float32")
    if t.shape[1] > _MOST_COLUMNS:
        refuse(f"{name} must have at most 2^30 columns")


def _unsort_rows(rows: torch.Tensor, affinities: Optional[torch.Tensor], row_of_pair: torch.Tensor) -> torch.Tensor:
    T, K = row_of_pair.shape
    H = rows.shape[1]
    if T * K * H == 0:
        return torch.zeros((T, H), dtype=rows.dtype, device=rows.device)
    out = torch.empty((T, H), dtype=rows.dtype, device=rows.device)
    rows = unit_rows(rows)
    if affinities is not None:
        affinities = affinities.contiguous()
    launch(rows.device, "b200moe_unsort_rows", rows.data_ptr(), _lib.dtype_code(rows), pitch_of(rows), T, K, H,
           row_of_pair.data_ptr(), _lib.ptr(affinities), _lib.F32 if affinities is None else _lib.dtype_code(affinities),
           out.data_ptr())
    return out


class _SortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, expert_index, num_experts):
        rows, plan = _sort(expert_index, num_experts, hidden)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(plan.expert_offsets, plan.row_of_pair)
        ctx.save_for_backward(plan.row_of_pair)
        return rows, plan.expert_offsets, plan.row_of_pair

    @staticmethod
    @once
    def backward(ctx, d_rows, _offsets, _row_of_pair):
        row_of_pair, = ctx.saved_tensors
        return (None if d_rows is None else _unsort_rows(d_rows, None, row_of_pair)), None, None


class _UnsortRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, affinities, row_of_pair, expert_offsets):
        # the rows are needed for the affinities' gradient only
        ctx.save_for_backward(rows if affinities is not None and affinities.requires_grad else None, affinities, row_of_pair,
                              expert_offsets)
        return _unsort_rows(rows, affinities, row_of_pair)

    @staticmethod
    @once
    def backward(ctx, d_out):
        rows, affinities, row_of_pair, offsets = ctx.saved_tensors
        T, K = row_of_pair.shape
        H = d_out.shape[1]
        want_rows, want_aff = ctx.needs_input_grad[:2]
        d_rows = torch.empty((T * K, H), dtype=d_out.dtype, device=d_out.device) if want_rows else None
        d_aff = torch.empty((T, K), dtype=affinities.dtype, device=d_out.device) if want_aff else None
        if T * K * H == 0:
            return d_rows, None if d_aff is None else d_aff.zero_(), None, None
        d_out = unit_rows(d_out)
        if want_aff:
            rows = unit_rows(rows)
        if affinities is not None:
            affinities = affinities.contiguous()
        launch(d_out.device, "b200moe_unsort_rows_backward", d_out.data_ptr(), pitch_of(d_out),
               rows.data_ptr() if want_aff else None, pitch_of(rows) if want_aff else H, _lib.dtype_code(d_out), T, K, H,
               offsets.numel() - 1, row_of_pair.data_ptr(), offsets.data_ptr(), _lib.ptr(affinities),
               _lib.F32 if affinities is None else _lib.dtype_code(affinities), _lib.ptr(d_rows), _lib.ptr(d_aff))
        return d_rows, d_aff, None, None


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
    if expert_index.dim() != 2 or expert_index.shape[0] != hidden.shape[0]:
        refuse("expert_index must be [T, K] with hidden's T")
    if not needs_grad(hidden):
        return _sort(expert_index, num_experts, hidden)
    rows, offsets, row_of_pair = _SortTokens.apply(hidden, expert_index, num_experts)
    return rows, SortedTokens(offsets, row_of_pair, int(num_experts))


def moe_unsort_tokens(rows: torch.Tensor, affinities: Optional[torch.Tensor], plan: SortedTokens) -> torch.Tensor:
    """``out[t] = sum over k of affinities[t, k] * rows[row of (t, k)]``: the experts' ``rows [T * K, H]`` (bf16 or fp32)
    back at their tokens, ``[T, H]`` in the rows' type.

    ``affinities [T, K]`` fp32 or bf16 (what ``router_topk(..., return_eager_affi=True)`` returns last), or None for a plain
    sum.  Products and sums are fp32, in the order of the choices, rounded once; a token without rows comes out zero.
    Differentiable in ``rows`` (rows behind the last expert get zero) and ``affinities`` (zero for a pair without a row).
    """
    T, K = _check_plan(plan)
    same_device(rows, affinities, plan.row_of_pair, plan.expert_offsets)
    _check_rows(rows, "rows")
    if rows.shape[0] != T * K:
        refuse(f"rows must hold T * K ({T * K}) rows, got {rows.shape[0]}")
    if affinities is not None and (affinities.shape != plan.row_of_pair.shape or
                                   affinities.dtype not in (torch.float32, torch.bfloat16)):
        refuse(f"affinities must be [T, K] = [{T}, {K}], float32 or bfloat16")
    if needs_grad(rows, affinities):
        return _UnsortRows.apply(rows, affinities, plan.row_of_pair, plan.expert_offsets)
    return _unsort_rows(rows, affinities, plan.row_of_pair)
