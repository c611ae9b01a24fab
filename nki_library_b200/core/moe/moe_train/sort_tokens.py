"""Token rows sorted by expert, and the experts' rows back at their tokens with the routing affinities applied."""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from .... import _lib
from .launch import native, refuse, same_device

MAX_EXPERTS = 1024
_ID_TYPES = (torch.int32, torch.uint32, torch.int64)
_MOST_COLUMNS = 2 ** 30


class SortedTokens(NamedTuple):
    """The order of the T * K (token, choice) pairs by (expert, token, choice), int32 on the device.

    Expert e owns rows ``expert_offsets[e]`` to ``expert_offsets[e + 1]``; pair (t, k) sits in row ``row_of_pair[t, k]``, or
    in none (-1) if its expert id lies outside ``[0, num_experts)``.
    """
    expert_offsets: torch.Tensor
    row_of_pair: torch.Tensor
    num_experts: int


def _sort(hidden: Optional[torch.Tensor], expert_index: torch.Tensor, num_experts: int):
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
    if expert_index.numel() >= 2 ** 31:
        refuse(f"T * K ({expert_index.numel()}) must be below 2^31")
    rows, offsets, row_of_pair = native().sort(hidden, expert_index, E)
    return rows, SortedTokens(offsets, row_of_pair, E)


def moe_sort_plan(expert_index: torch.Tensor, num_experts: int) -> SortedTokens:
    """Sort the pairs of ``expert_index [T, K]`` (int32, uint32 or int64).  Ids outside ``[0, num_experts)``, such as the -1
    of a dropped pair, get no row; equal ids of one token get a row each."""
    return _sort(None, expert_index, num_experts)[1]


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
    return _sort(hidden, expert_index, num_experts)


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
    return native().unsort(rows, affinities, plan.row_of_pair, plan.expert_offsets)
