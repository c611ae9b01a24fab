"""One product per expert on rows that are sorted by expert, with its gradients."""

from __future__ import annotations

import torch

from .launch import MOST_ROWS, native, refuse, same_device
from .sort_tokens import MAX_EXPERTS

MOST_COLUMNS = 2 ** 27


def product(rows: torch.Tensor, weight: torch.Tensor, expert_offsets: torch.Tensor, transpose: bool = False) -> torch.Tensor:
    """``rows[r] @ weight[e]``, with ``transpose`` ``rows[r] @ weight[e].T``, without a gradient."""
    return native().product(rows, weight, expert_offsets, transpose, False)


def weight_grad(rows: torch.Tensor, d_out: torch.Tensor, weight: torch.Tensor, expert_offsets: torch.Tensor) -> torch.Tensor:
    """Gradient of :func:`product` in ``weight``, laid out in memory as the weight is."""
    return native().weight_grad(rows, d_out, weight, expert_offsets)


def check_rows_and_weight(rows: torch.Tensor, weight: torch.Tensor, expert_offsets: torch.Tensor, name: str) -> None:
    if rows.dim() != 2 or rows.dtype != torch.bfloat16:
        refuse("rows must be bfloat16 [R, K]")
    if weight.dim() != 3 or weight.dtype != torch.bfloat16:
        refuse(f"{name} must be bfloat16 with one matrix per expert")
    E, K, N = weight.shape
    R, cols = rows.shape
    if cols != K:
        refuse(f"rows have {cols} columns, {name} contracts {K}")
    if K % 8 or N % 8 or not K or not N:
        refuse(f"both sizes of {name}'s matrices ({K}, {N}) must be multiples of 8")
    if not 1 <= E <= MAX_EXPERTS:
        refuse(f"between 1 and {MAX_EXPERTS} experts, got {E}")
    if expert_offsets.dtype != torch.int32 or expert_offsets.shape != (E + 1,) or not expert_offsets.is_contiguous():
        refuse(f"expert_offsets must be int32 [E + 1] = [{E + 1}]")
    if R > MOST_ROWS or max(K, N) > MOST_COLUMNS:
        refuse(f"at most 2^30 rows and matrices of at most 2^27 either way, got {R} rows and {K} x {N}")


def expert_linear(rows: torch.Tensor, weight: torch.Tensor, expert_offsets: torch.Tensor,
                  _check_status: bool = False) -> torch.Tensor:
    """``out[r] = rows[r] @ weight[e]`` for the rows ``expert_offsets[e]`` to ``expert_offsets[e + 1]`` of every expert e.

    ``rows [R, K]`` and ``weight [E, K, N]`` are bf16 (the reference's ``[E, H, 2, I]`` gate/up weight is taken as
    ``[E, H, 2 I]``), accumulation is fp32, the output ``[R, N]`` bf16.  ``expert_offsets`` (int32 ``[E + 1]``, on the device;
    :class:`SortedTokens` has it) is read by the kernels only and brought into ``[0, R]`` and ascending order there; rows of
    no expert come out zero.  K and N are multiples of 8.  A weight that lies in memory as ``[E, N, K]`` (a transposed view)
    is read where it is, and its gradient comes in that layout.

    Differentiable in ``rows`` (zero in rows of no expert) and ``weight`` (zero for an expert without rows); gradients are
    bf16, summed in fp32 over an expert's rows only, whatever the other rows hold.

    A product whose device-side wait runs out (it stands still for two seconds) ends and leaves NaN where it has written nothing;
    with ``_check_status`` the call and its backward pass wait for their products and raise.
    """
    same_device(rows, weight, expert_offsets)
    if weight.dim() == 4:
        weight = weight.flatten(2)
    check_rows_and_weight(rows, weight, expert_offsets, "weight")
    return native().linear(rows, weight, expert_offsets, _check_status)
