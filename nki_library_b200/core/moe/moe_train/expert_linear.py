"""One product per expert on rows that are sorted by expert, with its gradients."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .... import _lib
from .launch import MOST_ROWS, launch, needs_grad, once, pitch_of, refuse, same_device, tile_rows
from .sort_tokens import MAX_EXPERTS


def _readable(w: torch.Tensor) -> bool:
    """Matrices the kernels can read: contiguous columns, rows and matrices apart and on 16-byte boundaries."""
    E, rows, cols = w.shape
    matrix, pitch, unit = w.stride()
    return (unit == 1 and w.data_ptr() % 16 == 0 and (rows == 1 or pitch >= cols and pitch % 8 == 0) and
            (E == 1 or matrix >= cols and matrix % 8 == 0))


def _stored(weight: torch.Tensor) -> Tuple[torch.Tensor, bool]:
    """``weight [E, K, N]`` as matrices the kernels can read: (tensor, transposed).  Transposed ones lie in memory as
    [E, N, K], like the weights of linear layers; anything else is copied."""
    if _readable(weight):
        return weight, False
    turned = weight.transpose(1, 2)
    if _readable(turned):
        return turned, True
    return weight.clone(memory_format=torch.contiguous_format), False


MOST_COLUMNS = 2 ** 27
_LONG = 49 * 64  # contractions below this length are never cut into parts, and need no workspace


def _workspace(size: int, device: torch.device) -> Tuple[Optional[torch.Tensor], int]:
    return (torch.empty(size, dtype=torch.uint8, device=device), size) if size else (None, 0)


def product(rows: torch.Tensor, weight: torch.Tensor, expert_offsets: torch.Tensor, transpose: bool = False,
            check_status: bool = False) -> torch.Tensor:
    """``rows[r] @ weight[e]``, with ``transpose`` ``rows[r] @ weight[e].T``."""
    stored, turned = _stored(weight)
    E, D0, D1 = stored.shape
    contract_last = transpose != turned
    R = rows.shape[0]
    out = torch.empty((R, D0 if contract_last else D1), dtype=torch.bfloat16, device=rows.device)
    if R == 0:
        return out
    rows = tile_rows(rows)
    w_pitch = stored.stride(1)
    ws, ws_bytes = None, 0
    if rows.shape[1] >= _LONG:
        ws, ws_bytes = _workspace(_lib.load_library().b200moe_expert_product_workspace_bytes(int(contract_last), R, E, D0, D1),
                                  rows.device)
    status = torch.empty(2, dtype=torch.int32, device=rows.device)
    launch(rows.device, "b200moe_expert_product", rows.data_ptr(), pitch_of(rows), stored.data_ptr(), w_pitch,
           stored.stride(0) if E > 1 else D0 * w_pitch, int(contract_last), expert_offsets.data_ptr(), R, E, D0, D1,
           out.data_ptr(), _lib.ptr(ws), ws_bytes, status.data_ptr())
    if check_status:
        _lib.kernel_assert(int(status[0].item()) == 0, f"device-side wait expired in expert_linear (status {int(status[0].item())})")
    return out


def weight_grad(rows: torch.Tensor, d_out: torch.Tensor, weight: torch.Tensor, expert_offsets: torch.Tensor) -> torch.Tensor:
    """Gradient of :func:`product` in ``weight``, laid out in memory as the weight is."""
    E, K, N = weight.shape
    turned = _stored_turned(weight)
    a, b = (d_out, rows) if turned else (rows, d_out)
    M, W = (N, K) if turned else (K, N)
    if rows.shape[0] == 0:
        out = torch.zeros((E, M, W), dtype=torch.bfloat16, device=weight.device)
    else:
        out = torch.empty((E, M, W), dtype=torch.bfloat16, device=weight.device)
        a, b = tile_rows(a), tile_rows(b)
        status = torch.empty(2, dtype=torch.int32, device=weight.device)
        R, ws, ws_bytes = rows.shape[0], None, 0
        if R >= _LONG * E:
            ws, ws_bytes = _workspace(_lib.load_library().b200moe_expert_weight_grad_workspace_bytes(R, E, M, W), weight.device)
        launch(weight.device, "b200moe_expert_weight_grad", a.data_ptr(), pitch_of(a), b.data_ptr(), pitch_of(b),
               expert_offsets.data_ptr(), R, E, M, W, out.data_ptr(), _lib.ptr(ws), ws_bytes, status.data_ptr())
    return out.transpose(1, 2) if turned else out


def _stored_turned(weight: torch.Tensor) -> bool:
    return weight.stride(2) != 1 and weight.stride(1) == 1


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weight, expert_offsets, check_status):
        need_rows, need_weight = rows.requires_grad, weight.requires_grad
        ctx.save_for_backward(rows if need_weight else None, weight, expert_offsets)
        return product(rows, weight, expert_offsets, check_status=check_status)

    @staticmethod
    @once
    def backward(ctx, d_out):
        rows, weight, offsets = ctx.saved_tensors
        d_out = tile_rows(d_out)
        d_rows = product(d_out, weight, offsets, transpose=True) if ctx.needs_input_grad[0] else None
        d_weight = weight_grad(rows, d_out, weight, offsets) if ctx.needs_input_grad[1] else None
        return d_rows, d_weight, None, None


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
    """
    same_device(rows, weight, expert_offsets)
    if weight.dim() == 4:
        weight = weight.flatten(2)
    check_rows_and_weight(rows, weight, expert_offsets, "weight")
    if needs_grad(rows, weight):
        return _ExpertLinear.apply(rows, weight, expert_offsets, _check_status)
    return product(rows, weight, expert_offsets, check_status=_check_status)
