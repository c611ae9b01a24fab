"""The experts' part of a training step: sort, gate/up product, gated activation, down product, weighted sum."""

from __future__ import annotations

import torch

from .... import _lib
from ...utils.common_types import ActFnType
from .expert_linear import MOST_COLUMNS, check_rows_and_weight
from .launch import native, same_device
from .sort_tokens import moe_sort_tokens, moe_unsort_tokens


def moe_expert_mlp(rows: torch.Tensor, gate_up_proj_weight: torch.Tensor, down_proj_weight: torch.Tensor,
                   expert_offsets: torch.Tensor, activation_function: ActFnType = ActFnType.SiLU,
                   _check_status: bool = False) -> torch.Tensor:
    """The experts' MLP on sorted rows: ``(act(gate) * up) @ down_proj_weight[e]`` with ``[gate, up] = rows @
    gate_up_proj_weight[e]``; ``rows [R, H]``, weights ``[E, H, 2, I]`` (or ``[E, H, 2 I]``) and ``[E, I, H]``, all bf16.

    The three operators in a row (:func:`expert_linear`, :func:`moe_glu`, :func:`expert_linear`), but what lives until the
    backward pass is the input rows and the 8-bit checkpoint of gate and up only: the activation in front of the down
    product is computed again from the checkpoint for the gradient of ``down_proj_weight``.

    ``_check_status`` as in :func:`expert_linear`, of all products in both passes.
    """
    same_device(rows, gate_up_proj_weight, down_proj_weight, expert_offsets)
    A = _lib.kernel_assert
    if gate_up_proj_weight.dim() == 4:
        A(gate_up_proj_weight.shape[2] == 2, "gate_up_proj_weight must be [E, H, 2, I] or [E, H, 2 I]")
        gate_up_proj_weight = gate_up_proj_weight.flatten(2)
    check_rows_and_weight(rows, gate_up_proj_weight, expert_offsets, "gate_up_proj_weight")
    A(isinstance(activation_function, ActFnType), "activation_function must be an ActFnType")
    A(down_proj_weight.dim() == 3 and down_proj_weight.dtype == torch.bfloat16 and
      down_proj_weight.shape[0] == gate_up_proj_weight.shape[0] and
      2 * down_proj_weight.shape[1] == gate_up_proj_weight.shape[2], "down_proj_weight must be bfloat16 [E, I, H_out]")
    A(down_proj_weight.shape[1] % 8 == 0 and down_proj_weight.shape[2] % 8 == 0 and
      0 < down_proj_weight.shape[2] <= MOST_COLUMNS, "both sizes of down_proj_weight's matrices must be multiples of 8, at most 2^27")
    return native().mlp(rows, gate_up_proj_weight, down_proj_weight, expert_offsets, activation_function.value, _check_status)


def moe_experts_train(hidden: torch.Tensor, affinities: torch.Tensor, expert_index: torch.Tensor,
                      gate_up_proj_weight: torch.Tensor, down_proj_weight: torch.Tensor,
                      activation_function: ActFnType = ActFnType.SiLU, _check_status: bool = False) -> torch.Tensor:
    """The MoE layer behind its router, differentiable in ``hidden [T, H]``, ``affinities [T, K]`` and both weights:
    :func:`moe_sort_tokens` -> :func:`moe_expert_mlp` -> :func:`moe_unsort_tokens`.  ``expert_index [T, K]`` may hold ids
    outside ``[0, E)`` for dropped pairs; a token whose pairs are all dropped comes out zero.

    Gradients come from an 8-bit checkpoint of gate and up (see :func:`moe_glu`), whose values are off by up to 2^-4 of themselves; that
    of ``down_proj_weight`` is taken at the activation computed again from it, which is not bit for bit the one the forward pass
    multiplied.
    """
    same_device(hidden, affinities, expert_index, gate_up_proj_weight, down_proj_weight)
    rows, plan = moe_sort_tokens(hidden, expert_index, gate_up_proj_weight.shape[0])
    out = moe_expert_mlp(rows, gate_up_proj_weight, down_proj_weight, plan.expert_offsets, activation_function, _check_status)
    return moe_unsort_tokens(out, affinities, plan)
