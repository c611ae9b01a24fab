"""Gated activation between the expert products, with an 8-bit activation checkpoint for its backward pass."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .... import _lib
from ...utils.common_types import ActFnType
from .launch import MOST_ROWS, native, refuse

_MOST_I = 2 ** 26


def glu_forward(gate_up: torch.Tensor, act: int, keep: bool) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(m, kept)``; ``kept`` (the codes of all rows, then their scales) None unless ``keep``."""
    return native().glu_forward(gate_up, act, keep)


def glu_backward(d_m: Optional[torch.Tensor], kept: torch.Tensor, R: int, I: int, act: int,
                 want_m: bool = False) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``(d_gate_up, m)`` at the kept gate and up; the first None without ``d_m [R, I]``, the second unless wanted."""
    return native().glu_backward(d_m, kept, R, I, act, want_m)


def moe_glu(gate_up: torch.Tensor, activation_function: ActFnType = ActFnType.SiLU) -> torch.Tensor:
    """``act(gate) * up`` of ``gate_up [R, 2 I]`` (or ``[R, 2, I]``; gate first), bf16 with fp32 arithmetic, ``[R, I]``.

    Differentiable, and what is kept for the backward pass is not ``gate_up`` but 8-bit codes of it: e4m3 with one power of
    two per 32 columns, the smallest for which no finite value of the 32 exceeds 448 of it (8.25 bits a value; a kept value
    is off by at most 2^-4 of itself, or 2^-10 of the power).  The gradient is the formula's at the kept values.  Values that
    are not finite are kept as NaN and leave their neighbours' scale alone.  I is a multiple of 8.
    """
    if not gate_up.is_cuda:
        _lib.require_cuda(gate_up)
    if gate_up.dim() == 3 and gate_up.shape[1] == 2:
        gate_up = gate_up.flatten(1)
    if gate_up.dtype != torch.bfloat16 or gate_up.dim() != 2:
        refuse("gate_up must be bfloat16 [R, 2 I] or [R, 2, I]")
    if not isinstance(activation_function, ActFnType):
        refuse("activation_function must be an ActFnType")
    if gate_up.shape[1] == 0 or gate_up.shape[1] % 16:
        refuse(f"I must be a multiple of 8, gate_up has {gate_up.shape[1]} columns")
    if gate_up.shape[0] > MOST_ROWS or gate_up.shape[1] > 2 * _MOST_I:
        refuse(f"at most 2^30 rows of at most 2^27 columns, got {list(gate_up.shape)}")
    return native().glu(gate_up, activation_function.value)
