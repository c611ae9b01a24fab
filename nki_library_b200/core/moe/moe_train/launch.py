"""What the operators of the training pass share: checks of their arguments, and the way to the native code.

A call on a few rows is host work: refusals format their messages only when they refuse, and allocations, launches and the
nodes of the autograd graph are native (``csrc/autograd.cpp``).
"""

from __future__ import annotations

import torch

from .... import _lib

MOST_ROWS = 2 ** 30  # of a product or an activation: indices of tiles behind the last row stay below 2^31

_native = None


def refuse(message: str) -> None:
    _lib.kernel_assert(False, message)


def native():
    """The operators on tensors; their arguments have been checked."""
    global _native
    if _native is None:
        _lib.load_library()
        try:
            from .... import _autograd
        except ImportError as error:
            raise RuntimeError("nki_library_b200/_autograd.so is missing or does not fit this torch: build it with "
                               f"`python -m nki_library_b200.build` ({error})") from error
        _native = _autograd
    return _native


def same_device(first: torch.Tensor, *others) -> torch.device:
    """The CUDA device that all tensors (or None) live on."""
    device = first.device
    if device.type != "cuda":
        _lib.require_cuda(first)
    for t in others:
        if t is not None and t.device != device:
            _lib.require_cuda(t)
            refuse("all tensors must live on the same device")
    return device
