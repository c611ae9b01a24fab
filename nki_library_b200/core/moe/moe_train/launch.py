"""What the operators of the training pass share: the device and stream of a call, and rows the kernels can read.

A call on a few rows is host work: refusals format their messages only when they refuse, and the stream's handle is asked for
without an object around it (3 us each, four to ten times per training step).
"""

from __future__ import annotations

import torch

from .... import _lib

MOST_ROWS = 2 ** 30  # of a product or an activation: indices of tiles behind the last row stay below 2^31

_raw_stream = torch._C._cuda_getCurrentRawStream


def refuse(message: str) -> None:
    _lib.kernel_assert(False, message)


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


def launch(device: torch.device, name: str, *args) -> None:
    """Call an entry point on the current stream of ``device``, whichever device is current."""
    index = device.index
    if index == torch.cuda.current_device():
        _lib.call(name, *args, _raw_stream(index))
        return
    with torch.cuda.device(device):
        _lib.call(name, *args, _raw_stream(index))


def needs_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def once(backward):
    """``once_differentiable`` for the one case it is there for, a backward pass that is itself recorded
    (``create_graph=True``); the usual one does without its bookkeeping."""
    recorded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return recorded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def pitch_of(t: torch.Tensor) -> int:
    """Elements between two rows of a 2-D tensor with contiguous columns (a single row has none)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def unit_rows(t: torch.Tensor) -> torch.Tensor:
    """``t [rows, cols]`` itself if its columns are contiguous, else a copy."""
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def tile_rows(t: torch.Tensor) -> torch.Tensor:
    """``t [rows, cols]`` itself if its rows do not overlap and all start on 16-byte boundaries, else a copy."""
    if t.data_ptr() % 16 == 0 and t.stride(1) == 1:
        pitch = t.stride(0)
        if (pitch >= t.shape[1] and pitch * t.element_size() % 16 == 0) or t.shape[0] <= 1:
            return t
    return t.clone(memory_format=torch.contiguous_format)
