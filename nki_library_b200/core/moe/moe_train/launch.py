"""What the operators of the training pass share: the device and stream of a call, and rows the kernels can read."""

from __future__ import annotations

import torch

from .... import _lib


def same_device(*tensors) -> torch.device:
    _lib.require_cuda(*tensors)
    device = None
    for t in tensors:
        if t is not None:
            _lib.kernel_assert(device is None or t.device == device, "all tensors must live on the same device")
            device = t.device
    return device


def launch(device: torch.device, name: str, *args) -> None:
    """Call an entry point on the current stream of ``device``, whichever device is current."""
    if device.index == torch.cuda.current_device():
        _lib.call(name, *args, torch.cuda.current_stream().cuda_stream)
        return
    with torch.cuda.device(device):
        _lib.call(name, *args, torch.cuda.current_stream().cuda_stream)


def needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def pitch_of(t: torch.Tensor) -> int:
    """Elements between two rows of a 2-D tensor with contiguous columns (a single row has none)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def unit_rows(t: torch.Tensor) -> torch.Tensor:
    """``t [rows, cols]`` itself if its columns are contiguous, else a copy."""
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def tile_rows(t: torch.Tensor) -> torch.Tensor:
    """``t [rows, cols]`` itself if its rows do not overlap and all start on 16-byte boundaries, else a copy."""
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (
            t.shape[0] <= 1 or (t.stride(0) >= t.shape[1] and t.stride(0) * t.element_size() % 16 == 0)):
        return t
    return t.clone(memory_format=torch.contiguous_format)
