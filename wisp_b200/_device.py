"""What the stateless operators share: types, devices and streams of tensors."""
from __future__ import annotations

import contextlib

import torch

BF16, FP16, FP32 = 0, 1, 2          # enum wisp_dtype
DTYPES = {torch.bfloat16: BF16, torch.float16: FP16, torch.float32: FP32}

_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_same = contextlib.nullcontext()


def on(device: torch.device):
    """A context in which ``device`` is the current CUDA device."""
    return _same if device.index == _current_device() else torch.cuda.device(device)


def stream_of(device: torch.device) -> int:
    """The device's current stream as a ``cudaStream_t``."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def need_cuda(name: str, t: torch.Tensor) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor; got {type(t).__name__}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on a CUDA device; got {t.device}")
    return t.device


def same_device(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


def need_out(name: str, out: torch.Tensor, shape, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """An output given by the caller: contiguous, of this shape and type."""
    if out.device != device or out.dtype != dtype or tuple(out.shape) != tuple(shape) or not out.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")
    return out
