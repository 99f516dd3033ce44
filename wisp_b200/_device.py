"""What the stateless operators share: types, devices and streams of tensors.

These calls are short next to the work they queue only if the checks around
them are: one token's kernel takes two microseconds.  So devices are compared
by index, and the current device is switched only where it is another one.
"""
from __future__ import annotations

import torch

from . import _lib

BF16, FP16, FP32 = 0, 1, 2          # enum wisp_dtype
DTYPES = {torch.bfloat16: BF16, torch.float16: FP16, torch.float32: FP32}

_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    _raw_stream = torch._C._cuda_getCurrentRawStream


def launch(name: str, index: int, *args) -> None:
    """``wisp_<name>(*args, stream)`` on device ``index`` and its current stream; raises what the call reports."""
    fn = getattr(_lib._lib or _lib.lib(), name)
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def cuda_index(name: str, t: torch.Tensor) -> int:
    """The index of the CUDA device a tensor is on."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor; got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device; got {t.device}")
    return t.get_device()


def same_device(index: int, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and (not t.is_cuda or t.get_device() != index):
            raise ValueError(f"{name} is on {t.device}, not on cuda:{index}")


def need_out(name: str, out: torch.Tensor, shape, dtype: torch.dtype, index: int) -> torch.Tensor:
    """An output given by the caller: contiguous, of this shape and type."""
    if (out.dtype != dtype or tuple(out.shape) != tuple(shape) or not out.is_contiguous() or not out.is_cuda
            or out.get_device() != index):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{index}")
    return out
