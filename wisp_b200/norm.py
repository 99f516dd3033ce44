"""The norms before and after a decoder block, fused with the block's gate and the scaled residual sum."""
from __future__ import annotations

import torch

from ._device import DTYPES, cuda_index, launch, need_out

GATE_NONE, GATE_TOKEN, GATE_CHANNEL, GATE_FULL = 0, 1, 2, 3   # enum wisp_gate


def _rows(t: torch.Tensor, cols: int) -> tuple[torch.Tensor, int]:
    """``t [..., cols]`` as rows of one stride (a copy where its strides do not allow that)."""
    if t.is_contiguous():
        return t, cols
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= 0:
        return t, t.stride(0)
    return t.contiguous(), cols


def block_norm(y: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, *,
               post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
               eps: float = 1e-6, out: torch.Tensor | None = None, residual_out: torch.Tensor | None = None,
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """``(normed, new residual)`` after a block that returned ``y [..., H]`` (``wisp_block_norm``)::

        z = y                                                     # without post_weight
          = y * rsqrt(mean(y ** 2) + eps) * post_weight           # a norm after the block
        r = residual + scale * gate * z
        normed = r * rsqrt(mean(r ** 2) + eps) * weight           # the norm before the next block

    in fp32, ``r`` and ``normed`` rounded once each.  ``y`` is bf16, fp16 or fp32 (``normed`` likewise); ``residual``
    and the weights have its type or fp32.  ``gate`` has ``y``'s type: one value for each channel (``[H]``), for each
    token (``[..., 1]``) or for each element (``[..., H]``).  ``residual_out=residual`` updates the residual in place.
    At most 16384 channels."""
    index = cuda_index("y", y)
    dtype, shape = y.dtype, y.shape
    dt, rdt, wdt = DTYPES.get(dtype), DTYPES.get(residual.dtype), DTYPES.get(weight.dtype)
    if dt is None:
        raise TypeError(f"y must be bf16, fp16 or fp32; got {dtype}")
    if (rdt != dt and rdt != 2) or (wdt != dt and wdt != 2):
        raise TypeError(f"residual and weight must be {dtype} or fp32; got {residual.dtype} and {weight.dtype}")
    if len(shape) < 1 or residual.shape != shape:
        raise ValueError(f"residual must have y's shape {tuple(shape)}; got {tuple(residual.shape)}")
    cols = shape[-1]
    if weight.shape != (cols,) or not weight.is_contiguous():
        raise ValueError(f"weight must be contiguous [{cols}]; got {tuple(weight.shape)}")
    post_ptr = gate_ptr = None
    if post_weight is not None:
        if post_weight.shape != (cols,) or not post_weight.is_contiguous() or post_weight.dtype != weight.dtype:
            raise ValueError(f"post_weight must be contiguous [{cols}] of weight's type")
        post_ptr = post_weight.data_ptr()
    kind, gate_stride = GATE_NONE, 0
    if gate is not None:
        gshape = gate.shape
        if gate.dtype != dtype:
            raise TypeError(f"gate must be {dtype}; got {gate.dtype}")
        if gshape == (cols,):
            kind, gate = GATE_CHANNEL, gate.contiguous()
        elif len(gshape) == len(shape) and gshape[:-1] == shape[:-1] and gshape[-1] == 1:
            kind = GATE_TOKEN
            gate = gate if len(gshape) == 2 and gate.stride(0) >= 0 else gate.contiguous()
            gate_stride = gate.stride(0) if len(gshape) == 2 else 1
        elif gshape == shape:
            kind = GATE_FULL
            gate, gate_stride = _rows(gate, cols)
        else:
            raise ValueError(f"gate must be [{cols}], [..., 1] or [..., {cols}]; got {tuple(gshape)}")
        gate_ptr = gate.data_ptr()
    for t in (residual, weight, post_weight, gate):
        if t is not None and (not t.is_cuda or t.get_device() != index):
            raise ValueError(f"the tensors are on several devices: {t.device} and cuda:{index}")
    y, y_stride = _rows(y, cols)
    residual, r_stride = _rows(residual, cols)
    if out is None:
        out = torch.empty_like(y, memory_format=torch.contiguous_format)
    else:
        need_out("out", out, shape, dtype, index)
    if residual_out is None:
        residual_out = torch.empty_like(residual, memory_format=torch.contiguous_format)
    else:
        need_out("residual_out", residual_out, shape, residual.dtype, index)
    launch("wisp_block_norm", index, y.data_ptr(), y_stride, residual.data_ptr(), r_stride, weight.data_ptr(), post_ptr,
           gate_ptr, kind, gate_stride, dt, rdt, wdt, out.numel() // cols if cols else 0, cols, scale, eps,
           out.data_ptr(), residual_out.data_ptr())
    return out, residual_out


__all__ = ["block_norm"]
