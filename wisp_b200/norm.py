"""The norms before and after a decoder block, fused with the block's gate and the scaled residual sum."""
from __future__ import annotations

import torch

from . import _lib
from ._device import DTYPES, need_cuda, need_out, on, same_device, stream_of

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
    dev = need_cuda("y", y)
    same_device(dev, residual=residual, weight=weight, post_weight=post_weight, gate=gate)
    dt, rdt, wdt = DTYPES.get(y.dtype), DTYPES.get(residual.dtype), DTYPES.get(weight.dtype)
    if dt is None:
        raise TypeError(f"y must be bf16, fp16 or fp32; got {y.dtype}")
    for name, t in (("residual", residual), ("weight", weight)):
        if t.dtype not in (y.dtype, torch.float32):
            raise TypeError(f"{name} must be {y.dtype} or fp32; got {t.dtype}")
    if y.dim() < 1 or residual.shape != y.shape:
        raise ValueError(f"residual must have y's shape {tuple(y.shape)}; got {tuple(residual.shape)}")
    cols = y.shape[-1]
    if weight.shape != (cols,) or not weight.is_contiguous():
        raise ValueError(f"weight must be contiguous [{cols}]; got {tuple(weight.shape)}")
    if post_weight is not None and (post_weight.shape != (cols,) or not post_weight.is_contiguous()
                                    or post_weight.dtype != weight.dtype):
        raise ValueError(f"post_weight must be contiguous [{cols}] of weight's type")
    kind, gate_stride = GATE_NONE, 0
    if gate is not None:
        if gate.dtype != y.dtype:
            raise TypeError(f"gate must be {y.dtype}; got {gate.dtype}")
        if gate.shape == (cols,):
            kind, gate = GATE_CHANNEL, gate.contiguous()
        elif gate.dim() == y.dim() and gate.shape[:-1] == y.shape[:-1] and gate.shape[-1] == 1:
            kind = GATE_TOKEN
            gate = gate if gate.dim() == 2 and gate.stride(0) >= 0 else gate.contiguous()
            gate_stride = gate.stride(0) if gate.dim() == 2 else 1
        elif gate.shape == y.shape:
            kind = GATE_FULL
            gate, gate_stride = _rows(gate, cols)
        else:
            raise ValueError(f"gate must be [{cols}], [..., 1] or [..., {cols}]; got {tuple(gate.shape)}")
    shape = y.shape
    out = torch.empty(shape, dtype=y.dtype, device=dev) if out is None else need_out("out", out, shape, y.dtype, dev)
    if residual_out is None:
        residual_out = torch.empty(shape, dtype=residual.dtype, device=dev)
    else:
        need_out("residual_out", residual_out, shape, residual.dtype, dev)
    y, y_stride = _rows(y, cols)
    residual, r_stride = _rows(residual, cols)
    with on(dev):
        _lib.check(_lib.lib().wisp_block_norm(
            y.data_ptr(), y_stride, residual.data_ptr(), r_stride, weight.data_ptr(),
            None if post_weight is None else post_weight.data_ptr(), None if gate is None else gate.data_ptr(), kind,
            gate_stride, dt, rdt, wdt, out.numel() // cols if cols else 0, cols, scale, eps, out.data_ptr(),
            residual_out.data_ptr(), stream_of(dev)), "block_norm")
    return out, residual_out


__all__ = ["block_norm"]
