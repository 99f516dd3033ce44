"""Microscaled 4-bit floating point (MXFP4) for MoE experts: quantisation, products, a whole layer for a few tokens.

An :class:`Mx4Tensor` holds a matrix ``[..., K]`` as ``codes [..., K / 2]`` (uint8, two E2M1 values a byte, the even
column in the low nibble) and ``scales [..., K / 32]`` (uint8, E8M0: byte ``b`` stands for ``2 ** (b - 127)``, 255 for
NaN), the layout of MXFP4 checkpoints.  The functions run this package's sm_100a kernels on the tensors' device and
its current stream, return before their work is done, and may be captured into a CUDA graph.  There is no CPU
fallback and no autograd: weights in 4 bits are for serving.
"""
from __future__ import annotations

import torch

from . import _lib
from ._device import DTYPES, need_cuda, need_out, on, same_device, stream_of

BLOCK = 32


class Mx4Tensor:
    """Codes and scales of a matrix ``[..., K]``, ``K`` a multiple of 32, both contiguous uint8 (scales may be given
    as ``torch.float8_e8m0fnu``)."""

    __slots__ = ("codes", "scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor) -> None:
        if scales.dtype == torch.float8_e8m0fnu:
            scales = scales.view(torch.uint8)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError(f"codes and scales are uint8; got {codes.dtype} and {scales.dtype}")
        if (codes.dim() < 1 or codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] != 16 * scales.shape[-1]
                or codes.shape[-1] == 0):
            raise ValueError(f"codes [..., K / 2] and scales [..., K / 32] do not match: {tuple(codes.shape)} and "
                             f"{tuple(scales.shape)}")
        if codes.device != scales.device:
            raise ValueError(f"codes are on {codes.device}, scales on {scales.device}")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("codes and scales must be contiguous")
        self.codes, self.scales = codes, scales

    @property
    def shape(self) -> torch.Size:
        """Shape of the matrix that is held: ``[..., K]``."""
        return torch.Size((*self.codes.shape[:-1], 2 * self.codes.shape[-1]))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def __getitem__(self, i) -> "Mx4Tensor":
        """Indexes leading dimensions: ``experts[3]``, ``rows[:16]``."""
        if isinstance(i, tuple) and len(i) >= self.codes.dim():
            raise IndexError("the last dimension cannot be indexed")
        return Mx4Tensor(self.codes[i], self.scales[i])

    def __repr__(self) -> str:
        return f"Mx4Tensor(shape={tuple(self.shape)}, device={self.device})"


def mx4_quantize(x: torch.Tensor, out: Mx4Tensor | None = None) -> Mx4Tensor:
    """``x [..., K]`` (bf16, fp16 or fp32) to MXFP4 (``wisp_mx4_quantize``).

    Per block of 32 values along the last axis: scale ``2 ** (floor(log2(max|x|)) - 2)``, codes ``x / scale`` rounded
    to the nearest E2M1 value, ties to even, saturating at 6.  A block with an infinity or a NaN reads back as NaN; a
    block of zeros has scale byte 0.  Rows may lie apart (``x`` two-dimensional, its last axis contiguous and every
    row on a 16-byte boundary); anything else is made contiguous first."""
    dev = need_cuda("x", x)
    dt = DTYPES.get(x.dtype)
    if dt is None:
        raise TypeError(f"x must be bf16, fp16 or fp32; got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] == 0 or x.shape[-1] % BLOCK:
        raise ValueError(f"the last axis of x must be a multiple of {BLOCK}; got shape {tuple(x.shape)}")
    cols = x.shape[-1]
    size = x.element_size()
    if x.is_contiguous():
        stride = cols
    elif x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= cols and x.stride(0) * size % 16 == 0:
        stride = x.stride(0)
    else:
        x, stride = x.contiguous(), cols
    if x.data_ptr() % 16:
        x, stride = x.clone(memory_format=torch.contiguous_format), cols
    lead = x.shape[:-1]
    if out is None:
        out = Mx4Tensor.__new__(Mx4Tensor)
        out.codes = torch.empty((*lead, cols // 2), dtype=torch.uint8, device=dev)
        out.scales = torch.empty((*lead, cols // BLOCK), dtype=torch.uint8, device=dev)
    else:
        need_out("out.codes", out.codes, (*lead, cols // 2), torch.uint8, dev)
        need_out("out.scales", out.scales, (*lead, cols // BLOCK), torch.uint8, dev)
    with on(dev):
        _lib.check(_lib.lib().wisp_mx4_quantize(x.data_ptr(), dt, x.numel() // cols, cols, stride,
                                                out.codes.data_ptr(), out.scales.data_ptr(), stream_of(dev)),
                   "mx4_quantize")
    return out


def mx4_dequantize(q: Mx4Tensor, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of ``q`` (``wisp_mx4_dequantize``) as bf16 or fp32 (exact) or fp16 (rounded once where it cannot
    hold them)."""
    dev = need_cuda("q", q.codes)
    dt = DTYPES.get(dtype)
    if dt is None:
        raise TypeError(f"dtype must be bf16, fp16 or fp32; got {dtype}")
    shape = (*q.codes.shape[:-1], 2 * q.codes.shape[-1])
    out = torch.empty(shape, dtype=dtype, device=dev) if out is None else need_out("out", out, shape, dtype, dev)
    with on(dev):
        _lib.check(_lib.lib().wisp_mx4_dequantize(q.codes.data_ptr(), q.scales.data_ptr(), out.numel() // shape[-1],
                                                  shape[-1], out.data_ptr(), dt, stream_of(dev)), "mx4_dequantize")
    return out


__all__ = ["Mx4Tensor", "mx4_quantize", "mx4_dequantize"]
