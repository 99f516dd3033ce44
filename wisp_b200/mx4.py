"""Microscaled 4-bit floating point (MXFP4) for MoE experts: quantisation, products, a whole layer for a few tokens.

An :class:`Mx4Tensor` holds a matrix ``[..., K]`` as ``codes [..., K / 2]`` (uint8, two E2M1 values a byte, the even
column in the low nibble) and ``scales [..., K / 32]`` (uint8, E8M0: byte ``b`` stands for ``2 ** (b - 127)``, 255 for
NaN), the layout of MXFP4 checkpoints.  The functions run this package's sm_100a kernels on the tensors' device and
its current stream, return before their work is done, and may be captured into a CUDA graph.  There is no CPU
fallback and no autograd: weights in 4 bits are for serving.
"""
from __future__ import annotations

import torch

from ._bind import native

BLOCK = 32


class Mx4Tensor:
    """Codes and scales of a matrix ``[..., K]``, ``K`` a multiple of 32, both uint8 (scales may be given as
    ``torch.float8_e8m0fnu``) and contiguous; the matrices of a stack ``[S, N, K]`` may lie apart (slots that hold
    other tensors too)."""

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
        for t in (codes, scales):
            if not (t.is_contiguous() or (t.dim() == 3 and t.stride(2) == 1 and t.stride(1) == t.shape[2]
                                          and t.stride(0) >= t.shape[1] * t.shape[2])):
                raise ValueError("codes and scales must be contiguous, or a stack of contiguous matrices")
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


def _new(codes: torch.Tensor, scales: torch.Tensor) -> Mx4Tensor:
    """An Mx4Tensor of tensors made here: nothing to check."""
    t = Mx4Tensor.__new__(Mx4Tensor)
    t.codes, t.scales = codes, scales
    return t


def mx4_quantize(x: torch.Tensor, out: Mx4Tensor | None = None) -> Mx4Tensor:
    """``x [..., K]`` (bf16, fp16 or fp32) to MXFP4 (``wisp_mx4_quantize``).

    Per block of 32 values along the last axis: scale ``2 ** (floor(log2(max|x|)) - 2)``, codes ``x / scale`` rounded
    to the nearest E2M1 value, ties to even, saturating at 6.  A block with an infinity or a NaN reads back as NaN; a
    block of zeros has scale byte 0.  Rows may lie apart (``x`` two-dimensional, its last axis contiguous and every
    row on a 16-byte boundary); anything else is made contiguous first."""
    if out is None:
        return _new(*native.mx4_quantize(x, None, None))
    native.mx4_quantize(x, out.codes, out.scales)
    return out


def mx4_dequantize(q: Mx4Tensor, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of ``q`` (``wisp_mx4_dequantize``) as bf16 or fp32 (exact) or fp16 (rounded once where it cannot
    hold them)."""
    return native.mx4_dequantize(q.codes, q.scales, dtype, out)


def mx4_matmul(a: Mx4Tensor, w: Mx4Tensor, offsets: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Products of MXFP4 matrices on the block-scaled tensor cores (``wisp_mx4_matmul``).

    ``a [M, K]`` times ``w [N, K]`` transposed; or, grouped, ``w [G, N, K]`` with ``offsets [G + 1]`` (int32, ascending,
    on the device): rows ``offsets[g]`` to ``offsets[g + 1]`` times ``w[g]`` transposed, the products of MoE experts
    over rows sorted by expert.  Returns ``[M, N]`` bf16 (fp32 accumulation, one rounding).  Rows behind the last
    offset are left as they are in ``out`` (undefined in a new tensor)."""
    return native.mx4_matmul(a.codes, a.scales, w.codes, w.scales, offsets, out)


def mx4_synchronize(device: torch.device | None = None) -> None:
    """Wait for the device's current stream and raise if a bounded wait inside an :func:`mx4_matmul` or
    :func:`mx4_moe` has run out on the device, on whichever stream, since this was last called on this stream."""
    index = None if device is None else torch.device(device).index
    native.mx4_synchronize(torch.cuda.current_device() if index is None else index)


MOE_MAX_TOKENS = 64


def mx4_moe(x: torch.Tensor, w13: Mx4Tensor, w2: Mx4Tensor, top_k: int | None = None, *,
            router: torch.Tensor | None = None, renormalize: bool = True, topk_weights: torch.Tensor | None = None,
            topk_ids: torch.Tensor | None = None, expert_map: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """A whole MoE layer for at most 64 tokens, in one launch (``wisp_mx4_moe``): routing, gate-up, SiLU, down and the
    weighted sum, from MXFP4 experts and bf16 activations.  Inside the products a block of
    32 activations is a sum of eight MXFP4 terms, which hold a value to 2^-23 of the largest one in its block (and to
    2^-129 at best), a bf16 value of at least 2^-15 of it exactly.

    ``x [T, H]`` bf16; ``w13 [S, 2I, H]`` (gate rows, then up rows) and ``w2 [S, H, I]``.  Routing is either the
    layer's ``router [E, H]`` (bf16) with ``top_k``: softmax over the ``top_k`` largest products (over all of them and
    not renormalised with ``renormalize=False``), ties to the lower id; or ``topk_weights [T, k]`` (fp32) and
    ``topk_ids [T, k]`` (int32 or int64).  ``expert_map [E]`` (int32) gives each expert's slot, the row of ``w13`` and
    ``w2`` it lies in (a paged layer's ``expert_map_device``); without it the slot is the id.  Ids outside ``[0, E)``
    and experts without a slot contribute nothing.  Returns ``[T, H]`` bf16."""
    return native.mx4_moe(x, w13.codes, w13.scales, w2.codes, w2.scales, top_k, router, renormalize, topk_weights,
                          topk_ids, expert_map, out)


__all__ = ["Mx4Tensor", "mx4_quantize", "mx4_dequantize", "mx4_matmul", "mx4_moe", "mx4_synchronize"]
