"""The norms before and after a decoder block, fused with the block's gate and the scaled residual sum."""
from __future__ import annotations

import torch

from ._bind import native


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
    token (``[..., 1]``) or for each element (``[..., H]``).  ``residual_out=residual`` updates the residual in place; an
    output that overlaps an input in another way, or the other output, is refused.  At most 16384 channels.  No
    autograd: for serving."""
    return native.block_norm(y, residual, weight, post_weight, gate, scale, eps, out, residual_out)


__all__ = ["block_norm"]
