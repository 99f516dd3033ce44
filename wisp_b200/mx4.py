"""Microscaled 4-bit floating point (MXFP4) for MoE experts: quantisation, products, a whole layer for a few tokens.

An :class:`Mx4Tensor` holds a matrix ``[..., K]`` as ``codes [..., K / 2]`` (uint8, two E2M1 values a byte, the even
column in the low nibble) and ``scales [..., K / 32]`` (uint8, E8M0: byte ``b`` stands for ``2 ** (b - 127)``, 255 for
NaN), the layout of MXFP4 checkpoints.  The functions run this package's sm_100a kernels on the tensors' device and
its current stream, return before their work is done, and may be captured into a CUDA graph.  There is no CPU
fallback and no autograd: weights in 4 bits are for serving.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._device import DTYPES, cuda_index, launch, need_out, same_device

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
    index = cuda_index("x", x)
    dt = DTYPES.get(x.dtype)
    if dt is None:
        raise TypeError(f"x must be bf16, fp16 or fp32; got {x.dtype}")
    shape = x.shape
    if len(shape) < 1 or shape[-1] == 0 or shape[-1] % BLOCK:
        raise ValueError(f"the last axis of x must be a multiple of {BLOCK}; got shape {tuple(shape)}")
    cols = stride = shape[-1]
    if not x.is_contiguous():
        if len(shape) == 2 and x.stride(1) == 1 and x.stride(0) >= cols and x.stride(0) * x.element_size() % 16 == 0:
            stride = x.stride(0)
        else:
            x = x.contiguous()
    ptr = x.data_ptr()
    if ptr % 16:
        x, stride = x.clone(memory_format=torch.contiguous_format), cols
        ptr = x.data_ptr()
    lead = shape[:-1]
    if out is None:
        out = _new(x.new_empty((*lead, cols // 2), dtype=torch.uint8), x.new_empty((*lead, cols // BLOCK), dtype=torch.uint8))
    else:
        need_out("out.codes", out.codes, (*lead, cols // 2), torch.uint8, index)
        need_out("out.scales", out.scales, (*lead, cols // BLOCK), torch.uint8, index)
    launch("wisp_mx4_quantize", index, ptr, dt, x.numel() // cols, cols, stride, out.codes.data_ptr(),
           out.scales.data_ptr())
    return out


def mx4_dequantize(q: Mx4Tensor, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of ``q`` (``wisp_mx4_dequantize``) as bf16 or fp32 (exact) or fp16 (rounded once where it cannot
    hold them)."""
    codes = q.codes
    index = cuda_index("q", codes)
    if not (codes.is_contiguous() and q.scales.is_contiguous()):
        raise ValueError("mx4_dequantize takes contiguous matrices")
    dt = DTYPES.get(dtype)
    if dt is None:
        raise TypeError(f"dtype must be bf16, fp16 or fp32; got {dtype}")
    shape = (*codes.shape[:-1], 2 * codes.shape[-1])
    out = codes.new_empty(shape, dtype=dtype) if out is None else need_out("out", out, shape, dtype, index)
    launch("wisp_mx4_dequantize", index, codes.data_ptr(), q.scales.data_ptr(), out.numel() // shape[-1], shape[-1],
           out.data_ptr(), dt)
    return out


def mx4_matmul(a: Mx4Tensor, w: Mx4Tensor, offsets: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Products of MXFP4 matrices on the block-scaled tensor cores (``wisp_mx4_matmul``).

    ``a [M, K]`` times ``w [N, K]`` transposed; or, grouped, ``w [G, N, K]`` with ``offsets [G + 1]`` (int32, ascending,
    on the device): rows ``offsets[g]`` to ``offsets[g + 1]`` times ``w[g]`` transposed, the products of MoE experts
    over rows sorted by expert.  Returns ``[M, N]`` bf16 (fp32 accumulation, one rounding).  Rows behind the last
    offset are left as they are in ``out`` (undefined in a new tensor)."""
    index = cuda_index("a", a.codes)
    if a.codes.dim() != 2 or w.codes.dim() not in (2, 3) or w.codes.shape[-1] != a.codes.shape[1]:
        raise ValueError(f"a is [M, K], w [N, K] or [G, N, K]; got {tuple(a.shape)} and {tuple(w.shape)}")
    if not (a.codes.is_contiguous() and w.codes.is_contiguous() and w.scales.is_contiguous()):
        raise ValueError("mx4_matmul takes contiguous matrices")
    rows, half = a.codes.shape
    n = w.codes.shape[-2]
    groups = w.codes.shape[0] if w.codes.dim() == 3 else 1
    op = None
    if offsets is not None:
        if offsets.dtype != torch.int32 or offsets.shape != (groups + 1,) or not offsets.is_contiguous():
            raise ValueError(f"offsets must be a contiguous int32 [{groups + 1}] tensor; got {offsets.dtype} "
                             f"{tuple(offsets.shape)}")
        op = offsets.data_ptr()
    elif groups != 1:
        raise ValueError(f"{groups} groups need offsets")
    same_device(index, w=w.codes, offsets=offsets)
    out = (a.codes.new_empty((rows, n), dtype=torch.bfloat16) if out is None
           else need_out("out", out, (rows, n), torch.bfloat16, index))
    launch("wisp_mx4_matmul", index, a.codes.data_ptr(), a.scales.data_ptr(), rows, w.codes.data_ptr(),
           w.scales.data_ptr(), groups, n, 2 * half, op, out.data_ptr())
    return out


def mx4_synchronize(device: torch.device | None = None) -> None:
    """Wait for the device's current stream and raise if a bounded wait inside an :func:`mx4_matmul` ran out."""
    index = None if device is None else torch.device(device).index
    launch("wisp_mx4_sync", torch.cuda.current_device() if index is None else index)


MOE_MAX_TOKENS = 64


@functools.lru_cache(maxsize=256)
def _moe_workspace(tokens: int, experts: int, top_k: int, hidden: int, inter: int) -> int:
    n = ctypes.c_int64(0)
    _lib.check(_lib.lib().wisp_mx4_moe_workspace(tokens, experts, top_k, hidden, inter, ctypes.byref(n)), "mx4_moe")
    return n.value


def mx4_moe(x: torch.Tensor, w13: Mx4Tensor, w2: Mx4Tensor, top_k: int | None = None, *,
            router: torch.Tensor | None = None, renormalize: bool = True, topk_weights: torch.Tensor | None = None,
            topk_ids: torch.Tensor | None = None, expert_map: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """A whole MoE layer for at most 64 tokens, in one launch (``wisp_mx4_moe``): routing, gate-up, SiLU, down and the
    weighted sum, from MXFP4 experts and bf16 activations.

    ``x [T, H]`` bf16; ``w13 [S, 2I, H]`` (gate rows, then up rows) and ``w2 [S, H, I]``.  Routing is either the
    layer's ``router [E, H]`` (bf16) with ``top_k``: softmax over the ``top_k`` largest products (over all of them and
    not renormalised with ``renormalize=False``), ties to the lower id; or ``topk_weights [T, k]`` (fp32) and
    ``topk_ids [T, k]`` (int32 or int64).  ``expert_map [E]`` (int32) gives each expert's slot, the row of ``w13`` and
    ``w2`` it lies in (a paged layer's ``expert_map_device``); without it the slot is the id.  Ids outside ``[0, E)``
    and experts without a slot contribute nothing.  Returns ``[T, H]`` bf16."""
    index = cuda_index("x", x)
    if x.dtype != torch.bfloat16:
        raise TypeError(f"mx4_moe computes from bf16 activations; got {x.dtype}")
    if x.dim() != 2 or w13.codes.dim() != 3 or w2.codes.dim() != 3:
        raise ValueError("x is [T, H], w13 [S, 2I, H] and w2 [S, H, I]")
    tokens, hidden = x.shape
    slots, inter2, half = w13.codes.shape
    if 2 * half != hidden or inter2 % 2 or w2.codes.shape != (slots, hidden, inter2 // 4):
        raise ValueError(f"shapes do not match: x {tuple(x.shape)}, w13 {tuple(w13.shape)}, w2 {tuple(w2.shape)}")
    if tokens > MOE_MAX_TOKENS:
        raise ValueError(f"mx4_moe takes at most {MOE_MAX_TOKENS} tokens a call; got {tokens} (mx4_quantize and "
                         "mx4_matmul serve longer ones)")
    same_device(index, w13=w13.codes, w2=w2.codes, router=router, topk_weights=topk_weights, topk_ids=topk_ids,
                expert_map=expert_map)
    experts = slots if expert_map is None else expert_map.numel()
    if expert_map is not None and (expert_map.dtype != torch.int32 or not expert_map.is_contiguous()):
        raise TypeError("expert_map must be a contiguous int32 tensor")
    rp = ip = wp = None
    ids64 = 0
    if router is not None:
        if topk_ids is not None or topk_weights is not None or top_k is None:
            raise ValueError("give either router and top_k, or topk_weights and topk_ids")
        if router.dtype != torch.bfloat16 or tuple(router.shape) != (experts, hidden) or not router.is_contiguous():
            raise ValueError(f"router must be a contiguous bf16 [{experts}, {hidden}] tensor")
        rp = router.data_ptr()
    else:
        if topk_ids is None or topk_weights is None:
            raise ValueError("give either router and top_k, or topk_weights and topk_ids")
        if topk_ids.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"topk_ids must be int32 or int64; got {topk_ids.dtype}")
        if topk_ids.dim() != 2 or topk_ids.shape[0] != tokens or topk_weights.shape != topk_ids.shape:
            raise ValueError("topk_ids and topk_weights are [T, k]")
        if top_k is not None and top_k != topk_ids.shape[1]:
            raise ValueError(f"top_k is {top_k}, topk_ids {tuple(topk_ids.shape)}")
        top_k = topk_ids.shape[1]
        topk_ids, topk_weights = topk_ids.contiguous(), topk_weights.to(torch.float32).contiguous()
        ip, wp, ids64 = topk_ids.data_ptr(), topk_weights.data_ptr(), int(topk_ids.dtype == torch.int64)
    if x.stride(1) != 1 or (tokens > 1 and (x.stride(0) < hidden or x.stride(0) % 8)) or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    strides = None
    if not (w13.codes.is_contiguous() and w13.scales.is_contiguous() and w2.codes.is_contiguous()
            and w2.scales.is_contiguous()):
        strides = (ctypes.c_int64 * 4)(w13.codes.stride(0), w13.scales.stride(0), w2.codes.stride(0),
                                       w2.scales.stride(0))
    out = (x.new_empty((tokens, hidden)) if out is None
           else need_out("out", out, (tokens, hidden), torch.bfloat16, index))
    need = _moe_workspace(tokens, experts, top_k, hidden, inter2 // 2)
    ws = x.new_empty(need, dtype=torch.uint8)
    launch("wisp_mx4_moe", index, x.data_ptr(), x.stride(0), rp, ip, ids64, wp,
           None if expert_map is None else expert_map.data_ptr(), w13.codes.data_ptr(), w13.scales.data_ptr(),
           w2.codes.data_ptr(), w2.scales.data_ptr(), strides, slots, tokens, experts, top_k, hidden, inter2 // 2,
           int(renormalize), ws.data_ptr(), need, out.data_ptr())
    return out


__all__ = ["Mx4Tensor", "mx4_quantize", "mx4_dequantize", "mx4_matmul", "mx4_moe", "mx4_synchronize"]
