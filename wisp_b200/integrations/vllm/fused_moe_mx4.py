"""Paged MoE layers of MXFP4 experts.

``WispMoEStateMX4`` pages 4-bit experts the way :class:`WispMoEState` pages bf16 ones and ``WispMoEStateFP8`` pages
FP8 ones (src/wisp/integrations/vllm/fused_moe.py:126-490, fused_moe_fp8.py:61-145): the same LRU pager, counters and
methods.  An expert is 3.76 times smaller than in bf16, so a page-in moves that much less over the host link, a slot
takes that much less HBM and a decode step reads that much less of it.  The reference has no 4-bit layers.

An expert's codes and scales are one block of the host master, codes first, so that a page-in stays one copy a
projection; the compute (:func:`wisp_b200.mx4.mx4_moe`) reads the slots as they are, through the layer's expert map.
"""
from __future__ import annotations

import ctypes
import threading

import torch

from wisp_b200 import _lib
from wisp_b200.mx4 import MOE_MAX_TOKENS, Mx4Tensor, mx4_moe

from .fused_moe import WispMoEState, _Mode


def _blocks(t: Mx4Tensor) -> torch.Tensor:
    """One pinned block an expert: its codes, then its scales."""
    experts = t.codes.shape[0]
    return torch.cat((t.codes.reshape(experts, -1), t.scales.reshape(experts, -1)), 1).cpu().pin_memory()


class WispMoEStateMX4(WispMoEState):
    """Per-layer paging state of MXFP4 experts: ``w13 [E, 2I, H]`` (gate rows, then up rows) and ``w2 [E, H, I]`` as
    :class:`~wisp_b200.mx4.Mx4Tensor` (``H`` and ``I`` multiples of 32), on the CPU or a GPU; they are copied into
    pinned host memory.  The pager, counters and paging methods are those of :class:`WispMoEState`;
    ``slots_w13`` / ``slots_w2`` view the slots as ``Mx4Tensor``.  ``mode``: ``"paged"`` or ``"resident"``.  Hits,
    misses and evictions are counted; forwards are not (a forward here is one or more admission steps).

    A paged forward's kernels read the slots after it has returned.  The layer knows of them (``wisp_layer_used``), so
    that later page-ins, prefetches and resizes wait for them, on whichever stream they run; a lock keeps another
    thread's calls from coming between a forward's admission and its kernels."""

    def __init__(self, w13: Mx4Tensor, w2: Mx4Tensor, cap_experts: int, device, layer_idx: int,
                 mode: str = _Mode.PAGED) -> None:
        e, inter2, hidden = w13.shape if w13.codes.dim() == 3 else (0, 0, 0)
        if e == 0 or inter2 % 64 or tuple(w2.shape) != (e, hidden, inter2 // 2):
            raise ValueError(f"w13 [E, 2I, H] and w2 [E, H, I] do not match: {tuple(w13.shape)} and {tuple(w2.shape)}")
        self._mx4_shape = (int(hidden), int(inter2) // 2)
        self._primed = False
        self._lock = threading.RLock()
        super().__init__(_blocks(w13), _blocks(w2), cap_experts, mode, device, layer_idx)
        self._timeouts_told = self._timeouts()

    def _refresh_views(self) -> None:
        super()._refresh_views()
        hidden, inter = self._mx4_shape

        def view(scratch: torch.Tensor, rows: int, cols: int) -> Mx4Tensor:
            n = rows * cols // 2
            return Mx4Tensor(scratch[:, :n].unflatten(1, (rows, cols // 2)),
                             scratch[:, n:].unflatten(1, (rows, cols // 32)))

        self.slots_w13 = view(self.scratch_w13, 2 * inter, hidden)
        self.slots_w2 = view(self.scratch_w2, hidden, inter)

    def class_threshold(self) -> int:
        return 0                        # one compute class

    def forward(self, x: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor,
                out: torch.Tensor | None = None) -> torch.Tensor:
        """Paged (or resident) forward of ``x [T, H]`` bf16 with ``topk_weights [T, k]`` and ``topk_ids [T, k]``
        (int32 or int64).  A paged call admits the experts of its tokens group by group: consecutive tokens, at most
        64 and as many as the cap holds the experts of (first fit, fused_moe.py:1102-1168); a token that routes to
        more experts than the cap raises ``RuntimeError`` (mentioning sub-batch).  A token's result does not depend
        on the groups, the cap or the slots."""
        hidden, _ = self._mx4_shape
        if self.mode == _Mode.RESIDENT:
            self._check_primed()
        if x.dim() != 2 or x.shape[1] != hidden:
            raise ValueError(f"x must be [T, {hidden}]; got {tuple(x.shape)}")
        if topk_ids.dim() != 2 or topk_ids.shape[0] != x.shape[0] or topk_weights.shape != topk_ids.shape:
            raise ValueError(f"topk_weights and topk_ids must be [{x.shape[0]}, k]; got {tuple(topk_weights.shape)} and "
                             f"{tuple(topk_ids.shape)}")
        for name, t in (("x", x), ("topk_weights", topk_weights), ("topk_ids", topk_ids), ("out", out)):
            if t is not None and t.device != self.device:
                raise ValueError(f"{name} must be on {self.device}; got {t.device}")
        if x.dtype != torch.bfloat16:
            raise TypeError(f"a layer of 4-bit experts computes from bf16 activations; got {x.dtype}")
        if topk_ids.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"topk_ids must be int32 or int64; got {topk_ids.dtype}")
        if out is None:
            out = torch.empty((x.shape[0], hidden), dtype=x.dtype, device=x.device)
        elif out.shape != x.shape or out.dtype != x.dtype or not out.is_contiguous():
            raise ValueError(f"out must be contiguous bf16 {tuple(x.shape)}; got {out.dtype} {tuple(out.shape)}")
        if (out.untyped_storage().data_ptr() == x.untyped_storage().data_ptr()
                and (out.data_ptr(), out.stride()) != (x.data_ptr(), x.stride())):
            x = x.clone()               # a group's rows of out may lie where a later group's rows of x do

        def compute(a, b):
            mx4_moe(x[a:b], self.slots_w13, self.slots_w2, topk_weights=topk_weights[a:b], topk_ids=topk_ids[a:b],
                    expert_map=self.expert_map_device, out=out[a:b])

        if self.mode == _Mode.RESIDENT:
            for a in range(0, x.shape[0], MOE_MAX_TOKENS):
                compute(a, min(a + MOE_MAX_TOKENS, x.shape[0]))
            return out
        rows = topk_ids.tolist()        # the pager's step waits for the device too
        with self._lock:
            done = 0
            try:
                for a, b in self._groups(rows):
                    self.ensure_resident(topk_ids[a:b])
                    done = b
                    compute(a, b)
            finally:
                if done:
                    self._used(set().union(*rows[:done]))
        return out

    def _used(self, experts: set) -> None:
        """The kernels queued on the current stream read the slots of ``experts``."""
        ids = (ctypes.c_int32 * len(experts))(*experts)
        _lib.check(_lib.lib().wisp_layer_used(self._h, ids, len(ids), _lib.stream_ptr(
            torch.cuda.current_stream(self.device))), "layer_used")

    def _groups(self, rows: list):
        """Ranges of tokens that one kernel call takes."""
        tokens, a, held = len(rows), 0, set()
        for t, row in enumerate(rows):
            both = held | set(row)
            if t > a and (t - a == MOE_MAX_TOKENS or len(both) > self.cap_experts):
                yield a, t
                a, both = t, set(row)
            held = both
        if tokens:
            yield a, tokens

    def forward_router(self, x: torch.Tensor, router: torch.Tensor, top_k: int, renormalize: bool = True,
                       out: torch.Tensor | None = None) -> torch.Tensor:
        """A resident layer's forward of at most 64 tokens from its router weights ``[E, H]`` (bf16), in one kernel
        launch (a paged layer has to know the routed experts before it can page them in)."""
        if self.mode != _Mode.RESIDENT:
            raise ValueError("forward_router needs a resident layer; route first and call forward")
        self._check_primed()
        return mx4_moe(x, self.slots_w13, self.slots_w2, top_k, router=router, renormalize=renormalize,
                       expert_map=self.expert_map_device, out=out)

    def prime_identity(self) -> None:
        """Resident mode: identity map and full copy (fused_moe.py:242-258).  Waits for the layer's forwards before
        the copy and for the copy itself, so that forwards on any stream find the experts in their slots."""
        torch.cuda.synchronize(self.device)
        super().prime_identity()
        torch.cuda.current_stream(self.device).synchronize()
        self._primed = True

    def ensure_resident(self, needed_experts: torch.Tensor) -> None:
        with self._lock:
            super().ensure_resident(needed_experts)

    def pager_step(self, topk_ids: torch.Tensor):
        with self._lock:
            return super().pager_step(topk_ids)

    def prefetch_async(self, predicted_experts) -> None:
        with self._lock:
            super().prefetch_async(predicted_experts)

    def resize_cap(self, new_cap: int) -> None:
        with self._lock:
            super().resize_cap(new_cap)

    def _check_primed(self) -> None:
        if not self._primed:
            raise _lib.WispError(_lib.WISP_ERR_INVALID, "resident layer has no expert in its slots; call prime_identity "
                                                        "first")

    def _timeouts(self) -> int:
        """Waits inside 4-bit kernels that have run out on the layer's device so far."""
        n = ctypes.c_int64(0)
        with torch.cuda.device(self.device):
            _lib.check(_lib.lib().wisp_mx4_timeouts(_lib.stream_ptr(torch.cuda.current_stream()), ctypes.byref(n)))
        return n.value

    def synchronize(self) -> None:
        """Wait for this layer's queued work, on whichever streams, and raise the first error of its page-ins or kernels.
        A wait that ran out inside a 4-bit kernel is counted for the device, not for the layer: every layer there raises
        for it once."""
        torch.cuda.synchronize(self.device)
        super().synchronize()
        told, self._timeouts_told = self._timeouts_told, self._timeouts()
        if self._timeouts_told != told:
            raise _lib.WispError(_lib.WISP_ERR_TIMEOUT, "a wait inside a 4-bit kernel ran out; its output is not "
                                                        "complete")


__all__ = ["WispMoEStateMX4"]
