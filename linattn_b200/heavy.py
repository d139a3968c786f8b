"""A cache of fixed size that keeps the heavy hitters: attention-weight eviction.

Where the paged cache keeps every token and selects what a query reads, this one keeps, per
sequence and kv head, ``budget`` tokens: the first ``sinks``, the last ``recent`` and, of the
rest, the ones that have received the most attention weight (the eviction family of
``src/linattn/variants/eviction.py``, as a physical cache that holds nothing else).

    o, lse = packed_attention(q, k, v, cu)              # the prompts
    mass = attention_mass(q, k, lse, cu)                # what each key received
    cache.load(k, v, mass, cu)                          # cut to the budget
    while decoding:
        o = cache.step(q, k_new, v_new)                 # replace the least slot, attend, add up

``k, v (B, H_kv, budget, D)``: a (sequence, kv head) is one contiguous block of rows, so
decoding streams it; slots are not ordered by position (attention does not depend on the
order of its keys), ``pos`` says which token a slot holds.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from linattn_b200 import _lib as L

__all__ = ["HeavyCache"]


_STREAMS = 8  # streams whose arrival counts are there from the start


class HeavyCache:
    """``budget`` slots per (sequence, kv head) with accumulated attention weights.

    Every update runs on the device and on the current stream: no host copy of the lengths, and
    no allocation after the first step on a stream but for an output that is not given (``out``),
    so a decode step can be captured in a CUDA graph.  ``seen (B,)`` counts the tokens of each
    sequence; ``min(seen, budget)`` slots are in use.

    Calls that change the cache follow one another like any writes to a tensor: on one stream,
    or on streams that wait for each other.  ``attend(accumulate=False)`` only reads, and may run
    on several streams at once: each has scratch of its own, which stays for the cache's life
    (a captured graph holds its address).  Graphs captured on one stream share that stream's
    scratch, so of these only one runs at a time."""

    def __init__(self, batch: int, n_kv_heads: int, head_dim: int, budget: int, *, sinks: int = 0, recent: int = 1,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("HeavyCache lives in device memory (cuda)")
        if dtype not in (torch.bfloat16, torch.float16):
            raise NotImplementedError(f"HeavyCache holds bf16 or f16, not {dtype}")
        if head_dim not in (64, 128):
            raise NotImplementedError(f"head_dim must be 64 or 128, got {head_dim}")
        if batch < 1 or n_kv_heads < 1 or budget < 1:
            raise ValueError("batch, n_kv_heads and budget must be positive")
        if sinks < 0 or recent < 1 or sinks + recent > budget:
            raise ValueError(f"sinks >= 0, recent >= 1 and sinks + recent <= budget, got {sinks}, {recent}, {budget}")
        self.batch, self.n_kv_heads, self.head_dim, self.budget = batch, n_kv_heads, head_dim, budget
        self.sinks, self.recent, self.dtype = sinks, recent, dtype
        shape = (batch, n_kv_heads, budget)
        self.k = torch.zeros(*shape, head_dim, dtype=dtype, device=self.device)
        self.v = torch.zeros(*shape, head_dim, dtype=dtype, device=self.device)
        self.mass = torch.zeros(shape, dtype=torch.float32, device=self.device)
        self.pos = torch.zeros(shape, dtype=torch.int32, device=self.device)
        ints = torch.zeros(batch * (2 + _STREAMS * n_kv_heads), dtype=torch.int32, device=self.device)
        self.seen, self._ticket = ints[:batch], ints[batch:2 * batch]
        self._unit_tickets = list(ints[2 * batch:].view(_STREAMS, -1))  # attend()'s, one a stream
        self.device = self.k.device
        self._stream_tickets: dict = {}  # stream -> arrival counts
        self._scratch: dict = {}         # (stream, bytes) -> their address, the workspace's, the workspace
        self._desc = L.Heavy(self.k.data_ptr(), self.v.data_ptr(), self.mass.data_ptr(), self.pos.data_ptr(),
                             self.seen.data_ptr(), L.dtype_code(self.k), batch, n_kv_heads, budget, head_dim, sinks, recent)
        # what every call passes
        self._lib, self._ref, self._ticket_ptr = L.lib(), ctypes.byref(self._desc), self._ticket.data_ptr()
        self._maps = ctypes.create_string_buffer(L.HEAVY_MAPS)
        L.check(self._lib.linattn_heavy_maps(self._ref, self._maps))
        self._desc.maps = ctypes.addressof(self._maps)
        self._index = self.device.index
        self._plans: dict = {}  # checked arguments of append and attend, by shapes, strides and types
        self._status_ptr = L.status_word(self.device).data_ptr()
        self._scale = 1.0 / math.sqrt(head_dim)

    def reset(self) -> None:
        """Forget every token.  A cache whose call reported a wait that gave up needs this
        before its next call: the arrival counts may have stayed where that call left them."""
        self.seen.zero_()
        self._ticket.zero_()
        for tickets in self._unit_tickets:
            tickets.zero_()

    def load(self, k: torch.Tensor, v: torch.Tensor, mass: torch.Tensor, cu: torch.Tensor,
             rows: Optional[torch.Tensor] = None) -> None:
        """Take packed prompts ``k, v (N, H_kv, D)`` with offsets ``cu (S + 1,)`` and masses
        ``(H_kv, N)`` fp32: prompt ``s`` replaces row ``rows[s]`` (int32; default ``s``) of the
        cache; a row that is named twice ends up with a mixture.  One of at most ``budget`` tokens is kept whole; of a longer one the sinks, the
        recent tokens and those of most mass (lowest position on ties), by ascending position."""
        if L.current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.load(k, v, mass, cu, rows)
        dev = L.require_cuda(k, v, mass, cu, rows, self.k)
        if k.dim() != 3 or k.shape[1:] != (self.n_kv_heads, self.head_dim) or v.shape != k.shape:
            raise ValueError(f"k and v must be (N, {self.n_kv_heads}, {self.head_dim})")
        if k.dtype != self.dtype or v.dtype != self.dtype:
            raise ValueError(f"k and v must be {self.dtype} as the cache")
        if mass.shape != (self.n_kv_heads, k.shape[0]) or mass.dtype != torch.float32:
            raise ValueError("mass must be fp32 (H_kv, N)")
        if cu.dtype != torch.int32 or cu.dim() != 1 or cu.numel() < 1 or not cu.is_contiguous():
            raise ValueError("cu must be a contiguous int32 vector of sequence offsets (S + 1)")
        s = cu.numel() - 1
        if rows is not None and (rows.dtype != torch.int32 or rows.shape != (s,) or not rows.is_contiguous()):
            raise ValueError("rows must be a contiguous int32 vector of one cache row per sequence")
        k, v = _rows16(k), _rows16(v)
        if mass.stride(1) != 1:
            mass = mass.contiguous()
        L.check(self._lib.linattn_heavy_load(
            self._ref, k.data_ptr(), v.data_ptr(), L.strides2(k), L.strides2(v), k.shape[0], mass.data_ptr(),
            mass.stride(0), cu.data_ptr(), L.ptr(rows), s, self._status_ptr, L.raw_stream(dev.index)))
        if L.strict():
            L.check_status(dev)

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """Take ``(B, H_kv, T_new, D)`` keys / values, one token after the other: each fills the
        next empty slot or, in a full cache, replaces the slot of least mass (lowest slot on
        ties) outside the sinks and the last ``recent`` tokens (itself among them)."""
        if L.current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.append(k, v)
        key = (k.shape, k.stride(), v.shape, v.stride(), k.dtype, v.dtype, k.get_device(), v.get_device())
        plan = self._plans.get(key)
        if plan is None:
            plan = self._keep(key, self._plan_append(k, v))
        if plan[0] is None or (k.data_ptr() | v.data_ptr()) & 15:  # rows off the 16-byte grid
            return self.append(k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format))
        L.check(self._lib.linattn_heavy_append(self._ref, k.data_ptr(), v.data_ptr(), plan[0], plan[1], plan[2],
                                               self._ticket_ptr, self._status_ptr, L.raw_stream(self._index)))
        if L.strict():
            L.check_status(self.device)

    def _keep(self, key, plan):
        if len(self._plans) >= 256:
            self._plans.clear()
        self._plans[key] = plan
        return plan

    def _plan_append(self, k: torch.Tensor, v: torch.Tensor):
        """(strides of k, of v, T_new); (None,) where the rows have to be copied first."""
        shape = tuple(k.shape)
        if len(shape) != 4 or shape[:2] != (self.batch, self.n_kv_heads) or shape[3] != self.head_dim or v.shape != k.shape:
            raise ValueError(f"k and v must be ({self.batch}, {self.n_kv_heads}, T_new, {self.head_dim})")
        if k.dtype != self.dtype or v.dtype != self.dtype:
            raise ValueError(f"k and v must be {self.dtype} as the cache")
        L.require_cuda(k, v, self.k)
        if not (_on_grid(k) and _on_grid(v)):
            return (None,)
        return L.strides3(k), L.strides3(v), shape[2]

    def attend(self, q: torch.Tensor, *, scale: Optional[float] = None, accumulate: bool = True,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``o (B, H_q, 1, D)`` of one query token per sequence over the slots in use; with
        ``accumulate`` each slot's mass grows by its weights, summed over its group's heads."""
        if L.current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.attend(q, scale=scale, accumulate=accumulate, out=out)
        shape = q.shape
        key = (shape, q.stride(), q.dtype, q.get_device())
        plan = self._plans.get(key)
        if plan is None:
            plan = self._keep(key, self._plan_attend(q))
        hq, strides, dense, packed, need = plan
        if strides is None or q.data_ptr() & 15:  # rows off the 16-byte grid
            return self.attend(q.clone(memory_format=torch.contiguous_format), scale=scale, accumulate=accumulate, out=out)
        if out is None:
            out, out_strides = (torch.empty_like(q) if dense else q.new_empty(shape)), packed
        else:
            L.require_cuda(out, self.k)
            if out.shape != shape or out.dtype != self.dtype or out.stride(3) != 1:
                raise ValueError("out must have q's shape and dtype with contiguous channels")
            out_strides = L.strides2(out)
        stream = L.raw_stream(self._index)
        scratch = self._scratch.get((stream, need)) or self._new_scratch(stream, need)
        L.check(self._lib.linattn_heavy_attend(
            self._ref, q.data_ptr(), hq, strides, self._scale if scale is None else float(scale), 1 if accumulate else 0,
            out.data_ptr(), out_strides, scratch[0], scratch[1], need, self._status_ptr, stream))
        if L.strict():
            L.check_status(self.device)
        return out

    def _new_scratch(self, stream: int, need: int):
        """Workspace and arrival counts of attend() on a stream, kept: a graph may hold them."""
        tickets = self._stream_tickets.get(stream)
        if tickets is None:
            taken = len(self._stream_tickets)
            if taken < _STREAMS:
                tickets = self._unit_tickets[taken]
            elif torch.cuda.is_current_stream_capturing():  # zeros would be there after a replay only
                raise RuntimeError(f"attend() has run on {taken} streams: call it once on this one before capturing it")
            else:
                tickets = torch.zeros_like(self._unit_tickets[0])
                self._unit_tickets.append(tickets)
            self._stream_tickets[stream] = tickets
        workspace = torch.empty(need, dtype=torch.uint8, device=self.device)
        scratch = self._scratch[stream, need] = (tickets.data_ptr(), workspace.data_ptr(), workspace)
        return scratch

    def _plan_attend(self, q: torch.Tensor):
        """(H_q, strides of q or None where the rows have to be copied first, whether q is
        contiguous, strides of a new output, workspace bytes)."""
        shape = tuple(q.shape)
        if (len(shape) != 4 or shape[0] != self.batch or shape[1] < 1 or shape[1] % self.n_kv_heads
                or shape[2:] != (1, self.head_dim)):
            raise ValueError(f"q must be ({self.batch}, a multiple of {self.n_kv_heads}, 1, {self.head_dim}), got {shape}")
        if q.dtype != self.dtype:
            raise ValueError(f"q must be {self.dtype} as the cache")
        L.require_cuda(q, self.k)
        return (shape[1], L.strides2(q) if _on_grid(q) else None, q.is_contiguous(), L.i64_array((shape[1] * self.head_dim, self.head_dim)),
                self._lib.linattn_heavy_attend_workspace(self.batch, shape[1], self.n_kv_heads, self.budget))

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: Optional[float] = None,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One decode step: :meth:`append` the new token, then :meth:`attend` with its query."""
        self.append(k, v)
        return self.attend(q, scale=scale, out=out)


def _on_grid(x: torch.Tensor) -> bool:
    """Contiguous channels and strides of whole 16-byte pieces."""
    *outer, last = x.stride()
    return last == 1 and all(s & 7 == 0 for s in outer)


def _rows16(x: torch.Tensor) -> torch.Tensor:
    """x with contiguous channels and rows on 16 bytes."""
    return x if _on_grid(x) and x.data_ptr() & 15 == 0 else x.clone(memory_format=torch.contiguous_format)
