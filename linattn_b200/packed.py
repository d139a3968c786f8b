"""Whole prompts in one packed batch: causal attention, and the weight each key received.

* ``packed_attention``: causal attention with grouped heads over sequences laid out one
  after the other (``dense_attention`` of each, ``src/linattn/core.py:148-181``), on the
  tcgen05 tensor cores; queries may be a chunk at the end of longer keys.
* ``attention_mass``: for every key the softmax weight it got, summed over the queries
  that read it and its group's heads: what a cache of heavy hitters
  (:class:`linattn_b200.HeavyCache`) keeps tokens by.

Packed layout: ``q (N_q, H_q, D)``, ``k, v (N_k, H_kv, D)``, offsets ``cu_q, cu_k`` int32
``(S + 1,)`` on the device.  Nothing is read back from the device.
"""

from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch

from linattn_b200 import _lib as L

__all__ = ["packed_attention", "attention_mass"]


def _rows(name: str, x: torch.Tensor) -> torch.Tensor:
    """x with contiguous channels and 16-byte rows, as the tensor maps read it."""
    if x.dim() != 3:
        raise ValueError(f"{name} must be (tokens, heads, head_dim), got shape {tuple(x.shape)}")
    s0, s1, s2 = x.stride()
    if s2 != 1 or (s0 | s1) & 7 or s0 < 1 or s1 < 1 or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)  # (contiguous() may hand back an unaligned view)
    return x


def _offsets(name: str, cu: torch.Tensor) -> int:
    if cu.dtype != torch.int32 or cu.dim() != 1 or cu.numel() < 1 or not cu.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector of sequence offsets (S + 1)")
    return cu.numel() - 1


def _packed(q, k, cu_q, cu_k, max_q, max_k):
    """The checked arguments that both operators share."""
    if q.dtype != k.dtype:
        raise ValueError("q and k must have one dtype")
    q, k = _rows("q", q), _rows("k", k)
    nq, hq, d = q.shape
    nk, hkv, dk = k.shape
    if d != dk:
        raise ValueError(f"head_dim of q and k differ: {d} and {dk}")
    s = _offsets("cu_q", cu_q)
    if cu_k is None:
        if nq != nk:
            raise ValueError("without cu_k, q and k must hold the same tokens")
        cu_k = cu_q
    elif _offsets("cu_k", cu_k) != s:
        raise ValueError("cu_q and cu_k must describe the same number of sequences")
    return (q, k, cu_k, s, nq, nk, hq, hkv, d, nq if max_q is None else min(int(max_q), nq),
            nk if max_k is None else min(int(max_k), nk))


@functools.lru_cache(maxsize=1024)
def _attention_plan(device: int, nq: int, hq: int, hkv: int, d: int, s: int, max_q: int, max_k: int, n_splits: int):
    """(splits, workspace bytes); ``n_splits`` 0: the library's choice."""
    lib = L.lib()
    n = n_splits or lib.linattn_packed_attention_splits(nq, hq, hkv, s, max_q, max_k)
    return n, lib.linattn_packed_attention_workspace(nq, hq, d, n)


@functools.lru_cache(maxsize=1024)
def _mass_plan(device: int, nk: int, hq: int, hkv: int, s: int, max_q: int, max_k: int, window: int, n_splits: int):
    lib = L.lib()
    n = n_splits or lib.linattn_attention_mass_splits(hq, hkv, s, max_q, max_k, window)
    return n, lib.linattn_attention_mass_workspace(nk, hkv, n)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                     cu_k: Optional[torch.Tensor] = None, *, max_q: Optional[int] = None, max_k: Optional[int] = None,
                     causal: bool = True, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     lse_out: Optional[torch.Tensor] = None, n_splits: Optional[int] = None,
                     workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(o (N_q, H_q, D), lse (N_q, H_q) fp32)`` of packed sequences, bf16 or f16, D 64 or 128.

    Sequence ``s`` owns the query rows ``cu_q[s] : cu_q[s + 1]`` and the key rows ``cu_k[s] :
    cu_k[s + 1]`` (``cu_k`` None: the same); its last query stands at its last key, so query
    ``i`` reads keys ``j <= i + len_k - len_q`` (every key with ``causal=False``).  A query with
    nothing to read gets ``o = 0``, ``lse = -inf``.  A key past the sequence's end never reaches
    its outputs, whatever it holds; a later key of the same sequence must be finite.

    ``max_q`` / ``max_k``: the longest sequence's query / key rows, where the caller knows them
    (they size the grid; the default is all rows).  ``n_splits`` (default: chosen) cuts the key
    ranges when there are few rows; ``workspace``: fp32 scratch for it, allocated if None."""
    dev = L.require_cuda(q, k, v, cu_q, cu_k, out, lse_out, workspace)
    q, k, cu_k, s, nq, nk, hq, hkv, d, max_q, max_k = _packed(q, k, cu_q, cu_k, max_q, max_k)
    if v.dtype != k.dtype or v.shape != k.shape:
        raise ValueError("k and v must have one dtype and shape")
    v = _rows("v", v)
    if out is None:
        out = torch.empty((nq, hq, d), dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError("out must have q's shape and dtype with contiguous channels")
    if lse_out is None:
        lse_out = torch.empty((nq, hq), dtype=torch.float32, device=dev)
    elif lse_out.shape != (nq, hq) or lse_out.dtype != torch.float32 or not lse_out.is_contiguous():
        raise ValueError("lse_out must be a contiguous fp32 (N_q, H_q) tensor")
    n_splits, ws_bytes = _attention_plan(dev.index, nq, hq, hkv, d, s, max_q, max_k, n_splits or 0)
    if n_splits > 1:
        if workspace is None:
            workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        ws_bytes = workspace.numel() * workspace.element_size()
    L.check(L.lib().linattn_packed_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), L.dtype_code(q), nq, nk, hq, hkv, d, L.strides2(q), L.strides2(k),
        L.strides2(v), cu_q.data_ptr(), cu_k.data_ptr(), s, max_q, max_k, int(causal),
        d ** -0.5 if scale is None else float(scale), out.data_ptr(), L.strides2(out), lse_out.data_ptr(),
        n_splits, L.ptr(workspace), ws_bytes, L.status_word(dev).data_ptr(), L.raw_stream(dev.index)))
    if L.strict():
        L.check_status(dev)
    return out, lse_out


def attention_mass(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, cu_q: torch.Tensor,
                   cu_k: Optional[torch.Tensor] = None, *, max_q: Optional[int] = None, max_k: Optional[int] = None,
                   causal: bool = True, window: int = 0, scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None, n_splits: Optional[int] = None,
                   workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``mass (H_kv, N_k)`` fp32: ``mass[h, j]`` sums ``exp(scale q_i . k_j - lse_i)`` over the
    queries that read key ``j`` and the query heads of kv head ``h``.  ``lse (N_q, H_q)`` as
    :func:`packed_attention` returns it for the same ``q, k`` and offsets.  ``window > 0``:
    only each sequence's last ``window`` queries count.  The sums have a fixed order."""
    dev = L.require_cuda(q, k, lse, cu_q, cu_k, out, workspace)
    q, k, cu_k, s, nq, nk, hq, hkv, d, max_q, max_k = _packed(q, k, cu_q, cu_k, max_q, max_k)
    if lse.shape != (nq, hq) or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous fp32 (N_q, H_q) tensor")
    if window < 0:
        raise ValueError("window must be >= 0")
    if out is None:
        out = torch.empty((hkv, nk), dtype=torch.float32, device=dev)
    elif out.shape != (hkv, nk) or out.dtype != torch.float32 or out.stride(1) != 1:
        raise ValueError("out must be an fp32 (H_kv, N_k) tensor with contiguous rows")
    n_splits, ws_bytes = _mass_plan(dev.index, nk, hq, hkv, s, max_q, max_k, int(window), n_splits or 0)
    if n_splits > 1:
        if workspace is None:
            workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        ws_bytes = workspace.numel() * workspace.element_size()
    L.check(L.lib().linattn_attention_mass(
        q.data_ptr(), k.data_ptr(), L.dtype_code(q), nq, nk, hq, hkv, d, L.strides2(q), L.strides2(k), lse.data_ptr(),
        cu_q.data_ptr(), cu_k.data_ptr(), s, max_q, max_k, int(causal), int(window),
        d ** -0.5 if scale is None else float(scale), out.data_ptr(), out.stride(0), n_splits,
        L.ptr(workspace), ws_bytes, L.status_word(dev).data_ptr(), L.raw_stream(dev.index)))
    if L.strict():
        L.check_status(dev)
    return out
