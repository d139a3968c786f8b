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

from typing import NamedTuple, Optional, Tuple

import torch

from linattn_b200 import _lib as L

__all__ = ["packed_attention", "attention_mass"]


_PLANS: dict = {}  # checked arguments by shapes, strides and types (nothing of their contents or addresses)


class _Plan(NamedTuple):
    s: int
    nq: int
    nk: int
    hq: int
    hkv: int
    d: int
    max_q: int
    max_k: int
    n_splits: int
    ws_bytes: int
    dtype: int
    device: torch.device
    index: int         # of the device
    copies: tuple      # operands whose rows have to be copied first
    strides: tuple     # of the operands, as the library takes them
    out_strides: object
    dense: bool        # q is contiguous


def _layout(x):
    return None if x is None else (x.shape, x.stride(), x.dtype, x.get_device())


def _offsets(name: str, cu: torch.Tensor) -> int:
    if cu.dtype != torch.int32 or cu.dim() != 1 or cu.numel() < 1 or not cu.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector of sequence offsets (S + 1)")
    return cu.numel() - 1


def _on_grid(x: torch.Tensor) -> bool:
    """Contiguous channels and strides of whole 16-byte pieces, as the tensor maps read it."""
    s0, s1, s2 = x.stride()
    return s2 == 1 and not (s0 | s1) & 7 and s0 > 0 and s1 > 0


def _plan(q, k, v, cu_q, cu_k, max_q, max_k, window, n_splits) -> _Plan:
    """The checked arguments of attention (``window`` None) or mass (``v`` None)."""
    dev = L.require_cuda(q, k, v, cu_q, cu_k)
    operands = [("q", q), ("k", k)] + ([("v", v)] if v is not None else [])
    for name, x in operands:
        if x.dim() != 3:
            raise ValueError(f"{name} must be (tokens, heads, head_dim), got shape {tuple(x.shape)}")
    if q.dtype != k.dtype:
        raise ValueError("q and k must have one dtype")
    nq, hq, d = q.shape
    nk, hkv, dk = k.shape
    if d != dk:
        raise ValueError(f"head_dim of q and k differ: {d} and {dk}")
    if v is not None and (v.dtype != k.dtype or v.shape != k.shape):
        raise ValueError("k and v must have one dtype and shape")
    s = _offsets("cu_q", cu_q)
    if cu_k is None:
        if nq != nk:
            raise ValueError("without cu_k, q and k must hold the same tokens")
    elif _offsets("cu_k", cu_k) != s:
        raise ValueError("cu_q and cu_k must describe the same number of sequences")
    max_q = nq if max_q is None else min(int(max_q), nq)
    max_k = nk if max_k is None else min(int(max_k), nk)
    lib = L.lib()
    if window is None:
        n = n_splits or lib.linattn_packed_attention_splits(nq, hq, hkv, s, max_q, max_k)
        ws = lib.linattn_packed_attention_workspace(nq, hq, d, n)
    else:
        if window < 0:
            raise ValueError("window must be >= 0")
        n = n_splits or lib.linattn_attention_mass_splits(hq, hkv, s, max_q, max_k, window)
        ws = lib.linattn_attention_mass_workspace(nk, hkv, n)
    copies = tuple(not _on_grid(x) for _, x in operands)
    # a copy is contiguous
    strides = tuple(L.i64_array((x.shape[1] * d, d)) if c else L.strides2(x) for c, (_, x) in zip(copies, operands))
    return _Plan(s, nq, nk, hq, hkv, d, max_q, max_k, n, ws, L.dtype_code(q), dev, dev.index, copies, strides,
                 L.i64_array((hq * d, d)), q.is_contiguous())


def _planned(key, *args) -> _Plan:
    plan = _PLANS.get(key)
    if plan is None:
        if len(_PLANS) >= 1024:
            _PLANS.clear()
        plan = _PLANS[key] = _plan(*args)
    return plan


def _aligned(x: torch.Tensor, copy: bool, strides, plan: _Plan):
    """x on the 16-byte grid (a copy where it is not) and its strides."""
    if not copy and x.data_ptr() & 15 == 0:
        return x, strides
    return x.clone(memory_format=torch.contiguous_format), L.i64_array((x.shape[1] * plan.d, plan.d))


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
    (they size the grid; the default is all rows).  Rows of no sequence (padding of a fixed
    buffer) and rows of one beyond its first ``max_q`` are not written.  ``n_splits`` (default:
    chosen) cuts the key ranges when there are few rows; one part of 2^20 keys of like weight is
    2.6e-3 off (fp32 sums on the tensor cores, in proportion to the keys), so cut longer ranges.
    ``workspace``: fp32 scratch for the parts, allocated if None."""
    p = _planned((_layout(q), _layout(k), _layout(v), _layout(cu_q), _layout(cu_k), max_q, max_k, None, n_splits),
                 q, k, v, cu_q, cu_k, max_q, max_k, None, n_splits)
    if L.current_device() != p.index:
        with torch.cuda.device(p.index):
            return packed_attention(q, k, v, cu_q, cu_k, max_q=max_q, max_k=max_k, causal=causal, scale=scale, out=out,
                                    lse_out=lse_out, n_splits=n_splits, workspace=workspace)
    q, sq = _aligned(q, p.copies[0], p.strides[0], p)
    k, sk = _aligned(k, p.copies[1], p.strides[1], p)
    v, sv = _aligned(v, p.copies[2], p.strides[2], p)
    out_strides = p.out_strides
    if out is None:
        out = torch.empty_like(q) if p.dense else q.new_empty((p.nq, p.hq, p.d))
    else:
        L.require_cuda(q, out)
        if out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
            raise ValueError("out must have q's shape and dtype with contiguous channels")
        out_strides = L.strides2(out)
    if lse_out is None:
        lse_out = q.new_empty((p.nq, p.hq), dtype=torch.float32)
    elif lse_out.shape != (p.nq, p.hq) or lse_out.dtype != torch.float32 or not lse_out.is_contiguous() or lse_out.device != p.device:
        raise ValueError("lse_out must be a contiguous fp32 (N_q, H_q) tensor on q's device")
    ws_bytes = p.ws_bytes
    if p.n_splits > 1:
        if workspace is None:
            workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=p.device)
        L.require_cuda(q, workspace)
        ws_bytes = workspace.numel() * workspace.element_size()
    L.check(L.lib().linattn_packed_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), p.dtype, p.nq, p.nk, p.hq, p.hkv, p.d, sq, sk, sv, cu_q.data_ptr(),
        (cu_q if cu_k is None else cu_k).data_ptr(), p.s, p.max_q, p.max_k, 1 if causal else 0,
        p.d ** -0.5 if scale is None else float(scale), out.data_ptr(), out_strides, lse_out.data_ptr(),
        p.n_splits, L.ptr(workspace), ws_bytes, L.status_word(p.device).data_ptr(), L.raw_stream(p.index)))
    if L.strict():
        L.check_status(p.device)
    return out, lse_out


def attention_mass(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, cu_q: torch.Tensor,
                   cu_k: Optional[torch.Tensor] = None, *, max_q: Optional[int] = None, max_k: Optional[int] = None,
                   causal: bool = True, window: int = 0, scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None, n_splits: Optional[int] = None,
                   workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``mass (H_kv, N_k)`` fp32: ``mass[h, j]`` sums ``exp(scale q_i . k_j - lse_i)`` over the
    queries that read key ``j`` and the query heads of kv head ``h``.  ``lse (N_q, H_q)`` as
    :func:`packed_attention` returns it for the same ``q, k`` and offsets.  ``window > 0``:
    only each sequence's last ``window`` queries count.  The sums have a fixed order.
    Keys of no sequence, and keys of one beyond its first ``max_k``, are not written.  A row
    whose lse is -inf (it read nothing) or +inf adds nothing."""
    p = _planned((_layout(q), _layout(k), None, _layout(cu_q), _layout(cu_k), max_q, max_k, window, n_splits),
                 q, k, None, cu_q, cu_k, max_q, max_k, window, n_splits)
    if L.current_device() != p.index:
        with torch.cuda.device(p.index):
            return attention_mass(q, k, lse, cu_q, cu_k, max_q=max_q, max_k=max_k, causal=causal, window=window, scale=scale,
                                  out=out, n_splits=n_splits, workspace=workspace)
    q, sq = _aligned(q, p.copies[0], p.strides[0], p)
    k, sk = _aligned(k, p.copies[1], p.strides[1], p)
    if lse.shape != (p.nq, p.hq) or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != p.device:
        raise ValueError("lse must be a contiguous fp32 (N_q, H_q) tensor on q's device")
    if out is None:
        out = q.new_empty((p.hkv, p.nk), dtype=torch.float32)
    elif out.shape != (p.hkv, p.nk) or out.dtype != torch.float32 or out.stride(1) != 1 or out.device != p.device:
        raise ValueError("out must be an fp32 (H_kv, N_k) tensor with contiguous rows on q's device")
    ws_bytes = p.ws_bytes
    if p.n_splits > 1:
        if workspace is None:
            workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=p.device)
        L.require_cuda(q, workspace)
        ws_bytes = workspace.numel() * workspace.element_size()
    L.check(L.lib().linattn_attention_mass(
        q.data_ptr(), k.data_ptr(), p.dtype, p.nq, p.nk, p.hq, p.hkv, p.d, sq, sk, lse.data_ptr(), cu_q.data_ptr(),
        (cu_q if cu_k is None else cu_k).data_ptr(), p.s, p.max_q, p.max_k, 1 if causal else 0, int(window),
        p.d ** -0.5 if scale is None else float(scale), out.data_ptr(), out.stride(0), p.n_splits, L.ptr(workspace),
        ws_bytes, L.status_word(p.device).data_ptr(), L.raw_stream(p.index)))
    if L.strict():
        L.check_status(p.device)
    return out
