"""Packed attention and the heavy-hitter cache at the C boundary: bad arguments are turned
away on the host before any launch (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from linattn_b200 import _lib as L

P = ctypes.c_void_p(4096)
I2, I3 = (L.c_i64 * 2)(128, 128), (L.c_i64 * 3)(128, 128, 128)


def _attention(**kw):
    a = dict(q=P, k=P, v=P, dtype=L.BF16, nq=64, nk=64, hq=8, hkv=2, d=128, qs=I2, ks=I2, vs=I2, cu_q=P, cu_k=P, s=1,
             max_q=64, max_k=64, causal=1, scale=0.1, out=P, os=I2, lse=P, splits=1, ws=None, ws_bytes=0, status=None,
             stream=None)
    a.update(kw)
    return L.lib().linattn_packed_attention(*a.values())


def _mass(**kw):
    a = dict(q=P, k=P, dtype=L.BF16, nq=64, nk=64, hq=8, hkv=2, d=128, qs=I2, ks=I2, lse=P, cu_q=P, cu_k=P, s=1, max_q=64,
             max_k=64, causal=1, window=0, scale=0.1, mass=P, stride=64, splits=1, ws=None, ws_bytes=0, status=None,
             stream=None)
    a.update(kw)
    return L.lib().linattn_attention_mass(*a.values())


@pytest.mark.parametrize("call", [_attention, _mass])
@pytest.mark.parametrize("bad,rc", [
    (dict(q=None), 1), (dict(cu_q=None), 1), (dict(dtype=L.F32), 2), (dict(d=96), 2), (dict(hq=9), 1),
    (dict(hq=258, hkv=2), 2), (dict(nq=-1), 1), (dict(s=-1), 1), (dict(scale=0.0), 1), (dict(scale=float("nan")), 1),
    (dict(q=ctypes.c_void_p(4098)), 1), (dict(ks=(L.c_i64 * 2)(129, 128)), 1), (dict(splits=0), 1),
    (dict(splits=2), 1), (dict(nk=1 << 30), 2),
])
def test_packed_arguments(call, bad, rc):
    assert call(**bad) == rc
    assert L.lib().linattn_last_error()


def test_packed_nothing_to_do():
    assert _attention(nq=0) == 0
    assert _attention(s=0) == 0
    assert _mass(nk=0) == 0
    assert _mass(s=0) == 0


def test_packed_plans():
    lib = L.lib()
    assert lib.linattn_packed_attention_workspace(100, 8, 128, 1) == 0
    assert lib.linattn_packed_attention_workspace(100, 8, 128, 3) == 3 * 100 * 8 * 129 * 4
    assert lib.linattn_attention_mass_workspace(100, 2, 1) == 0
    assert lib.linattn_attention_mass_workspace(100, 2, 4) == 4 * 100 * 2 * 4
    for args in ((0, 8, 2, 1, 0, 0), (64, 8, 2, 1, 64, 64), (64, 8, 2, 1, 64, 0)):
        assert lib.linattn_packed_attention_splits(*args) == 1
    assert lib.linattn_attention_mass_splits(8, 2, 0, 0, 0, 0) == 1


def _heavy(**kw):
    a = dict(k=4096, v=4096, mass=4096, pos=4096, seen=4096, dtype=L.F16, batch=2, n_kv_heads=2, budget=64, head_dim=64,
             sinks=1, recent=8, maps=None)
    a.update(kw)
    return L.Heavy(*a.values())


@pytest.mark.parametrize("bad,rc", [
    (dict(k=None), 1), (dict(dtype=L.FP8E4M3), 2), (dict(batch=0), 1), (dict(budget=0), 1), (dict(budget=1 << 25), 2),
    (dict(head_dim=4), 2), (dict(sinks=-1), 1), (dict(recent=0), 1), (dict(sinks=60), 1), (dict(mass=4100), 1),
])
def test_heavy_cache_arguments(bad, rc):
    lib = L.lib()
    assert lib.linattn_heavy_append(_heavy(**bad), P, P, I3, I3, 1, P, None, None) == rc
    assert lib.linattn_heavy_load(_heavy(**bad), P, P, I2, I2, 10, P, 10, P, None, 1, None, None) == rc


def test_heavy_calls():
    lib = L.lib()
    assert lib.linattn_heavy_maps(_heavy(dtype=L.F32), P) == 2
    assert lib.linattn_heavy_maps(_heavy(), None) == 1
    assert lib.linattn_heavy_append(_heavy(), None, P, I3, I3, 1, P, None, None) == 1
    assert lib.linattn_heavy_append(_heavy(), P, P, (L.c_i64 * 3)(4, 64, 64), I3, 1, P, None, None) == 1
    assert lib.linattn_heavy_append(_heavy(), P, P, I3, I3, -1, P, None, None) == 1
    assert lib.linattn_heavy_append(_heavy(), P, P, I3, I3, 0, P, None, None) == 0
    assert lib.linattn_heavy_load(_heavy(), P, P, I2, I2, 10, P, 10, P, None, 3, None, None) == 1  # more than rows
    assert lib.linattn_heavy_load(_heavy(), P, P, I2, I2, 10, None, 10, P, None, 1, None, None) == 1
    assert lib.linattn_heavy_load(_heavy(), P, P, I2, I2, 10, P, 10, P, None, 0, None, None) == 0
    bad = [dict(cache=_heavy(dtype=L.F32)), dict(cache=_heavy(head_dim=128 + 64)), dict(hq=3), dict(scale=-1.0), dict(q=None),
           dict(qs=(L.c_i64 * 2)(64, 63)), dict(ticket=None), dict(ws=None), dict(ws_bytes=64)]
    for b in bad:
        a = dict(cache=_heavy(), q=P, hq=4, qs=(L.c_i64 * 2)(256, 64), scale=0.1, acc=1, out=P, os=(L.c_i64 * 2)(256, 64),
                 ticket=P, ws=P, ws_bytes=1 << 30, status=None, stream=None)
        a.update(b)
        assert lib.linattn_heavy_attend(*a.values()) in (1, 2)


def test_operators_refuse_cpu_tensors():
    from linattn_b200 import HeavyCache, attention_mass, packed_attention

    q, cu = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        packed_attention(q, q, q, cu)
    with pytest.raises(ValueError, match="CUDA"):
        attention_mass(q, q, torch.zeros(4, 2), cu)
    with pytest.raises(ValueError, match="cuda"):
        HeavyCache(1, 1, 64, 8, device="cpu")


def test_heavy_append_of_no_tokens():
    """An empty tensor's address is NULL: nothing to do, not an error."""
    lib = L.lib()
    assert lib.linattn_heavy_append(_heavy(), None, None, I3, I3, 0, P, None, None) == 0
    assert lib.linattn_heavy_append(_heavy(budget=0), None, None, I3, I3, 0, P, None, None) == 1
