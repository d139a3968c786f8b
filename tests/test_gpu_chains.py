"""Kernels that start ahead of the previous one's end, without the pause that the strict mode
makes after every call: results are those of the same calls one at a time."""

from __future__ import annotations

import math

import pytest
import torch

from tests import test_gpu_heavy, test_gpu_packed

pytestmark = pytest.mark.gpu


@pytest.fixture
def no_pauses(cuda, monkeypatch):
    monkeypatch.setenv("LINATTN_B200_STRICT", "0")
    return cuda


def _listed(b, hq, hkv, d, pages, size, n, tq=1):
    """q, contiguous K and V, lists of n of their pages, and the attention over these."""
    g = torch.Generator(device="cuda").manual_seed(pages)
    q = torch.randn(b, hq, tq, d, generator=g, device="cuda").to(torch.bfloat16)
    k, v = (torch.randn(b, hkv, pages * size, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    ids = torch.rand(b, hkv, tq, pages, generator=g, device="cuda").argsort(-1)[..., :n].to(torch.int32).contiguous()
    return q, k, v, ids


@pytest.mark.parametrize("splits", [1, 3])
def test_sparse_attention_on_one_workspace(no_pauses, splits):
    """Calls right behind one another that share a workspace, and so the counter that hands out
    the work: it is cleared for a call only after the call before has ended."""
    from linattn_b200.block_sparse import kv_contiguous, lists_desc, sparse_attention

    b, hq, hkv, d, pages, size, n, tq = 2, 8, 2, 128, 40, 64, 24, 96
    q, k, v, ids = _listed(b, hq, hkv, d, pages, size, n, tq)
    kv, lists = kv_contiguous(k, v, size), lists_desc(ids, hkv)
    work = torch.empty(1 << 24, dtype=torch.float32, device="cuda")
    want = sparse_attention(q, kv, lists, n_splits=splits, workspace=work)
    torch.cuda.synchronize()
    assert want.isfinite().all()
    outs = [torch.full_like(q, math.nan) for _ in range(40)]
    for o in outs:
        sparse_attention(q, kv, lists, out=o, n_splits=splits, workspace=work)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_sparse_attention_over_the_last_queries_memory(no_pauses):
    """A workspace in the memory of the query that the cache's attend still reads (as an
    allocator hands it out again)."""
    from linattn_b200.block_sparse import kv_contiguous, lists_desc, sparse_attention

    cache, g = test_gpu_heavy._filled(16, 8, 128, 3000, torch.bfloat16, 8)
    hq = 32
    work = torch.empty(1 << 22, dtype=torch.float32, device="cuda")
    q = work.view(torch.bfloat16)[: 16 * hq * 128].view(16, hq, 1, 128)
    values = torch.randn(q.shape, generator=g, device="cuda").to(torch.bfloat16)
    q2, k, v, ids = _listed(2, 8, 2, 128, 40, 64, 24)
    kv, lists = kv_contiguous(k, v, 64), lists_desc(ids, 2)
    want, want2 = cache.attend(values, accumulate=False), sparse_attention(q2, kv, lists, n_splits=1)
    for _ in range(20):
        q.copy_(values)
        o = cache.attend(q, accumulate=False)
        o2 = sparse_attention(q2, kv, lists, n_splits=1, workspace=work)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(o2, want2)


def test_heavy_steps_without_pauses(no_pauses):
    test_gpu_heavy.test_steps_right_after_one_another(no_pauses)


def test_packed_calls_without_pauses(no_pauses):
    test_gpu_packed.test_packed_after_its_producers(no_pauses)
