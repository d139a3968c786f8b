"""Launches go to the tensors' device, whichever is current (one GPU: the current device and the
guard that changes it are stood in for)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def other_device(cuda, monkeypatch):
    """Another device seems to be current; every look at the current stream notes which one is."""
    from linattn_b200 import _lib as L

    monkeypatch.setenv("LINATTN_B200_STRICT", "0")
    state = {"now": 1, "launches": []}

    class Guard:
        def __init__(self, device):
            self.index = device if isinstance(device, int) else device.index

        def __enter__(self):
            self.before, state["now"] = state["now"], self.index

        def __exit__(self, *_):
            state["now"] = self.before

    stream = L.raw_stream

    def raw_stream(index):
        state["launches"].append(state["now"] == index)
        return stream(index)

    monkeypatch.setattr(L, "current_device", lambda: state["now"])
    monkeypatch.setattr(L, "raw_stream", raw_stream)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    return state


def test_launches_go_to_the_tensors_device(other_device):
    from linattn_b200 import HeavyCache, attention_mass, packed_attention

    d, n = 64, 90
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(n, h, d, generator=g, device="cuda").half() for h in (4, 2, 2))
    new = torch.randn(2, 1, 2, 1, d, generator=g, device="cuda").half()
    one = torch.randn(1, 4, 1, d, generator=g, device="cuda").half()
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    results = []
    for current in (0, 1):
        other_device["now"] = current
        o, lse = packed_attention(q, k, v, cu)
        mass = attention_mass(q, k, lse, cu)
        cache = HeavyCache(1, 2, d, 32, dtype=torch.float16)
        cache.load(k, v, mass, cu)
        results.append([o, lse, mass, cache.step(one, new[0], new[1]), cache.mass.clone(), cache.seen.clone()])
        assert other_device["now"] == current
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert len(other_device["launches"]) == 10 and all(other_device["launches"])
