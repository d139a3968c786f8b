"""Prompts to a cache of heavy hitters, then decoding from it: one attention layer's part of
a serving loop, on random inputs.

    python examples/heavy_hitter_decode.py --lens 6000,900,3500 --budget 1024 --tokens 64

The prompts run packed (``packed_attention``), their keys' attention masses decide what the
cache keeps (``attention_mass``, ``HeavyCache.load``), and every decoded token replaces the
slot that has mattered least (``HeavyCache.step``, captured once as a CUDA graph).
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from linattn_b200 import HeavyCache, attention_mass, packed_attention  # noqa: E402


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--lens", default="6000,900,3500")
    ap.add_argument("--budget", type=int, default=1024)
    ap.add_argument("--sinks", type=int, default=4)
    ap.add_argument("--recent", type=int, default=256)
    ap.add_argument("--window", type=int, default=0, help="prompt queries that vote (0: all)")
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--head-dim", type=int, default=128)
    a = ap.parse_args(argv)
    lens = [int(x) for x in a.lens.split(",")]
    b, n, hq, hkv, d = len(lens), sum(lens), a.heads, a.kv_heads, a.head_dim
    gen = torch.Generator(device="cuda").manual_seed(0)

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(torch.bfloat16)

    # prompts: sequences one after the other
    q, k, v = rand(n, hq, d), rand(n, hkv, d), rand(n, hkv, d)
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    longest = max(lens)
    o, lse = packed_attention(q, k, v, cu, max_q=longest, max_k=longest)
    mass = attention_mass(q, k, lse, cu, max_q=longest, max_k=longest, window=a.window)
    cache = HeavyCache(b, hkv, d, a.budget, sinks=a.sinks, recent=a.recent)
    cache.load(k, v, mass, cu)

    # decode: the step's buffers are fixed, so it replays as one graph
    q1, k1, v1, out = rand(b, hq, 1, d), rand(b, hkv, 1, d), rand(b, hkv, 1, d), rand(b, hq, 1, d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.step(q1, k1, v1, out=out)  # once outside the capture
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.step(q1, k1, v1, out=out)
    tokens = [(rand(b, hq, 1, d), rand(b, hkv, 1, d), rand(b, hkv, 1, d)) for _ in range(a.tokens - 1)]
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for new in tokens:
        for buf, x in zip((q1, k1, v1), new):
            buf.copy_(x)
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    used = cache.seen.clamp(max=a.budget).tolist()
    res = {"prompt_tokens": n, "decoded": a.tokens, "seen": cache.seen.tolist(), "slots_used": used,
           "kept_of_prompt": [int((cache.pos[i, 0, :u] < m).sum()) for i, (u, m) in enumerate(zip(used, lens))],
           "us_per_step": 1e3 * start.elapsed_time(end) / max(1, a.tokens - 1), "finite": bool(o.isfinite().all() and out.isfinite().all())}
    print(res)
    return res


if __name__ == "__main__":
    main()
