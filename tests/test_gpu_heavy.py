"""The heavy-hitter cache: load and append bit for bit against plain Python, attend against
float64 (tolerances: the output's rounding u |o|, the weights' error e A from fp32 scores of
D exact products and a hi + lo split of 2^-16; masses by the same e)."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _cu(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def _order(mass):
    """Sort key of one mass: NaN above everything."""
    return math.inf if mass != mass else mass, mass != mass


def _kept(mass, budget, sinks, recent):
    n = len(mass)
    if n <= budget:
        return list(range(n))
    rest = sorted(range(sinks, n - recent), key=lambda i: (_order(mass[i])[1], _order(mass[i])[0], -i), reverse=True)
    return sorted(list(range(sinks)) + rest[: budget - sinks - recent] + list(range(n - recent, n)))


LOADS = [
    # lens, budget, sinks, recent, H, D, dtype
    ([1, 0, 7, 8, 9], 8, 1, 2, 2, 64, torch.bfloat16),
    ([100, 640, 33], 32, 4, 8, 3, 128, torch.float16),
    ([5000, 4097], 1000, 0, 1, 2, 64, torch.float16),
    ([700], 64, 4, 60, 1, 128, torch.bfloat16),      # nothing is left to choose
    ([900, 2], 257, 3, 200, 2, 64, torch.bfloat16),
    ([70001], 300, 2, 30, 1, 64, torch.float16),     # more tokens than a CTA's registers hold
    ([20000], 12000, 4, 4000, 2, 64, torch.bfloat16),
]


@pytest.mark.parametrize("case", range(len(LOADS)))
@pytest.mark.parametrize("kind", ["random", "ties", "nan", "zero"])
def test_load(cuda, case, kind):
    from linattn_b200 import HeavyCache

    lens, budget, sinks, recent, h, d, dtype = LOADS[case]
    g = torch.Generator().manual_seed(case)
    n = sum(lens)
    k, v = torch.randn(n, h, d, generator=g).to(dtype), torch.randn(n, h, d, generator=g).to(dtype)
    mass = torch.exp(torch.randn(h, n, generator=g))
    if kind == "ties":
        mass = (mass * 3).round()
    elif kind == "nan":
        mass[torch.rand(h, n, generator=g) < 0.05] = math.nan
        mass[torch.rand(h, n, generator=g) < 0.05] = math.inf
    elif kind == "zero":
        mass = torch.where(torch.rand(h, n, generator=g) < 0.5, 0.0, -0.0)
    b = len(lens) + 2
    rows = torch.randperm(b, generator=g)[: len(lens)].to(torch.int32)
    cache = HeavyCache(b, h, d, budget, sinks=sinks, recent=recent, dtype=dtype)
    cache.pos.fill_(-9)
    cache.seen.fill_(3)
    # K and V as strided views: heads outermost
    kk = k.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    cache.load(kk, v.cuda(), mass.cuda(), _cu(lens), rows.cuda())
    at = 0
    seen = torch.full((b,), 3)
    for s, m in enumerate(lens):
        r = int(rows[s])
        seen[r] = m
        for x in range(h):
            keep = _kept(mass[x, at:at + m].tolist(), budget, sinks, recent)
            idx = torch.tensor(keep, dtype=torch.long)
            c = len(keep)
            assert cache.pos[r, x, :c].tolist() == keep
            assert (cache.pos[r, x, c:] == -9).all()
            assert torch.equal(cache.k[r, x, :c].cpu(), k[at + idx, x])
            assert torch.equal(cache.v[r, x, :c].cpu(), v[at + idx, x])
            assert torch.equal(cache.mass[r, x, :c].cpu().nan_to_num(-1), mass[x, at + idx].nan_to_num(-1))
        at += m
    assert torch.equal(cache.seen.cpu().long(), seen)


@pytest.mark.parametrize("budget,sinks,recent,steps,t_new", [(7, 1, 2, 20, 1), (64, 4, 16, 90, 1), (13, 0, 1, 9, 5),
                                                             (32, 2, 30, 40, 3), (1, 0, 1, 4, 1)])
def test_append(cuda, budget, sinks, recent, steps, t_new):
    """Tokens one after the other, with masses that change in between as attention changes them."""
    from linattn_b200 import HeavyCache

    b, h, d, dtype = 3, 2, 64, torch.bfloat16
    g = torch.Generator().manual_seed(budget)
    cache = HeavyCache(b, h, d, budget, sinks=sinks, recent=recent, dtype=dtype)
    state = [[[] for _ in range(h)] for _ in range(b)]  # slots of (pos, mass, k, v)
    seen = 0
    for step in range(steps):
        k, v = torch.randn(b, h, t_new, d, generator=g).to(dtype), torch.randn(b, h, t_new, d, generator=g).to(dtype)
        cache.append(k.cuda().transpose(1, 2).contiguous().transpose(1, 2), v.cuda())
        for t in range(t_new):
            now = seen + t
            for i in range(b):
                for x in range(h):
                    slots = state[i][x]
                    new = [now, 0.0, k[i, x, t], v[i, x, t]]
                    if len(slots) < budget:
                        slots.append(new)
                    else:
                        may = [(m, s) for s, (p, m, _, _) in enumerate(slots) if sinks <= p <= now - recent]
                        slots[min(may)[1]] = new
        seen += t_new
        for i in range(b):
            for x in range(h):
                c = len(state[i][x])
                assert cache.pos[i, x, :c].tolist() == [p for p, _, _, _ in state[i][x]]
                assert cache.mass[i, x, :c].tolist() == [m for _, m, _, _ in state[i][x]]
                assert torch.equal(cache.k[i, x, :c].cpu(), torch.stack([y for _, _, y, _ in state[i][x]]))
                assert torch.equal(cache.v[i, x, :c].cpu(), torch.stack([y for _, _, _, y in state[i][x]]))
        assert cache.seen.tolist() == [seen] * b
        # few distinct weights, so that ties are common
        add = torch.randint(0, 3, cache.mass.shape, generator=g).float()
        cache.mass += add.cuda()
        for i in range(b):
            for x in range(h):
                for s, slot in enumerate(state[i][x]):
                    slot[1] += float(add[i, x, s])


def test_append_reports_slots_that_cannot_go(cuda, monkeypatch):
    from linattn_b200 import HeavyCache
    from linattn_b200 import _lib as L

    monkeypatch.setenv("LINATTN_B200_STRICT", "0")
    cache = HeavyCache(1, 1, 64, 8, sinks=2, recent=2, dtype=torch.float16)
    cache.seen.fill_(8)  # positions were never written: every slot says 0, a sink
    before = cache.k.clone()
    L.read_status(cuda)
    cache.append(torch.ones(1, 1, 1, 64, dtype=torch.float16, device="cuda"), torch.ones(1, 1, 1, 64, dtype=torch.float16, device="cuda"))
    assert L.read_status(cuda) & L.DEV_BAD_ID
    assert torch.equal(cache.k, before)


def _check_attend(cache, q, o, before, after, scale, accumulate):
    b, hq, _, d = q.shape
    g = hq // cache.n_kv_heads
    u = U[q.dtype]
    for i in range(b):
        n = min(int(cache.seen[i]), cache.budget)
        for x in range(cache.n_kv_heads):
            k, v = cache.k[i, x, :n].double(), cache.v[i, x, :n].double()
            add, slack = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
            for h in range(x * g, x * g + g):
                got = o[i, h, 0].double()
                if n == 0:
                    assert (got == 0).all()
                    continue
                y = q[i, h, 0].double()
                e = (d * 2.0 ** -24 * scale * (k.abs() @ y.abs())).max() + 2.0 ** -20
                p = torch.softmax(k @ y * scale, 0)
                want, mag = p @ v, p @ v.abs()
                tiny = n * 2.0 ** -25 * v.abs().max() if q.dtype == torch.float16 else 0.0
                assert ((got - want).abs() <= u * 1.01 * want.abs() + (2 * e + 2.0 ** -15) * mag + tiny).all()
                add += p
                slack += p * (4 * e)
            m0, m1 = before[i, x].double(), after[i, x].double()
            assert torch.equal(m0[n:], m1[n:])
            if accumulate:
                assert ((m1[:n] - m0[:n] - add).abs() <= slack + 2.0 ** -22 * (m0[:n] + add)).all()
            else:
                assert torch.equal(m0, m1)


@pytest.mark.parametrize("seen,budget,hq,hkv,d,dtype", [
    ([0, 1, 15, 16, 17, 500], 300, 8, 2, 128, torch.bfloat16),
    ([128, 129, 5], 129, 3, 3, 64, torch.float16),
    ([1000], 640, 24, 2, 128, torch.float16),          # G = 12
    ([77, 200], 100, 40, 1, 64, torch.bfloat16),       # G = 40: more heads than one pass takes
    ([6000, 3333], 5000, 10, 2, 128, torch.bfloat16),  # G = 5
    ([40000], 33000, 4, 1, 64, torch.float16),         # scores go through the workspace
])
@pytest.mark.parametrize("accumulate", [True, False])
def test_attend(cuda, seen, budget, hq, hkv, d, dtype, accumulate):
    from linattn_b200 import HeavyCache

    g = torch.Generator().manual_seed(budget)
    b = len(seen)
    cache = HeavyCache(b, hkv, d, budget, dtype=dtype)
    cache.k.copy_(torch.randn(b, hkv, budget, d, generator=g))
    cache.v.copy_(torch.randn(b, hkv, budget, d, generator=g))
    cache.mass.copy_(torch.rand(b, hkv, budget, generator=g))
    cache.seen.copy_(torch.tensor(seen))
    for i, n in enumerate(seen):  # slots that are not in use hold anything
        cache.k[i, :, n:] = math.nan
        cache.v[i, :, n:] = math.inf
    q = torch.randn(b, hq, 1, d, generator=g).to(dtype).cuda() * 2
    before = cache.mass.clone()
    scale = 0.9 / math.sqrt(d)
    o = cache.attend(q, scale=scale, accumulate=accumulate)
    assert o.shape == q.shape and o.dtype == dtype
    _check_attend(cache, q, o, before, cache.mass, scale, accumulate)
    # the same again, from a strided query into a wider output, on another stream
    cache.mass.copy_(before)
    first = o.clone()
    qs = torch.cat([q, q], 3)[..., :d]
    wide = torch.zeros(b, hq, 1, 2 * d, dtype=dtype, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attend(qs, scale=scale, accumulate=accumulate, out=wide[..., d:])
    side.synchronize()
    assert torch.equal(wide[..., d:], first) and (wide[..., :d] == 0).all()


@pytest.mark.parametrize("batch,budget,hq", [(70, 40, 8), (33, 400, 8), (3, 2000, 8), (40, 301, 48), (45, 4000, 8), (30, 1900, 64)])
def test_attend_shares(cuda, batch, budget, hq):
    """Many short sequences to a CTA and many CTAs to a sequence, some of them empty; units that
    one CTA has whole, of the sizes whose scores stay in tensor memory and of larger ones."""
    from linattn_b200 import HeavyCache

    hkv, d, dtype = 4, 64, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(batch)
    cache = HeavyCache(batch, hkv, d, budget, dtype=dtype)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    cache.mass.uniform_(generator=g)
    cache.seen.copy_(torch.randint(0, 2 * budget, (batch,), generator=g, device="cuda")
                     * (torch.rand(batch, generator=g, device="cuda") < 0.8))
    q = torch.randn(batch, hq, 1, d, generator=g, device="cuda").to(dtype)
    for _ in range(2):  # the arrival counts are back at zero
        before = cache.mass.clone()
        o = cache.attend(q)
        _check_attend(cache, q, o, before, cache.mass, 1 / math.sqrt(d), True)


@pytest.mark.parametrize("budget,hq,dtype", [(1024, 4, torch.bfloat16), (1023, 16, torch.float16), (4222, 4, torch.float16),
                                             (301, 32, torch.bfloat16), (2050, 64, torch.bfloat16)])
def test_attend_whole_units(cuda, budget, hq, dtype):
    """As many full units as the GPU has SMs, twice: every CTA has whole ones, its last among them."""
    from linattn_b200 import HeavyCache

    hkv, d = 4, 128
    batch = max(1, torch.cuda.get_device_properties(0).multi_processor_count * 2 // hkv)
    g = torch.Generator(device="cuda").manual_seed(budget)
    cache = HeavyCache(batch, hkv, d, budget, dtype=dtype)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    cache.mass.uniform_(generator=g)
    cache.seen.fill_(budget)
    q = torch.randn(batch, hq, 1, d, generator=g, device="cuda").to(dtype)
    for _ in range(2):
        before = cache.mass.clone()
        o = cache.attend(q)
        _check_attend(cache, q, o, before, cache.mass, 1 / math.sqrt(d), True)


def test_unaligned_rows(cuda):
    """Rows off the 16-byte grid and channels that are not next to one another are copied first."""
    from linattn_b200 import HeavyCache

    b, h, d, dtype = 2, 2, 64, torch.float16
    g = torch.Generator().manual_seed(2)
    x = torch.randn(3, b, h, 1, d, generator=g).to(dtype).cuda()
    caches = [HeavyCache(b, h, d, 16, dtype=dtype) for _ in range(3)]

    def odd(t):
        base = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")
        base[1:] = t.flatten()
        return base[1:].view(t.shape)

    def across(t):
        return t.transpose(2, 3).contiguous().transpose(2, 3)

    outs = []
    for c, f in zip(caches, (lambda t: t, odd, across)):
        c.append(f(x[0]), f(x[1]))
        outs.append(c.attend(f(x[2])))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[2].v)


def test_attend_nan_reaches_its_head_only(cuda):
    from linattn_b200 import HeavyCache

    cache = HeavyCache(1, 1, 64, 32, dtype=torch.bfloat16)
    cache.k.normal_()
    cache.v.normal_()
    cache.seen.fill_(32)
    q = torch.randn(1, 4, 1, 64, device="cuda", dtype=torch.bfloat16)
    q[0, 2] = math.nan
    o = cache.attend(q)
    assert o[0, 2].isnan().all() and o[0, [0, 1, 3]].isfinite().all()


def test_heavy_refusals(cuda):
    from linattn_b200 import HeavyCache

    with pytest.raises(ValueError, match="sinks"):
        HeavyCache(1, 1, 64, 8, sinks=4, recent=5)
    with pytest.raises(ValueError, match="recent"):
        HeavyCache(1, 1, 64, 8, recent=0)
    with pytest.raises(NotImplementedError):
        HeavyCache(1, 1, 96, 8)
    with pytest.raises(NotImplementedError):
        HeavyCache(1, 1, 64, 8, dtype=torch.float32)
    with pytest.raises(ValueError, match="cuda"):
        HeavyCache(1, 1, 64, 8, device="cpu")
    c = HeavyCache(2, 2, 64, 8, dtype=torch.float16)
    x = torch.zeros(2, 2, 1, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="must be"):
        c.append(x[:1], x[:1])
    with pytest.raises(ValueError, match="must be"):
        c.append(x.bfloat16(), x.bfloat16())
    with pytest.raises(ValueError, match="CUDA"):
        c.append(x.cpu(), x.cpu())
    with pytest.raises(ValueError, match="multiple"):
        c.attend(torch.zeros(2, 3, 1, 64, dtype=torch.float16, device="cuda"))
    with pytest.raises(ValueError, match="scale"):
        c.attend(x, scale=0.0)
    p = torch.zeros(10, 2, 64, dtype=torch.float16, device="cuda")
    m = torch.zeros(2, 10, device="cuda")
    with pytest.raises(ValueError, match="mass"):
        c.load(p, p, m.half(), _cu([10]))
    with pytest.raises(ValueError, match="rows"):
        c.load(p, p, m, _cu([4, 3, 3]))
    with pytest.raises(ValueError, match="int32"):
        c.load(p, p, m, _cu([10]).long())


def test_prompt_to_decode(cuda):
    """Prompts to the cache and on to single tokens, eagerly and as one CUDA graph; the masses
    that decide are those of the float64 attention over the same slots."""
    from linattn_b200 import HeavyCache, attention_mass, packed_attention

    lens, hq, hkv, d, budget, dtype = [400, 90, 1000], 8, 2, 128, 128, torch.bfloat16
    g = torch.Generator().manual_seed(1)
    n, b = sum(lens), len(lens)
    q, k, v = (torch.randn(n, h, d, generator=g).to(dtype).cuda() for h in (hq, hkv, hkv))
    cu = _cu(lens)
    _, lse = packed_attention(q, k, v, cu, max_q=max(lens))
    mass = attention_mass(q, k, lse, cu, max_q=max(lens), max_k=max(lens))
    caches = [HeavyCache(b, hkv, d, budget, sinks=4, recent=32, dtype=dtype) for _ in range(2)]
    for c in caches:
        c.load(k, v, mass, cu)
    eager, graphed = caches
    qs = torch.randn(60, b, hq, 1, d, generator=g).to(dtype).cuda()
    kn, vn = (torch.randn(60, b, hkv, 1, d, generator=g).to(dtype).cuda() for _ in range(2))
    qd, kd, vd, out = qs[0].clone(), kn[0].clone(), vn[0].clone(), torch.empty_like(qs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # set up outside the capture
        graphed.step(qd, kd, vd, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graphed.load(k, v, mass, cu)
    import os

    strict = os.environ.pop("LINATTN_B200_STRICT", None)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphed.step(qd, kd, vd, out=out)
    finally:
        if strict is not None:
            os.environ["LINATTN_B200_STRICT"] = strict
    for i in range(60):
        before = eager.mass.clone()
        pos = eager.pos.clone()
        o = eager.step(qs[i], kn[i], vn[i])
        new = eager.pos != pos
        before[new] = 0
        _check_attend(eager, qs[i], o, before, eager.mass, 1 / math.sqrt(d), True)
        qd.copy_(qs[i])
        kd.copy_(kn[i])
        vd.copy_(vn[i])
        graph.replay()
        assert torch.equal(out, o)
    for name in ("k", "v", "mass", "pos", "seen"):
        assert torch.equal(getattr(eager, name), getattr(graphed, name)), name
    assert eager.seen.tolist() == [m + 60 for m in lens]


def test_steps_right_after_one_another(cuda):
    """Prompt, masses, load and decode steps without a pause give what they give one at a time."""
    from linattn_b200 import HeavyCache, attention_mass, packed_attention

    hq, hkv, d, budget = 8, 2, 128, 96
    lens = [300, 40, 777]
    n = sum(lens)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(12, n, hq, d, generator=g, device="cuda").to(torch.bfloat16)
    new = torch.randn(6, 2, len(lens), hkv, 1, d, generator=g, device="cuda").to(torch.bfloat16)
    ends = torch.tensor([0] + lens, device="cuda")

    def chain(pause):
        cache = HeavyCache(len(lens), hkv, d, budget, dtype=torch.bfloat16, sinks=4, recent=16)
        outs = []
        for r in range(3):  # the cache is loaded again, over what the steps before made of it
            cu = ends.cumsum(0, dtype=torch.int32)
            pause()
            q, k, v = x[4 * r], x[4 * r + 1][:, :hkv], x[4 * r + 2][:, :hkv]
            o, lse = packed_attention(q, k, v, cu)
            pause()
            mass = attention_mass(q, k, lse, cu, window=200)
            pause()
            cache.load(k, v, mass, cu)
            pause()
            outs += [o, mass]
            for s in range(2):
                cache.append(new[2 * r + s, 0], new[2 * r + s, 1])
                pause()
                outs.append(cache.attend(o[:len(lens)].unsqueeze(2).contiguous()))
                pause()
            outs += [cache.k.clone(), cache.v.clone(), cache.mass.clone(), cache.pos.clone(), cache.seen.clone()]
        return outs

    want = chain(torch.cuda.synchronize)
    for _ in range(5):
        got = chain(lambda: None)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_append_of_no_tokens(cuda):
    from linattn_b200 import HeavyCache

    cache = HeavyCache(2, 2, 64, 8, dtype=torch.float16)
    x = torch.ones(2, 2, 3, 64, dtype=torch.float16, device="cuda")
    cache.append(x, x)
    cache.append(x[:, :, :0], x[:, :, :0])
    cache.append(torch.empty(2, 2, 0, 64, dtype=torch.float16, device="cuda"), torch.empty(2, 2, 0, 64, dtype=torch.float16, device="cuda"))
    assert cache.seen.tolist() == [3, 3]


def _filled(batch, hkv, d, budget, dtype, seed):
    from linattn_b200 import HeavyCache

    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = HeavyCache(batch, hkv, d, budget, dtype=dtype)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    cache.mass.uniform_(generator=g)
    cache.pos.copy_(torch.arange(budget, device="cuda"))
    cache.seen.fill_(budget)
    return cache, g


def test_captured_attend_outlives_larger_calls(cuda, monkeypatch):
    """A graph's scratch stays its own when later calls need more, and other tensors are made."""
    monkeypatch.setenv("LINATTN_B200_STRICT", "0")
    cache, g = _filled(2, 2, 128, 9000, torch.bfloat16, 3)
    q = torch.randn(2, 8, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    many = torch.randn(2, 64, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    before = cache.mass.clone()
    want, want_mass = cache.attend(q), cache.mass.clone()
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        cache.attend(q, out=out)  # set up outside the capture
        with torch.cuda.graph(graph, stream=side):
            cache.attend(q, out=out)
        cache.attend(many)
    torch.cuda.current_stream().wait_stream(side)
    cache.attend(many)
    sizes = sorted({s[-1].numel() for s in cache._scratch.values()})
    others = [torch.full((n // 4,), 7.0, device="cuda") for n in sizes for _ in range(4)]
    with torch.cuda.stream(side):
        others += [torch.full((n // 4,), 7.0, device="cuda") for n in sizes for _ in range(4)]
    torch.cuda.synchronize()
    cache.mass.copy_(before)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(bool((x == 7).all()) for x in others)
    assert torch.equal(out, want) and torch.equal(cache.mass, want_mass)


def test_attend_without_weights_on_streams_at_once(cuda, monkeypatch):
    """Calls that only read the cache do not meet, on more streams than have counts from the start."""
    from linattn_b200 import heavy

    monkeypatch.setenv("LINATTN_B200_STRICT", "0")
    cache, g = _filled(1, 2, 128, 2500, torch.float16, 4)
    n = heavy._STREAMS + 2
    q = [torch.randn(1, 16, 1, 128, generator=g, device="cuda").to(torch.float16) for _ in range(n)]
    mass = cache.mass.clone()
    want = [cache.attend(x, accumulate=False) for x in q]
    outs = [[torch.empty_like(x) for _ in range(20)] for x in q]
    streams = [torch.cuda.Stream() for _ in range(n)]
    torch.cuda.synchronize()
    for r in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                cache.attend(q[i], accumulate=False, out=outs[i][r])
    torch.cuda.synchronize()
    for i in range(n):
        assert all(torch.equal(o, want[i]) for o in outs[i])
    assert torch.equal(cache.mass, mass)
    assert all(bool((t == 0).all()) for t in cache._unit_tickets)
    # the counts of a further stream would be zero after a replay only: refused, not wrong
    late = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(graph, stream=late):
            cache.attend(q[0], accumulate=False, out=outs[0][0])


def test_reset_after_a_call_that_gave_up(cuda):
    """Arrival counts that an abandoned call has left are gone after reset()."""
    from linattn_b200 import HeavyCache

    b, h, d, budget, dtype = 2, 2, 64, 700, torch.float16
    g = torch.Generator(device="cuda").manual_seed(6)
    n = 2000
    k, v = (torch.randn(n, h, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    mass, q = torch.rand(h, n, generator=g, device="cuda"), torch.randn(b, 8, 1, d, generator=g, device="cuda").to(dtype)
    new = torch.randn(2, b, h, 1, d, generator=g, device="cuda").to(dtype)
    results = []
    for left in (0, 1, 40):
        cache = HeavyCache(b, h, d, budget, dtype=dtype)
        cache._ticket.fill_(left)
        for t in cache._unit_tickets:
            t.fill_(left)
        cache.reset()
        cache.load(k, v, mass, _cu([900, 1100]))
        outs = [cache.step(q, new[i], new[1 - i], out=torch.full_like(q, math.nan)) for i in range(2)]
        results.append(outs + [cache.mass.clone(), cache.pos.clone(), cache.seen.clone()])
    for other in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], other))
    assert results[0][-1].tolist() == [902, 1102]
