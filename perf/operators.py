"""Cases of the heavy-hitter serving path, from the prompt to single tokens.

Five operators, each in its plain form (elementary torch operations in 32 bits) and through
the framework:

* ``attn``   packed causal attention with grouped heads: outputs and log-sum-exps;
* ``mass``   the attention weight that each key of a prompt has received;
* ``load``   eviction of a prompt to a fixed budget per sequence and kv head;
* ``append`` one new token per sequence into a full cache, replacing the slot of least weight;
* ``attend`` one query token per sequence over the kept slots, adding its weights up.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a burst of short requests: latency
        {"name": "attn short requests", "op": "attn", "lens": "1,17,64,33,128,5,90,46", "past": "0", "hq": 32, "hkv": 8,
         "d": 128, "dtype": "bf16"},
        # one prefill batch of ragged prompts
        {"name": "attn ragged batch", "op": "attn", "lens": "2048,511,1300,77,1024,1,1999,832,400", "past": "0", "hq": 32,
         "hkv": 8, "d": 128, "dtype": "bf16"},
        # a chunk of a prompt whose earlier tokens are there already
        {"name": "attn chunk on a prefix", "op": "attn", "lens": "384", "past": "15737", "hq": 16, "hkv": 2, "d": 64,
         "dtype": "f16"},
        # one long prompt
        {"name": "attn long prompt", "op": "attn", "lens": "16384", "past": "0", "hq": 32, "hkv": 8, "d": 128,
         "dtype": "bf16"},
        # the last 64 queries of each prompt look back over it
        {"name": "mass observation window", "op": "mass", "lens": "4000,2311,901,6144", "past": "0", "window": 64, "hq": 32,
         "hkv": 8, "d": 128, "dtype": "f16"},
        # every query of a long prompt counts
        {"name": "mass long prompt", "op": "mass", "lens": "16384", "past": "0", "window": 0, "hq": 32, "hkv": 8, "d": 128,
         "dtype": "bf16"},
        # a long prompt cut to a small budget
        {"name": "load long prompt", "op": "load", "lens": "32768", "budget": 2048, "sinks": 4, "recent": 512, "hkv": 8,
         "d": 128, "dtype": "bf16"},
        # a batch of ragged prompts, some below the budget
        {"name": "load ragged batch", "op": "load", "lens": "8192,5000,1023,64,7777,2500,1025,3000,6001,1,4096,4095,900,2048,1500,8000",
         "budget": 1024, "sinks": 1, "recent": 255, "hkv": 8, "d": 64, "dtype": "f16"},
        # single tokens, one user and many
        {"name": "append one user", "op": "append", "batch": 1, "budget": 512, "sinks": 4, "recent": 64, "hkv": 8, "d": 128,
         "dtype": "bf16"},
        {"name": "append many users", "op": "append", "batch": 64, "budget": 4096, "sinks": 4, "recent": 1024, "hkv": 8,
         "d": 128, "dtype": "bf16"},
        {"name": "attend one user", "op": "attend", "batch": 1, "budget": 2048, "short": 0, "hq": 32, "hkv": 8, "d": 128,
         "dtype": "bf16"},
        {"name": "attend many users", "op": "attend", "batch": 64, "budget": 4096, "short": 5, "hq": 32, "hkv": 8, "d": 128,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _parts(rng, total, most):
    """`total` cut into at most `most` ragged lengths."""
    n = min(total, rng.randint(1, most))
    cuts = sorted(rng.sample(range(1, total), n - 1)) if n > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    op = rng.choice(["attn", "attn", "mass", "load", "append", "attend"])
    d, dtype = rng.choice([64, 128, 128]), rng.choice(["bf16", "f16"])
    hkv = rng.choice([1, 2, 4, 8])
    case = {"op": op, "d": d, "dtype": dtype, "hkv": hkv}
    if op in ("attn", "mass"):
        lens = _parts(rng, _log_int(rng, 24, 8192), 12)
        past = [_log_int(rng, 1, 4096) if rng.random() < 0.5 else 0 for _ in lens] if sum(lens) < 2048 and rng.random() < 0.5 else [0]
        case.update(hq=hkv * rng.choice([1, 2, 3, 4]) if hkv == 8 else hkv * rng.choice([1, 2, 4, 5, 7, 8]),
                    lens=",".join(map(str, lens)), past=",".join(map(str, past)))
        if op == "mass":
            case["window"] = rng.choice([0, 0, _log_int(rng, 8, 256)])
    elif op == "load":
        budget = _log_int(rng, 64, 4096)
        recent = rng.randint(1, budget // 2)
        case.update(lens=",".join(str(_log_int(rng, 16, 32768)) for _ in range(rng.randint(1, 12))), budget=budget,
                    sinks=rng.choice([0, 1, 4]), recent=recent)
    elif op == "append":
        budget = _log_int(rng, 64, 8192)
        case.update(batch=_log_int(rng, 1, 64), budget=budget, sinks=rng.choice([0, 1, 4]), recent=rng.randint(1, budget // 2))
    else:
        case.update(batch=_log_int(rng, 1, 64), budget=_log_int(rng, 16, 4096), short=rng.choice([0, 1, 7]),
                    hq=hkv * rng.choice([1, 2, 4, 5, 8]))
    return case


def _ints(text):
    return [int(x) for x in text.split(",")]


def _lens(case):
    """Query and key lengths of each sequence."""
    lq = _ints(case["lens"])
    past = _ints(case.get("past", "0"))
    past = past * len(lq) if len(past) == 1 else past
    return lq, [a + b for a, b in zip(lq, past)]


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def _counts(case):
    """Slots in use of each sequence of an `attend` batch: every `short`-th one is still filling."""
    b, n, s = case["batch"], case["budget"], case["short"]
    return [max(1, (n * (i + 1)) // (2 * b)) if s and i % s == s - 1 else n for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    d, hkv = case["d"], case["hkv"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    op = case["op"]
    s = {"op": op, "case": case}
    if op in ("attn", "mass"):
        lq, lk = _lens(case)
        hq = case["hq"]
        k = randn(sum(lk), hkv, d)
        k += (torch.rand(sum(lk), 1, 1, generator=g, device="cuda") < 0.01) * (0.3 * randn(1, hkv, d))  # a few keys that all queries like
        q = randn(sum(lq), hq, d)
        s.update(q=q.to(dt), k=k.to(dt), cu_q=_cu(lq), cu_k=_cu(lk), max_q=max(lq), max_k=max(lk), scale=1.0 / math.sqrt(d))
        if op == "attn":
            s["v"] = randn(sum(lk), hkv, d).to(dt)
        else:
            s["window"] = case["window"]
            s["lse"] = _lse(s["q"], s["k"], lq, lk, s["scale"])
    elif op == "load":
        lens = _ints(case["lens"])
        n, b, m = sum(lens), len(lens), case["budget"]
        s.update(k=randn(n, hkv, d).to(dt), v=randn(n, hkv, d).to(dt), mass=torch.exp(1.5 * randn(hkv, n)), cu=_cu(lens), lens=lens)
        _slots(s, b, hkv, m, d, dt, case["sinks"], case["recent"])
    elif op == "append":
        b, m = case["batch"], case["budget"]
        s.update(k_new=randn(b, hkv, 1, d).to(dt), v_new=randn(b, hkv, 1, d).to(dt))
        _slots(s, b, hkv, m, d, dt, case["sinks"], case["recent"])
        s["slot_k"].copy_(randn(b, hkv, m, d))
        s["slot_v"].copy_(randn(b, hkv, m, d))
        s["slot_mass"].copy_(torch.exp(1.5 * randn(b, hkv, m)))
        s["slot_pos"].copy_(torch.arange(m, device="cuda"))
        s["slot_pos"][:, :, case["sinks"]:] += 100  # tokens in between went before
        s["seen"].fill_(m + 100)
    else:
        b, m, hq = case["batch"], case["budget"], case["hq"]
        s.update(q=randn(b, hq, 1, d).to(dt), scale=1.0 / math.sqrt(d))
        _slots(s, b, hkv, m, d, dt, 0, 1)
        s["slot_k"].copy_(randn(b, hkv, m, d))
        s["slot_v"].copy_(randn(b, hkv, m, d))
        s["slot_mass"].copy_(torch.exp(1.5 * randn(b, hkv, m)))
        s["slot_pos"].copy_(torch.arange(m, device="cuda"))
        s["seen"].copy_(torch.tensor(_counts(case), dtype=torch.int32))
    return s


def _slots(s, b, hkv, m, d, dt, sinks, recent):
    """The cache that the program keeps: K, V, accumulated weight and position of each slot."""
    s.update(sinks=sinks, recent=recent, budget=m)
    if own:
        from linattn_b200 import HeavyCache

        c = HeavyCache(b, hkv, d, m, sinks=sinks, recent=recent, dtype=dt)
        s.update(cache=c, slot_k=c.k, slot_v=c.v, slot_mass=c.mass, slot_pos=c.pos, seen=c.seen)
    else:
        s.update(slot_k=torch.zeros(b, hkv, m, d, dtype=dt, device="cuda"), slot_v=torch.zeros(b, hkv, m, d, dtype=dt, device="cuda"),
                 slot_mass=torch.zeros(b, hkv, m, device="cuda"), slot_pos=torch.zeros(b, hkv, m, dtype=torch.int32, device="cuda"),
                 seen=torch.zeros(b, dtype=torch.int32, device="cuda"))


def _lse(q, k, lq, lk, scale):
    """Log-sum-exps (N_q, H_q) that the prompt's attention has left."""
    out = torch.empty(q.shape[0], q.shape[1], device="cuda")
    rep = q.shape[1] // k.shape[1]
    q0 = k0 = 0
    for a, b in zip(lq, lk):
        kk = k[k0:k0 + b].float()
        for lo in range(0, a, 1024):
            n = min(1024, a - lo)
            s = torch.matmul(q[q0 + lo:q0 + lo + n].float().transpose(0, 1).reshape(k.shape[1], rep * n, -1), kk.permute(1, 2, 0))
            s = s.view(k.shape[1], rep, n, b).mul_(scale)
            seen = torch.arange(b, device="cuda")[None] <= torch.arange(lo, lo + n, device="cuda")[:, None] + (b - a)
            s.masked_fill_(~seen, -math.inf)
            out[q0 + lo:q0 + lo + n] = torch.logsumexp(s, -1).reshape(-1, n).T
        q0, k0 = q0 + a, k0 + b
    return out


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ---- the framework's operators ---------------------------------------------------------
def _own_attn(s):
    from linattn_b200 import packed_attention

    o, lse = packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], max_q=s["max_q"], max_k=s["max_k"], scale=s["scale"])
    return {"o": o, "lse": lse}


def _own_mass(s):
    from linattn_b200 import attention_mass

    return attention_mass(s["q"], s["k"], s["lse"], s["cu_q"], s["cu_k"], max_q=s["max_q"], max_k=s["max_k"], window=s["window"],
                          scale=s["scale"])


def _cache_of(s):
    return {"k": s["slot_k"], "v": s["slot_v"], "mass": s["slot_mass"], "pos": s["slot_pos"], "seen": s["seen"]}


def _own_load(s):
    s["cache"].load(s["k"], s["v"], s["mass"], s["cu"])
    return _cache_of(s)


def _own_append(s):
    s["cache"].append(s["k_new"], s["v_new"])
    return _cache_of(s)


def _own_attend(s):
    return {"o": s["cache"].attend(s["q"], scale=s["scale"]), "mass": s["slot_mass"]}


# ---- plain forms -------------------------------------------------------------------------
def _scores(s):
    """Scaled scores (H_kv, G, queries, keys) in 32 bits, the pairs that may meet and the queries' log-sum-exps, if given."""
    q, k = s["q"].float(), s["k"].float()
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    at_q, at_k = torch.arange(q.shape[0], device=q.device), torch.arange(k.shape[0], device=q.device)
    seq_q, seq_k = torch.searchsorted(cu_q, at_q, right=True) - 1, torch.searchsorted(cu_k, at_k, right=True) - 1
    if s.get("window"):  # the other queries do not count
        late = at_q >= cu_q[seq_q + 1] - s["window"]
        q, at_q, seq_q, s = q[late], at_q[late], seq_q[late], {**s, "lse": s["lse"][late]}
    nq, hq, d = q.shape
    hkv = k.shape[1]
    # position of a query among its sequence's keys: the last query stands at the last key
    pos_q = at_q - cu_q[seq_q + 1] + (cu_k[1:] - cu_k[:-1])[seq_q]
    pos_k = at_k - cu_k[seq_k]
    meet = (seq_q[:, None] == seq_k[None]) & (pos_k[None] <= pos_q[:, None])
    x = torch.matmul(q.view(nq, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d), k.permute(1, 2, 0))
    return x.view(hkv, hq // hkv, nq, -1).mul_(s["scale"]), meet, s.get("lse")


def _plain_attn(s):
    x, meet, _ = _scores(s)
    hkv, g, nq, nk = x.shape
    x.masked_fill_(~meet, -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(hkv, g * nq, nk), s["v"].float().transpose(0, 1)).view(hkv, g, nq, -1)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + total.log()).squeeze(-1)
    return {"o": o.permute(2, 0, 1, 3).reshape(nq, hkv * g, -1).to(s["q"].dtype), "lse": lse.permute(2, 0, 1).reshape(nq, -1)}


def _plain_mass(s):
    x, meet, lse = _scores(s)
    hkv, g, nq, nk = x.shape
    x.sub_(lse.view(nq, hkv, g).permute(1, 2, 0)[..., None]).exp_().masked_fill_(~meet, 0.0)
    return x.sum((1, 2))


def _plain_load(s):
    cu, m, hkv = s["cu"].long(), s["budget"], s["k"].shape[1]
    n = cu[1:] - cu[:-1]
    at = torch.arange(max(s["lens"]), device="cuda")
    row = torch.clamp(cu[:-1, None] + at, max=s["k"].shape[0] - 1)  # (B, longest)
    w = s["mass"][:, row].transpose(0, 1)  # (B, H_kv, longest)
    kept = (at < s["sinks"]) | (at >= n[:, None] - s["recent"])
    w = torch.where(kept[:, None], math.inf, w)
    w = torch.where((at >= n[:, None])[:, None], -math.inf, w)
    best = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :m]
    best = torch.where(best < n[:, None, None], best, at.numel()).sort(-1).values  # ascending; none left last
    have = best < n[:, None, None]
    head = torch.arange(hkv, device="cuda")[None, :, None]
    src = row[torch.arange(n.numel(), device="cuda")[:, None, None], torch.where(have, best, 0)]
    j = best.shape[-1]
    for name, x in (("slot_k", s["k"][src, head]), ("slot_v", s["v"][src, head])):
        s[name][:, :, :j] = torch.where(have[..., None], x, s[name][:, :, :j])
    s["slot_mass"][:, :, :j] = torch.where(have, s["mass"][head, src], s["slot_mass"][:, :, :j])
    s["slot_pos"][:, :, :j] = torch.where(have, best.int(), s["slot_pos"][:, :, :j])
    s["seen"].copy_(n)
    return _cache_of(s)


def _plain_append(s):
    m = s["budget"]
    p = s["seen"][:, None, None]
    slot = torch.arange(m, device="cuda")
    free = (s["slot_pos"] >= s["sinks"]) & (s["slot_pos"] <= p - s["recent"])
    w = torch.where(free, s["slot_mass"], math.inf)
    least = torch.where(free & (w == w.amin(-1, keepdim=True)), slot, m).amin(-1, keepdim=True)
    at = torch.where(p < m, p.long(), least)  # a slot that is still empty, or the one that goes
    wide = at[..., None].expand(-1, -1, -1, s["k_new"].shape[-1])
    s["slot_k"].scatter_(2, wide, s["k_new"])
    s["slot_v"].scatter_(2, wide, s["v_new"])
    s["slot_mass"].scatter_(2, at, 0.0)
    s["slot_pos"].scatter_(2, at, p.expand_as(at).contiguous())
    s["seen"] += 1
    return _cache_of(s)


def _plain_attend(s):
    b, hkv, m, d = s["slot_k"].shape
    q = s["q"].float().view(b, hkv, -1, d)
    x = torch.matmul(q, s["slot_k"].float().transpose(2, 3)).mul_(s["scale"])
    there = torch.arange(m, device="cuda") < s["seen"].clamp(max=m)[:, None]
    x.masked_fill_(~there[:, None, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    x = x / x.sum(-1, keepdim=True)
    s["slot_mass"] += x.sum(2)
    return {"o": torch.matmul(x, s["slot_v"].float()).view(b, -1, 1, d).to(s["q"].dtype), "mass": s["slot_mass"]}


_OWN = {"attn": _own_attn, "mass": _own_mass, "load": _own_load, "append": _own_append, "attend": _own_attend}
_PLAIN = {"attn": _plain_attn, "mass": _plain_mass, "load": _plain_load, "append": _plain_append, "attend": _plain_attend}


# ---- what a pass cannot do without -------------------------------------------------------
def _pairs(lq, lk, window=0):
    """(query, key) pairs that meet."""
    n = 0
    for a, b in zip(lq, lk):
        w = min(a, window) if window else a
        n += w * b - w * (w - 1) // 2
    return n


def work(case):
    d, hkv, e = case["d"], case["hkv"], 2
    op = case["op"]
    if op in ("attn", "mass"):
        lq, lk = _lens(case)
        hq, nk, w = case["hq"], sum(lk), case.get("window", 0)
        nq = sum(min(a, w) if w else a for a in lq)
        pairs = _pairs(lq, lk, w)
        if op == "attn":
            return {"bytes": 2 * nq * hq * d * e + 2 * nk * hkv * d * e + nq * hq * 4, "flops": 4 * d * pairs * hq}
        return {"bytes": nq * hq * (d * e + 4) + nk * hkv * (d * e + 4), "flops": 2 * d * pairs * hq}
    if op == "load":
        lens = _ints(case["lens"])
        kept = sum(min(n, case["budget"]) for n in lens)
        return {"bytes": hkv * (4 * sum(lens) + kept * (4 * d * e + 8)), "flops": 0}
    if op == "append":
        return {"bytes": case["batch"] * hkv * (8 * case["budget"] + 4 * d * e + 8), "flops": 0}
    n = sum(_counts(case))
    return {"bytes": n * hkv * (2 * d * e + 8) + 2 * case["batch"] * case["hq"] * d * e, "flops": 4 * d * n * case["hq"]}


# ---- the definition in 64 bits ---------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"attn": _exact_attn, "mass": _exact_mass, "load": _exact_load, "append": _exact_append, "attend": _exact_attend}[case["op"]](case, s)


def _exact_rows(case, s):
    """(sequence's first query, key, lengths, kv head, q head, scores) one head of one sequence at a time."""
    lq, lk = _lens(case)
    rep = case["hq"] // case["hkv"]
    q0 = k0 = 0
    for a, b in zip(lq, lk):
        future = torch.ones(a, b, dtype=torch.bool, device="cuda").triu(b - a + 1)
        for h in range(case["hq"]):
            x = s["q"][q0:q0 + a, h].double() @ s["k"][k0:k0 + b, h // rep].double().T
            yield q0, k0, a, b, h // rep, h, x * s["scale"], future
        q0, k0 = q0 + a, k0 + b


def _exact_attn(case, s):
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for q0, k0, a, b, hk, h, x, future in _exact_rows(case, s):
        x[future] = -math.inf
        lse[q0:q0 + a, h] = torch.logsumexp(x, -1)
        o[q0:q0 + a, h] = torch.softmax(x, -1) @ s["v"][k0:k0 + b, hk].double()
    return {"o": o, "lse": lse}


def _exact_mass(case, s):
    out = torch.zeros(case["hkv"], s["k"].shape[0], dtype=torch.float64, device="cuda")
    for q0, k0, a, b, hk, h, x, future in _exact_rows(case, s):
        w = torch.exp(x - s["lse"][q0:q0 + a, h, None].double())
        w[future] = 0
        out[hk, k0:k0 + b] += w[a - min(a, case["window"]) if case["window"] else 0:].sum(0)
    return out


def _exact_load(case, s):
    lens, m = _ints(case["lens"]), case["budget"]
    k, v, w = s["slot_k"].double().cpu(), s["slot_v"].double().cpu(), s["slot_mass"].double().cpu()
    mass, ks, vs = s["mass"].cpu(), s["k"].double().cpu(), s["v"].double().cpu()
    first = 0
    for b, n in enumerate(lens):
        for h in range(case["hkv"]):
            x = mass[h, first:first + n].tolist()
            held = [i for i in range(n) if i < case["sinks"] or i >= n - case["recent"]]
            rest = sorted((i for i in range(case["sinks"], max(case["sinks"], n - case["recent"]))), key=lambda i: (-x[i], i))
            keep = list(range(n)) if n <= m else sorted(held + rest[:m - len(held)])
            at = torch.tensor(keep)
            k[b, h, :len(keep)], v[b, h, :len(keep)], w[b, h, :len(keep)] = ks[first + at, h], vs[first + at, h], mass[h, first + at].double()
        first += n
    return {"k": k, "v": v, "mass": w, "pos": None, "seen": None}


def _exact_append(case, s):
    k, v, w = s["slot_k"].double(), s["slot_v"].double(), s["slot_mass"].double()
    mass, pos = s["slot_mass"].cpu().tolist(), s["slot_pos"].cpu().tolist()
    for b, now in enumerate(s["seen"].tolist()):
        for h in range(case["hkv"]):
            may = [i for i in range(case["budget"]) if case["sinks"] <= pos[b][h][i] <= now - case["recent"]]
            at = now if now < case["budget"] else min(may, key=lambda i: (mass[b][h][i], i))
            k[b, h, at], v[b, h, at], w[b, h, at] = s["k_new"][b, h, 0].double(), s["v_new"][b, h, 0].double(), 0.0
    return {"k": k, "v": v, "mass": w, "pos": None, "seen": None}


def _exact_attend(case, s):
    rep = case["hq"] // case["hkv"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    w = s["slot_mass"].double()
    for b, n in enumerate(_counts(case)):
        for h in range(case["hq"]):
            p = torch.softmax((s["slot_k"][b, h // rep, :n].double() @ s["q"][b, h, 0].double()) * s["scale"], 0)
            o[b, h, 0] = p @ s["slot_v"][b, h // rep, :n].double()
            w[b, h // rep, :n] += p
    return {"o": o, "mass": w}
