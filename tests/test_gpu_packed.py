"""Packed prompt attention and attention mass against float64, per sequence and head.

Tolerances, from the arithmetic (u = 2^-8 for bf16, the unit roundoff, 2^-11 for f16; A = sum_j p_ij |v_j|):

* a score is a sum of D exact products in fp32: its error is at most D 2^-24 sum |q k|, times
  the scale; with the exponential's 2^-21 that is the relative error `e` of a weight;
* o: each weight is rounded once to 16 bits (u A), the result once more (u |o|); f16 weights
  below 2^-14 of the row's largest lose at most 2^-25 each;
* lse: the absolute error of a sum of positive terms with relative error e;
* mass: relative error e (the lse given is the fp32 one that the oracle uses too), and
  2^-20 for the fp32 sums.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _cu(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def _inputs(seed, lq, lk, hq, hkv, d, dtype):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(lq), hq, d, generator=g).to(dtype).cuda()
    k = torch.randn(sum(lk), hkv, d, generator=g).to(dtype).cuda()
    v = torch.randn(sum(lk), hkv, d, generator=g).to(dtype).cuda()
    return q, k, v


def _blocks(q, k, lq, lk, scale, causal):
    """(rows of q, rows of k, q head, kv head, scores, visible, error of a score) of each head of each sequence."""
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    q0 = k0 = 0
    for a, b in zip(lq, lk):
        see = torch.ones(a, b, dtype=torch.bool, device="cuda")
        if causal:
            see = see.tril(b - a)
        for h in range(hq):
            x, y = q[q0:q0 + a, h].double(), k[k0:k0 + b, h * hkv // hq].double()
            err = d * 2.0 ** -24 * scale * (x.abs() @ y.abs().T)
            yield slice(q0, q0 + a), slice(k0, k0 + b), h, h * hkv // hq, (x @ y.T) * scale, see, err
        q0, k0 = q0 + a, k0 + b


def _check_attention(o, lse, q, k, v, lq, lk, scale, causal):
    u = U[q.dtype]
    for rq, rk, h, hk, s, see, err in _blocks(q, k, lq, lk, scale, causal):
        if s.shape[0] == 0:
            continue
        got, got_lse = o[rq, h].double(), lse[rq, h].double()
        none = ~see.any(1)
        assert torch.equal(got[none], torch.zeros_like(got[none]))
        assert (got_lse[none] == -math.inf).all()
        if none.all():
            continue
        s, see, err, got, got_lse = s[~none], see[~none], err[~none], got[~none], got_lse[~none]
        s = s.masked_fill(~see, -math.inf)
        want_lse = torch.logsumexp(s, 1)
        e = (err.masked_fill(~see, 0).amax(1) + 2.0 ** -20)
        assert ((got_lse - want_lse).abs() <= 2 * e + 2.0 ** -22 * want_lse.abs()).all()
        p = torch.softmax(s, 1)
        vv = v[rk, hk].double()
        want, mag = p @ vv, p @ vv.abs()
        tiny = s.shape[1] * 2.0 ** -25 * vv.abs().max() if q.dtype == torch.float16 else 0.0
        bound = (u * 1.02 + 2 * e[:, None]) * mag + u * 1.02 * want.abs() + tiny
        assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


CASES = [
    # lens of queries, of keys, H_q, H_kv, D, dtype, causal
    ([1], [1], 1, 1, 128, torch.bfloat16, True),
    ([5, 0, 1, 130], [5, 0, 1, 130], 8, 2, 128, torch.bfloat16, True),
    ([64, 65, 63, 256, 257], [64, 65, 63, 256, 257], 4, 4, 64, torch.float16, True),
    ([127, 128, 129], [127, 128, 129], 6, 2, 128, torch.float16, True),      # G = 3: row tiles of 126 rows
    ([300, 41], [300, 41], 10, 2, 64, torch.bfloat16, True),                 # G = 5
    ([3, 77], [3, 77], 128, 1, 128, torch.bfloat16, True),                   # one token to a row tile
    ([33, 7], [33, 7], 70, 1, 64, torch.float16, True),
    ([1, 1, 1], [700, 1, 129], 16, 2, 128, torch.bfloat16, True),            # single tokens on a prefix
    ([40, 200], [1000, 333], 8, 4, 128, torch.float16, True),                # chunks on a prefix
    ([50, 20, 300], [17, 0, 128], 8, 2, 128, torch.bfloat16, True),          # more queries than keys: empty rows
    ([100, 31], [260, 500], 8, 8, 64, torch.bfloat16, False),
    ([1100], [1100], 8, 2, 128, torch.bfloat16, True),
    (list(range(40)), list(range(40)), 4, 2, 64, torch.bfloat16, True),                       # two sequences to a lane
    ([3 * i % 50 for i in range(70)], [5 * i % 90 for i in range(70)], 2, 1, 64, torch.float16, True),  # more than 64
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("splits", [None, 1, 3])
def test_packed_attention(cuda, case, splits):
    from linattn_b200 import packed_attention

    lq, lk, hq, hkv, d, dtype, causal = CASES[case]
    q, k, v = _inputs(case, lq, lk, hq, hkv, d, dtype)
    scale = 1.3 / math.sqrt(d)
    o, lse = packed_attention(q, k, v, _cu(lq), _cu(lk), max_q=max(lq), max_k=max(lk), causal=causal, scale=scale,
                              n_splits=splits)
    assert o.shape == q.shape and o.dtype == dtype and lse.shape == q.shape[:2] and lse.dtype == torch.float32
    _check_attention(o, lse, q, k, v, lq, lk, scale, causal)
    again, lse2 = packed_attention(q, k, v, _cu(lq), _cu(lk), causal=causal, scale=scale, n_splits=splits)
    if splits is not None:  # without the longest lengths: the same tiles
        assert torch.equal(again, o) and torch.equal(lse2, lse)


@pytest.mark.parametrize("splits", [8, 9, 32])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(6, 2, 128, torch.float16), (5, 1, 64, torch.bfloat16)])
def test_packed_attention_many_parts(cuda, splits, hq, hkv, d, dtype):
    """Parts of one key tile, and parts that are left without any."""
    from linattn_b200 import packed_attention

    lq, lk = [7, 130, 0, 33], [3000, 140, 5, 20]
    q, k, v = _inputs(splits, lq, lk, hq, hkv, d, dtype)
    o, lse = packed_attention(q, k, v, _cu(lq), _cu(lk), n_splits=splits)
    _check_attention(o, lse, q, k, v, lq, lk, d ** -0.5, True)


def test_packed_after_its_producers(cuda):
    """Offsets and rows that the kernels right before write, calls whose inputs are the last one's outputs."""
    from linattn_b200 import attention_mass, packed_attention

    d = 64
    for round_ in range(20):
        lens = [1 + (7 * round_ + 13 * i) % 90 for i in range(9)]
        n = torch.tensor([0] + lens, device="cuda")
        g = torch.Generator(device="cuda").manual_seed(round_)
        x = torch.randn(sum(lens), 4, d, generator=g, device="cuda")
        busy = torch.randn(1 << 20, device="cuda")
        for _ in range(3):
            busy = busy.sin()
        cu = n.cumsum(0, dtype=torch.int32)
        q = x.to(torch.float16)
        o, lse = packed_attention(q, q, q, cu)
        o2, lse2 = packed_attention(o, o, q, cu, n_splits=2)
        mass = attention_mass(o, o, lse2, cu, n_splits=3)
        o3, _ = packed_attention(o2, o, o2, cu)
        _check_attention(o, lse, q, q, q, lens, lens, d ** -0.5, True)
        _check_attention(o2, lse2, o, o, q, lens, lens, d ** -0.5, True)
        assert abs(float(mass.double().sum()) - sum(lens) * 4) <= 1e-4 * sum(lens) * 4
        again, _ = packed_attention(o2, o, o2, cu)
        assert torch.equal(o3, again)


def test_packed_attention_growing_scores(cuda):
    """Scores that keep rising move the running maximum on every key tile."""
    from linattn_b200 import packed_attention

    n, d = 700, 128
    q, k, v = _inputs(3, [n], [n], 4, 2, d, torch.bfloat16)
    k = (k.float() * torch.linspace(0.1, 6.0, n, device="cuda")[:, None, None]).to(torch.bfloat16)
    o, lse = packed_attention(q, k, v, _cu([n]))
    _check_attention(o, lse, q, k, v, [n], [n], 1 / math.sqrt(d), True)


def test_packed_attention_strides_and_stream(cuda):
    from linattn_b200 import packed_attention

    lens, hq, hkv, d = [90, 300], 8, 2, 128
    q, k, v = _inputs(4, lens, lens, hq, hkv, d, torch.bfloat16)
    want, want_lse = packed_attention(q, k, v, _cu(lens))
    # heads outermost, K and V as halves of one buffer, an output inside a wider one
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    kv = torch.cat([k, v], 2)
    wide = torch.full((sum(lens), hq, 2 * d), 7.0, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o, lse = packed_attention(qt, kv[..., :d], kv[..., d:], _cu(lens), out=wide[..., d:])
    side.synchronize()
    assert torch.equal(o, want) and torch.equal(lse, want_lse)
    assert (wide[..., :d] == 7).all()
    # rows that are not on 16 bytes are copied first
    odd = torch.empty(sum(lens), hq, d + 1, dtype=torch.bfloat16, device="cuda")
    odd[..., :d] = q
    assert torch.equal(packed_attention(odd[..., :d], k, v, _cu(lens))[0], want)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_packed_neighbours_do_not_leak(cuda, bad):
    """Inf and NaN of one sequence reach no other's outputs or masses."""
    from linattn_b200 import attention_mass, packed_attention

    lens, hq, hkv, d = [70, 45, 200, 13], 6, 2, 128
    q, k, v = _inputs(5, lens, lens, hq, hkv, d, torch.bfloat16)
    cu = _cu(lens)
    o, lse = packed_attention(q, k, v, cu)
    mass = attention_mass(q, k, lse, cu)
    lo, hi = int(cu[1]), int(cu[2])
    for x in (q, k, v):
        x[lo:hi] = bad
    o2, lse2 = packed_attention(q, k, v, cu)
    mass2 = attention_mass(q, k, lse2, cu)
    rest = torch.ones(sum(lens), dtype=torch.bool, device="cuda")
    rest[lo:hi] = False
    assert torch.equal(o2[rest], o[rest]) and torch.equal(lse2[rest], lse[rest])
    assert torch.equal(mass2[:, rest], mass[:, rest])
    assert o2[~rest].isnan().all()


def test_packed_offsets_out_of_range_are_reported(cuda, monkeypatch):
    """Offsets beyond the buffers are clamped; the status word says so."""
    from linattn_b200 import _lib as L
    from linattn_b200 import attention_mass, packed_attention

    monkeypatch.setenv("LINATTN_B200_STRICT", "0")
    q, k, v = _inputs(6, [100], [100], 4, 2, 64, torch.float16)
    cu = torch.tensor([0, 60, 140], dtype=torch.int32, device="cuda")
    L.read_status(cuda)
    o, lse = packed_attention(q, k, v, cu)
    assert L.read_status(cuda) & L.DEV_BAD_ID
    good, good_lse = packed_attention(q, k, v, _cu([60, 40]))
    assert torch.equal(o, good) and torch.equal(lse, good_lse)
    mass = attention_mass(q, k, lse, cu)
    assert L.read_status(cuda) & L.DEV_BAD_ID
    assert torch.equal(mass, attention_mass(q, k, lse, _cu([60, 40])))


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("window,splits", [(0, None), (0, 3), (1, 1), (50, 2)])
def test_attention_mass(cuda, case, window, splits):
    from linattn_b200 import attention_mass

    lq, lk, hq, hkv, d, dtype, causal = CASES[case]
    q, k, _ = _inputs(case + 50, lq, lk, hq, hkv, d, dtype)
    scale = 1.3 / math.sqrt(d)
    lse = torch.full(q.shape[:2], -math.inf, device="cuda")
    for rq, rk, h, hk, s, see, _ in _blocks(q, k, lq, lk, scale, causal):
        if s.numel():
            lse[rq, h] = torch.logsumexp(s.masked_fill(~see, -math.inf), 1).float()
    got = attention_mass(q, k, lse, _cu(lq), _cu(lk), max_q=max(lq), max_k=max(lk), causal=causal, window=window,
                         scale=scale, n_splits=splits)
    want = torch.zeros(hkv, sum(lk), dtype=torch.float64, device="cuda")
    slack = torch.zeros_like(want)
    for rq, rk, h, hk, s, see, err in _blocks(q, k, lq, lk, scale, causal):
        if not s.numel():
            continue
        see = see.clone()
        if window and window < s.shape[0]:
            see[: s.shape[0] - window] = False
        p = torch.exp(s - lse[rq, h].double()[:, None]).masked_fill(~see, 0)
        rel = err + 2.0 ** -20 + 2.0 ** -22 * lse[rq, h].double().abs().nan_to_num(posinf=0)[:, None]
        want[hk, rk] += p.sum(0)
        slack[hk, rk] += (p * 2 * rel).sum(0)
    assert got.shape == want.shape and got.dtype == torch.float32
    assert ((got.double() - want).abs() <= slack + 2.0 ** -20 * want).all()
    again = attention_mass(q, k, lse, _cu(lq), _cu(lk), causal=causal, window=window, scale=scale,
                           n_splits=splits if splits else 1)
    if splits:
        assert torch.equal(again, got)


@pytest.mark.parametrize("lens,hq,hkv,d", [([600, 30, 250], 8, 2, 128), ([385, 232], 20, 4, 64), ([900], 16, 1, 128)])
def test_mass_of_chosen_splits(cuda, lens, hq, hkv, d):
    """The chosen number of splits, one, and as many as query tiles give the same sums."""
    from linattn_b200 import attention_mass, packed_attention

    q, k, v = _inputs(21, lens, lens, hq, hkv, d, torch.float16)
    cu = _cu(lens)
    _, lse = packed_attention(q, k, v, cu, max_q=max(lens), max_k=max(lens))
    one = attention_mass(q, k, lse, cu, max_q=max(lens), max_k=max(lens), n_splits=1).double()
    for splits in (None, 13, 64):
        got = attention_mass(q, k, lse, cu, max_q=max(lens), max_k=max(lens), n_splits=splits).double()
        # fp32 sums of the same positive terms in another order: each rounds at most once a term
        assert ((got - one).abs() <= 2 * max(lens) * (hq // hkv) * 2.0 ** -24 * one).all()


def test_mass_sums_to_the_queries(cuda):
    """Every query hands out a weight of 1 per head: the masses of a sequence sum to them."""
    from linattn_b200 import attention_mass, packed_attention

    lens, hq, hkv, d = [1500, 3, 640], 8, 2, 128
    q, k, v = _inputs(8, lens, lens, hq, hkv, d, torch.bfloat16)
    _, lse = packed_attention(q, k, v, _cu(lens))
    mass = attention_mass(q, k, lse, _cu(lens)).double()
    at = 0
    for n in lens:
        total = mass[:, at:at + n].sum(1)
        # lse and the weights come from one product: the error of a row's sum is that of its lse
        assert ((total / (n * hq // hkv) - 1).abs() <= 1e-4).all()
        at += n


def test_packed_without_keys_or_queries(cuda):
    from linattn_b200 import attention_mass, packed_attention

    q, k, v = _inputs(11, [5], [7], 4, 2, 64, torch.bfloat16)
    o, lse = packed_attention(q, k[:0], v[:0], _cu([5]), _cu([0]))
    assert (o == 0).all() and (lse == -math.inf).all()
    o, lse = packed_attention(q[:0], k, v, _cu([0]), _cu([7]))
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    assert (attention_mass(q[:0], k, lse, _cu([0]), _cu([7])) == 0).all()
    assert attention_mass(q, k[:0], torch.zeros(5, 4, device="cuda"), _cu([5]), _cu([0])).shape == (2, 0)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")  # no sequence at all
    assert packed_attention(q[:0], k[:0], v[:0], none)[0].shape == (0, 4, 64)


def test_packed_broadcast_heads(cuda):
    """K and V expanded over heads (stride 0) and single heads with odd strides."""
    from linattn_b200 import packed_attention

    q, k, v = _inputs(12, [50], [50], 4, 1, 64, torch.float16)
    cu = _cu([50])
    want = packed_attention(q, k.expand(-1, 2, -1).contiguous(), v.expand(-1, 2, -1).contiguous(), cu)[0]
    assert torch.equal(packed_attention(q, k.expand(-1, 2, -1), v.expand(-1, 2, -1), cu)[0], want)
    one = packed_attention(q, k, v, cu)[0]
    assert torch.equal(packed_attention(q, k.as_strided(k.shape, (64, 3, 1)), v, cu)[0], one)


def test_packed_refusals(cuda):
    from linattn_b200 import attention_mass, packed_attention

    q, k, v = _inputs(9, [8], [8], 4, 2, 64, torch.float16)
    cu = _cu([8])
    _, lse = packed_attention(q, k, v, cu)
    with pytest.raises(NotImplementedError):
        packed_attention(q.float(), k.float(), v.float(), cu)
    with pytest.raises(NotImplementedError):
        packed_attention(q[..., :32].contiguous(), k[..., :32].contiguous(), v[..., :32].contiguous(), cu)
    with pytest.raises(ValueError, match="dtype"):
        packed_attention(q, k.bfloat16(), v, cu)
    with pytest.raises(ValueError, match="multiple"):
        packed_attention(q[:, :3].contiguous(), k, v, cu)
    with pytest.raises(ValueError, match="int32"):
        packed_attention(q, k, v, cu.long())
    with pytest.raises(ValueError, match="scale"):
        packed_attention(q, k, v, cu, scale=-1.0)
    with pytest.raises(ValueError, match="workspace"):
        packed_attention(q, k, v, cu, n_splits=2, workspace=torch.empty(4, device="cuda"))
    with pytest.raises(ValueError, match="same tokens"):
        packed_attention(q, k[:4], v[:4], cu)
    with pytest.raises(ValueError, match="lse"):
        attention_mass(q, k, lse[:, :2], cu)
    with pytest.raises(ValueError, match="window"):
        attention_mass(q, k, lse, cu, window=-1)
    with pytest.raises(ValueError, match="out"):
        attention_mass(q, k, lse, cu, out=torch.empty(2, 9, device="cuda"))
    with pytest.raises(ValueError, match="CUDA"):
        packed_attention(q.cpu(), k.cpu(), v.cpu(), cu.cpu())


@pytest.mark.parametrize("kind,hq,hkv,d,dtype", [
    ("below a tile", 16, 8, 128, torch.bfloat16), ("below a tile", 8, 8, 64, torch.float16),
    ("more than 64", 16, 8, 128, torch.float16), ("more than 64", 8, 8, 64, torch.bfloat16),
    ("row tiles in turn", 8, 8, 128, torch.bfloat16), ("row tiles in turn", 8, 8, 64, torch.float16),
])
def test_packed_many_ragged_items(cuda, kind, hq, hkv, d, dtype):
    """Several work items of one key tile to a CTA, whose V rows past the sequence (here the
    next one's NaN and Inf) are cleared while the next items' tiles are already loaded."""
    from linattn_b200 import packed_attention

    if kind == "row tiles in turn":  # items whose second row tile is empty, then ones whose first reads nothing
        lq = [100 if i % 2 else 2 * (128 * hkv // hq) - i for i in range(60)]
        lk = [100 if i % 2 else 100 - i for i in range(60)]
    else:
        n = 64 if kind == "below a tile" else 110
        lq = lk = [1 + (37 * i) % 127 for i in range(n)]
    q, k, v = _inputs(31, lq, lk, hq, hkv, d, dtype)
    cu_q, cu_k = _cu(lq), _cu(lk)
    clean = [packed_attention(q, k, v, cu_q, cu_k, max_q=max(lq), max_k=max(lk), n_splits=n) for n in (1, None)]
    for o, lse in clean:
        _check_attention(o, lse, q, k, v, lq, lk, d ** -0.5, True)
    rest = torch.zeros(sum(lq), dtype=torch.bool, device="cuda")
    for s in range(0, len(lq), 3):  # every third sequence is sound, its neighbours are not
        rest[int(cu_q[s]):int(cu_q[s + 1])] = True
    for s in range(len(lq)):
        if s % 3:
            k[int(cu_k[s]):int(cu_k[s + 1])] = math.nan
            v[int(cu_k[s]):int(cu_k[s + 1])] = math.nan if s % 2 else math.inf
    o, lse = clean[0]
    for _ in range(3):
        o2, lse2 = packed_attention(q, k, v, cu_q, cu_k, max_q=max(lq), max_k=max(lk), n_splits=1)
        assert torch.equal(o2[rest], o[rest]) and torch.equal(lse2[rest], lse[rest])


@pytest.mark.parametrize("splits", [None, 1, 3])
@pytest.mark.parametrize("lq,lk,before,after,hq,hkv,d,dtype,max_q", [
    ([1] * 8, [4000] * 8, 0, 56, 8, 2, 128, torch.bfloat16, None),               # single tokens in a fixed buffer
    ([200], [8000], 0, 1500, 8, 8, 64, torch.float16, None),                     # a chunk
    ([0, 33, 1, 150], [0, 900, 300, 150], 7, 3, 6, 2, 128, torch.float16, None), # G = 3, rows before the first one
    ([3, 0, 5] * 30, [500, 9, 0] * 30, 5, 40, 4, 2, 64, torch.bfloat16, None),   # more sequences than a search step
    ([2] * 1100, [300] * 1100, 33, 70, 2, 1, 64, torch.float16, None),           # than two
    ([40, 300, 90], [600, 700, 90], 2, 9, 8, 2, 128, torch.bfloat16, 77),        # longer than the caller says
    ([10, 90] * 40, [600, 90] * 40, 0, 0, 8, 2, 64, torch.bfloat16, 21),
])
def test_packed_rows_of_no_sequence_are_left_alone(cuda, splits, lq, lk, before, after, hq, hkv, d, dtype, max_q):
    """Padding of a fixed buffer, and rows beyond the longest sequence that the caller names,
    keep what `out` and `lse_out` hold, whatever the number of parts."""
    from linattn_b200 import packed_attention

    n = before + sum(lq) + after
    q, k, v = _inputs(41, [n], lk, hq, hkv, d, dtype)
    cu_q = _cu(lq) + before
    out = torch.full_like(q, 7.0)
    lse = torch.full((n, hq), 5.0, device="cuda")
    scratch = torch.full((32 * n * hq * (d + 1),), math.nan, device="cuda")  # what no part writes shows
    packed_attention(q, k, v, cu_q, _cu(lk), max_q=max_q or max(lq), max_k=max(lk), out=out, lse_out=lse, n_splits=splits,
                     workspace=scratch)
    inside = torch.zeros(n, dtype=torch.bool, device="cuda")
    at = before
    for m in lq:
        inside[at:at + min(m, max_q or m)] = True
        at += m
    assert (out[~inside] == 7).all() and (lse[~inside] == 5).all()
    want, want_lse = packed_attention(q[before:n - after].contiguous(), k, v, _cu(lq), _cu(lk), n_splits=1)
    ours = inside[before:n - after]
    # either side rounds its weights and its outputs once (2 u max |v|), and has a score's error e
    # (scale sum |q k| is below 1.5 sqrt(d) here)
    e = d * 2.0 ** -24 * 1.5 * d ** 0.5 + 2.0 ** -20
    got, ref = out[before:n - after][ours].double(), want[ours].double()
    assert ((got - ref).abs() <= (4.1 * U[dtype] + 4 * e) * v.abs().max().double()).all()
    got, ref = lse[before:n - after][ours].double(), want_lse[ours].double()
    assert torch.equal(got == -math.inf, ref == -math.inf)
    assert ((got - ref).nan_to_num(0).abs() <= 4 * e).all()


@pytest.mark.parametrize("splits", [None, 1, 3])
@pytest.mark.parametrize("lens,before,after,hq,hkv,d,max_k", [
    ([200, 0, 513, 1], 9, 300, 8, 2, 128, None),
    ([900, 700, 40], 0, 5, 4, 2, 64, 300),        # longer than the caller says, inside a tile
    ([900, 700, 40], 3, 0, 4, 2, 64, 512),        # and at its end
    ([7, 0, 30] * 40, 1, 1, 6, 2, 64, None),
    ([80, 3] * 600, 0, 33, 2, 1, 64, 50),
])
def test_mass_of_no_sequence_is_left_alone(cuda, splits, lens, before, after, hq, hkv, d, max_k):
    """Keys of no sequence, and keys beyond the longest sequence that the caller names, keep
    what `out` holds, whatever the number of splits."""
    from linattn_b200 import attention_mass, packed_attention

    n = before + sum(lens) + after
    q, k, v = _inputs(43, [n], [n], hq, hkv, d, torch.bfloat16)
    cu = _cu(lens) + before
    _, lse = packed_attention(q, k, v, cu)
    want = attention_mass(q, k, lse, cu, n_splits=1).double()
    out = torch.full((hkv, n), 7.0, device="cuda")
    attention_mass(q, k, lse, cu, max_q=max(lens), max_k=max_k or max(lens), out=out, n_splits=splits,
                   workspace=torch.full((64 * hkv * n,), math.nan, device="cuda"))
    inside = torch.zeros(n, dtype=torch.bool, device="cuda")
    at = before
    for m in lens:
        inside[at:at + min(m, max_k or m)] = True
        at += m
    assert (out[:, ~inside] == 7).all()
    # fp32 sums of the same positive terms in another order: each rounds at most once a term
    assert ((out.double() - want).abs() <= 2 * max(lens) * (hq // hkv) * 2.0 ** -24 * want)[:, inside].all()


def test_mass_of_rows_without_a_finite_lse(cuda):
    """A row whose lse is infinite adds nothing."""
    from linattn_b200 import attention_mass, packed_attention

    q, k, v = _inputs(44, [300], [300], 4, 2, 64, torch.float16)
    cu = _cu([300])
    _, lse = packed_attention(q, k, v, cu)
    for n in (1, 3):
        some = lse.clone()
        some[::3, 1], some[1::3, 2] = math.inf, -math.inf
        got = attention_mass(q, k, some, cu, n_splits=n)
        some[::3, 1] = -math.inf
        assert torch.equal(got, attention_mass(q, k, some, cu, n_splits=n))
        assert not torch.equal(got, attention_mass(q, k, lse, cu, n_splits=n))


def test_packed_part_that_outlasts_a_wait(cuda):
    """One part of 2.4e8 keys runs for longer than a bounded wait: no warp takes that for a fault.
    Scores of 0: lse = log(keys), whose fp32 sum of whole numbers below 2^28 is exact."""
    from linattn_b200 import _lib as L
    from linattn_b200 import packed_attention

    n, d = 240_000_005, 64
    if torch.cuda.mem_get_info()[0] < 3 * n * d:
        pytest.skip("needs 46 GB")
    q = torch.ones(1, 1, d, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(n, 1, d, dtype=torch.bfloat16, device="cuda")
    o, lse = packed_attention(q, k, k, _cu([1]), _cu([n]), n_splits=1)
    assert L.read_status(cuda) == 0
    assert (o == 0).all()
    assert abs(float(lse) - math.log(n)) <= 2.0 ** -19 * math.log(n)
    del k
    torch.cuda.empty_cache()
