"""The cache that keeps the most attended tokens and received weights where keys, values or logits are infinite or NaN."""

import math

import pytest
import torch

import heavy_hitter_attention as hha
import kept_reference as ref
import shared_prefix_attention as spa

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(seed, dtype, *shapes):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to(dtype) for s in shapes]


def ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)


def odd(x):
    """x with rows at an odd element, off their units."""
    room = torch.zeros(*x.shape[:-1], x.shape[-1] + 3, dtype=x.dtype, device=x.device)
    room[..., 1:1 + x.shape[-1]] = x
    return room[..., 1:1 + x.shape[-1]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,n,m,d,counts", [
    # rows that stay in LDS, a block of 32 not full
    (1, 1, 1, 5, 64, 64, None), (2, 4, 2, 9, 70, 64, [9, 4]), (1, 6, 2, 33, 150, 93, None), (3, 2, 2, 100, 300, 128, [99, 1, 64]),
    # tiles of rows, the last not full
    (1, 2, 2, 257, 257, 64, None), (2, 4, 1, 130, 200, 128, [130, 77]), (2, 2, 1, 190, 333, 40, [3, 190]),
    (1, 3, 3, 200, 200, 93, [131])])
def test_received_weights_of_keys_that_hide(b, h, hk, n, m, d, counts, dtype):
    """Keys whose logits are -inf for every row receive 0, whatever fills up a block of rows; the others what they do."""
    q, k, pk = make(b + n + m + d, dtype, (b, h, n, d), (b, hk, m, d), (1, hk, 50, d))
    q[..., 0] = 1.0
    hide = torch.zeros(m, dtype=torch.bool)
    hide[2::7] = True
    finite = k.clone()
    k[:, :, hide, 0] = -math.inf
    want = ref.received(q, finite, counts=counts, hide=hide)
    assert (want[0][:, :, hide] == 0).all()
    lse = spa.shared_prefix_attention(q.to(DEV), k.to(DEV), k.to(DEV).nan_to_num(0.0, 0.0, 0.0), pk.to(DEV), pk.to(DEV),
                                      counts=ints(counts), with_lse=True)[1]
    given = ref.received(q, finite, counts=counts, hide=hide, lse=lse.cpu())
    for view in (lambda x: x, odd):
        got = hha.received_attention(view(q.to(DEV)), view(k.to(DEV)), counts=ints(counts))
        assert got[:, :, hide.to(DEV)].eq(0).all()
        assert ref.over(got, want) <= 1.0
        got = hha.received_attention(view(q.to(DEV)), view(k.to(DEV)), counts=ints(counts), lse=lse)
        assert ref.over(got, given) <= 1.0


def cache_of(dtype, streams=2, heads=4, kv=2, kept=12, recent=5, d=32, dv=24):
    c = hha.HeavyHitterStreamingAttention(d, dv, streams=streams, heads=heads, kv_heads=kv, kept=kept, recent=recent, dtype=dtype,
                                          device=DEV)
    return c, ref.Cache(streams, kv, kept, recent)


def token(c, seed):
    return make(seed, c.dtype, (c.streams, c.heads, c.dim), (c.streams, c.kv_heads, c.dim), (c.streams, c.kv_heads, c.value_dim))


def follow(c, want, q, k=None, v=None, prefix=None):
    """A step or query of both, the statement from the cache's own weights: the same tokens, outputs and weights within their
    bounds."""
    want.adopt(c.weights.cpu())
    kw = {} if prefix is None else dict(prefix=[x.to(DEV) for x in prefix])
    if k is None:
        got = c.query(q.to(DEV), **kw)
    else:
        got = c.step(q.to(DEV), k.to(DEV), v.to(DEV), **kw)
        want.update(k, v)
    value, near = want.query(q, 1 / math.sqrt(c.dim), prefix, None if prefix is None else prefix[0].shape[1])
    fine = torch.isfinite(value).all(-1)
    assert ref.over(got.cpu()[fine], (value[fine], near[fine])) <= 1.0 and not torch.isfinite(got.cpu()[~fine]).any()
    weights, bound, positions = want.state()
    torch.cuda.synchronize()
    assert torch.equal(c.positions.cpu(), positions)
    assert ref.over(c.weights, (weights, bound)) <= 1.0
    return got


# 3e38: finite, with logits beyond fp32; fp16 has no such value
BAD = [(x, t) for x in (math.nan, math.inf, 3e38) for t in DTYPES if not (x == 3e38 and t == torch.float16)]
PATHS = [dict(), dict(heads=40, kv=1, streams=1), dict(heads=16, kv=1, streams=1, kept=1400, recent=9),
         dict(kept=3000, recent=9, streams=1)]


@pytest.mark.parametrize("bad,dtype", BAD)
@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("kw", PATHS)
def test_tokens_with_keys_that_are_not_finite_leave_first(kw, prefix, bad, dtype):
    """Two of the tokens that a full cache holds for their weights, in slots that are not the first."""
    c, want = cache_of(dtype, **kw)
    n = c.kept + c.recent + 40
    k, v = make(1, dtype, (c.streams, c.kv_heads, n, c.dim), (c.streams, c.kv_heads, n, c.value_dim))
    w = torch.rand(c.streams, c.kv_heads, n, generator=torch.Generator().manual_seed(2)) + 1.0
    k[0, 0, [20, 33], 0], w[0, 0, [20, 33]] = bad, 9.0
    c.start(k.to(DEV), v.to(DEV), w.to(DEV))
    want.start(k, v, w)
    pk, pv = make(3, dtype, (c.kv_heads, 60, c.dim), (c.kv_heads, 60, c.value_dim))
    for t in range(5):
        q, k, v = token(c, 10 + t)
        q[..., 0] = 3.0
        out = follow(c, want, q, k, v, (pk, pv) if prefix else None)
        group = c.heads // c.kv_heads
        # the first step finds them out; the next two send one away each, before their queries
        assert torch.isfinite(out).all() if t > 1 else out[0, :group].isnan().all()
        assert torch.isfinite(out[0, group:]).all() and torch.isfinite(out[1:]).all() and torch.isfinite(c.weights).all()
    assert not {20, 33} & set(c.positions[0, 0].tolist())


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_that_come_with_such_keys(dtype):
    """Two while the cache fills: they hold their slots until it is full, and leave then."""
    c, want = cache_of(dtype)
    for t in range(30):
        q, k, v = token(c, 50 + t)
        if t in (3, 6):
            k[1, 0, 5] = math.nan
        out = follow(c, want, q, k, v)
        assert torch.isfinite(out[0]).all()
    assert torch.isfinite(out).all() and not {3, 6} & set(c.positions[1, 0].tolist())


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_with_such_keys(dtype):
    """All rows that see the key have weights of NaN, so no token a weight; the streams get rid of it all the same."""
    c, _ = cache_of(dtype)
    q, k, v = make(4, dtype, (c.streams, c.heads, 40, c.dim), (c.streams, c.kv_heads, 40, c.dim), (c.streams, c.kv_heads, 40, c.value_dim))
    k[0, 1, 3, 7] = math.nan
    c.prefill(q.to(DEV), k.to(DEV), v.to(DEV))
    assert torch.isfinite(c.weights).all() and 3 in c.positions[0, 1].tolist()
    for t in range(3):
        out = c.step(*(x.to(DEV) for x in token(c, 80 + t)))
    assert torch.isfinite(out).all() and 3 not in c.positions[0, 1].tolist()


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_without_queries(dtype):
    """Weights of 0 all over: the first query finds the tokens out."""
    c, want = cache_of(dtype)
    for t in range(40):
        q, k, v = token(c, 200 + t)
        if t in (2, 9):
            k[0, 0] = -math.inf
        c.update(k.to(DEV), v.to(DEV))
        want.update(k, v)
    assert torch.equal(c.positions.cpu(), want.state()[2]) and {2, 9} <= set(c.positions[0, 0].tolist())
    for t in range(4):
        q, k, v = token(c, 300 + t)
        out = follow(c, want, q, k, v)
    assert torch.isfinite(out).all() and not {2, 9} & set(c.positions[0, 0].tolist())


@pytest.mark.parametrize("bad,dtype", BAD + [(-math.inf, t) for t in DTYPES])
@pytest.mark.parametrize("kw", PATHS)
def test_queries_that_are_not_finite_blame_no_token(kw, bad, dtype):
    c, want = cache_of(dtype, **kw)
    n = c.kept + c.recent + 10
    k, v = make(5, dtype, (c.streams, c.kv_heads, n, c.dim), (c.streams, c.kv_heads, n, c.value_dim))
    k[:, :, ::3] *= 16.0
    w = torch.rand(c.streams, c.kv_heads, n, generator=torch.Generator().manual_seed(6))
    c.start(k.to(DEV), v.to(DEV), w.to(DEV))
    want.start(k, v, w)
    for t in range(3):
        q, k, v = token(c, 400 + t)
        q[0, 1, 2] = bad
        follow(c, want, q, k, v)
        assert c.weights.ge(0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_of_empty_streams_behind_a_prefix_that_hides(dtype):
    """Rows that are there with logits of -inf alone give NaN, as a softmax of them; no rows at all zero."""
    c, _ = cache_of(dtype, streams=4)
    q = token(c, 1)[0]
    q[..., 0] = 1.0
    pk, pv = make(2, dtype, (2, c.kv_heads, 60, c.dim), (2, c.kv_heads, 60, c.value_dim))
    pk[..., 0] = -math.inf
    got = c.query(q.to(DEV), prefix=(pk.to(DEV), pv.to(DEV)), prefix_lengths=ints([60, 0]))
    assert got[:2].isnan().all() and got[2:].eq(0).all()
    got = c.query(q.to(DEV), prefix=(pk.to(DEV), pv.to(DEV)))
    assert got.isnan().all() and c.weights.eq(0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv", [129, 171])
def test_more_key_heads_than_half_the_compute_units(kv, dtype):
    c, want = cache_of(dtype, streams=1, heads=kv, kv=kv, kept=1190, recent=9, d=96, dv=100)
    k, v = make(7, dtype, (1, kv, 1230, c.dim), (1, kv, 1230, c.value_dim))
    w = torch.rand(1, kv, 1230, generator=torch.Generator().manual_seed(8))
    c.start(k.to(DEV), v.to(DEV), w.to(DEV))
    want.start(k, v, w)
    for t in range(2):
        q, k, v = token(c, 500 + t)
        follow(c, want, q, k, v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first", [0.0, 1000.0, 3.0e5])
@pytest.mark.parametrize("kw", PATHS[:1] + PATHS[3:])
def test_weights_are_fp32_sums(kw, first, dtype):
    """Many queries without tokens between them: every addition rounds at 2^-24 of the weight that comes out, and what a query
    adds is as near as a step's is."""
    c, _ = cache_of(dtype, **kw)
    n, queries, scale = c.recent + c.kept, 300, 1 / math.sqrt(c.dim)
    k, v = make(9, dtype, (c.streams, c.kv_heads, n, c.dim), (c.streams, c.kv_heads, n, c.value_dim))
    c.start(k.to(DEV), v.to(DEV), torch.full((c.streams, c.kv_heads, n), first, device=DEV))
    q = make(10, dtype, (queries, c.streams, c.heads, c.dim))[0]
    for t in range(queries):
        c.query(q[t].to(DEV))
    group = c.heads // c.kv_heads
    rows = q.double().view(queries, c.streams, c.kv_heads, group, c.dim).permute(1, 2, 0, 3, 4).flatten(2, 3)
    p, _, rel, _ = zip(*(ref._weights(rows[s, h], k[s, h].double(), torch.zeros(rows.shape[2], n, dtype=torch.bool), scale, c.dim)
                         for s in range(c.streams) for h in range(c.kv_heads)))
    p, rel = torch.stack(p), torch.stack(rel)
    want = (first + p.sum(1)).view(c.streams, c.kv_heads, n)
    near = ((p * (2 * rel + ref.F24 * (group + 8))).sum(1)).view(want.shape) + queries * ref.F24 * want
    at = c.positions.cpu()
    assert (at >= 0).sum(-1).eq(n).all()
    for s in range(c.streams):
        for h in range(c.kv_heads):
            held = at[s, h] >= 0
            got = c.weights[s, h].cpu()[held]
            assert ref.over(got, (want[s, h][at[s, h][held]], near[s, h][at[s, h][held]])) <= 1.0
