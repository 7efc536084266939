"""The cache that keeps the most attended tokens on the GPU against its float64 statement: what it holds slot by slot,
outputs and weights within the bounds that the statement derives from the roundings."""

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


def same_rows(cache, want):
    """Slots, tokens and rows are those of the statement, exactly."""
    keys, values, positions, weights = (x.cpu() for x in cache.items())
    assert torch.equal(positions, want.state()[2])
    for s in range(want.streams):
        for h in range(want.kv_heads):
            for i, x in enumerate(want.heads[s][h]["slots"]):
                assert torch.equal(keys[s, h, i], torch.zeros_like(keys[s, h, i]) if x is None else x[2]), (s, h, i)
                assert torch.equal(values[s, h, i], torch.zeros_like(values[s, h, i]) if x is None else x[3]), (s, h, i)
    assert torch.equal(weights, cache.weights.cpu()) and bool((weights[positions < 0] == 0).all())


def follow(cache, want, q, k=None, v=None, prefix=None, plen=None, scale=None):
    """One step (or query) of both; the statement starts from the cache's own weights."""
    want.adopt(cache.weights.cpu())
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    kw = {} if prefix is None else dict(prefix=[x.to(DEV) for x in prefix], prefix_lengths=ints([plen] if plen is not None else None))
    if k is None:
        got = cache.query(q.to(DEV), **kw)
    else:
        got = cache.step(q.to(DEV), k.to(DEV), v.to(DEV), **kw)
        want.update(k, v)
    out = want.query(q, scale, prefix, plen if plen is not None else (None if prefix is None else prefix[0].shape[1]))
    weights, bound, positions = want.state()
    torch.cuda.synchronize()
    assert torch.equal(cache.positions.cpu(), positions)
    assert ref.over(got, out) <= 1.0
    assert ref.over(cache.weights, (weights, bound)) <= 1.0
    return got


SHAPES = [  # streams heads kv kept recent d dv steps
    (1, 1, 1, 1, 1, 1, 1, 6),
    (1, 2, 1, 3, 2, 16, 24, 14),
    (2, 4, 2, 40, 31, 64, 64, 110),
    (1, 3, 1, 30, 1, 33, 40, 70),
    (2, 2, 2, 5, 64, 93, 77, 90),
    (1, 40, 1, 20, 12, 32, 64, 50),
    (3, 8, 2, 70, 25, 128, 128, 110),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("streams,heads,kv,kept,recent,d,dv,steps", SHAPES)
def test_steps_from_empty(streams, heads, kv, kept, recent, d, dv, steps, dtype):
    cache = hha.HeavyHitterStreamingAttention(d, dv, streams=streams, heads=heads, kv_heads=kv, kept=kept, recent=recent,
                                              dtype=dtype)
    want = ref.Cache(streams, kv, kept, recent)
    for t in range(steps):
        q, k, v = make(1000 + t, dtype, (streams, heads, d), (streams, kv, d), (streams, kv, dv))
        follow(cache, want, q, k, v)
        assert cache.lengths.tolist() == [t + 1] * streams
        if t % 5 == 3:
            follow(cache, want, q.flip(0))
        if t % 7 == 4:  # a token that no query follows
            want.adopt(cache.weights.cpu())
            cache.update(k.to(DEV), v.to(DEV))
            want.update(k, v)
            assert torch.equal(cache.positions.cpu(), want.state()[2])
            break
    same_rows(cache, want)
    for t in range(steps, steps + 2 * recent + 4 if streams * heads < 20 else steps + 4):
        q, k, v = make(1000 + t, dtype, (streams, heads, d), (streams, kv, d), (streams, kv, dv))
        follow(cache, want, q, k, v)
    same_rows(cache, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("streams,heads,kv,kept,recent,d,dv,steps", SHAPES)
def test_steps_of_full_caches(streams, heads, kv, kept, recent, d, dv, steps, dtype):
    cache = hha.HeavyHitterStreamingAttention(d, dv, streams=streams, heads=heads, kv_heads=kv, kept=kept, recent=recent,
                                              dtype=dtype)
    want = ref.Cache(streams, kv, kept, recent)
    n = 2 * (kept + recent)
    k, v = make(5, dtype, (streams, kv, n, d), (streams, kv, n, dv))
    w = torch.rand(streams, kv, n, generator=torch.Generator().manual_seed(6))
    cache.start(k.to(DEV), v.to(DEV), w.to(DEV))
    want.start(k, v, w)
    same_rows(cache, want)
    for t in range(12):
        q, k, v = make(2000 + t, dtype, (streams, heads, d), (streams, kv, d), (streams, kv, dv))
        follow(cache, want, q, k, v)
    same_rows(cache, want)


def rows(streams, kv, n, d, dv, dtype, seed=0):
    return make(seed, dtype, (streams, kv, n, d), (streams, kv, n, dv))


@pytest.mark.parametrize("kind", ["random", "equal", "two", "extreme", "signs"])
@pytest.mark.parametrize("streams,kv,n,kept,recent,counts", [
    (1, 1, 1, 1, 1, None), (2, 1, 40, 16, 8, None), (3, 2, 100, 37, 5, [100, 0, 41]), (2, 2, 3000, 1000, 77, [2999, 1078]),
    (1, 2, 2500, 31, 1, None), (4, 1, 64, 100, 20, [64, -1, 1, 99]), (1, 1, 5000, 1500, 3400, None),
    # more rows than are held in registers, and caches of more tiles than compute units
    (1, 1, 9000, 500, 100, None), (40, 4, 60, 40, 9, [60, 0, 3, -1] * 10), (2, 4, 17000, 1000, 200, [17000, 16383])])
def test_start(streams, kv, n, kept, recent, counts, kind):
    """Which tokens of a prompt stay: random weights, equal ones (the first stay), two values, extremes, both signs."""
    dtype, d, dv = torch.bfloat16, 16, 8
    k, v = rows(streams, kv, n, d, dv, dtype)
    g = torch.Generator().manual_seed(n)
    w = torch.rand(streams, kv, n, generator=g)
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "two":
        w = (w > 0.6).float()
    elif kind == "extreme":
        for i, x in enumerate((math.inf, 0.0, math.nan, 1e-45, 3e38, -0.0, 1e-38, -math.inf)):
            w[..., i::11] = x
    elif kind == "signs":
        w = w - 0.5
    cache = hha.HeavyHitterStreamingAttention(d, dv, streams=streams, heads=kv, kept=kept, recent=recent, dtype=dtype)
    want = ref.Cache(streams, kv, kept, recent)
    old = rows(streams, kv, 3, d, dv, dtype, seed=9)
    ow = torch.ones(streams, kv, 3)
    cache.start(*(x.to(DEV) for x in (*old, ow)))  # what streams without a new prompt keep
    want.start(*old, ow)
    cache.start(k.to(DEV), v.to(DEV), w.to(DEV), counts=ints(counts))
    want.start(k, v, w, counts)
    same_rows(cache, want)
    got, held = cache.weights.cpu(), want.state()[0]
    assert torch.equal(got.double(), held)
    assert cache.lengths.tolist() == [3 if counts is not None and counts[s] <= 0 else
                                      min(n, n if counts is None else counts[s]) for s in range(streams)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("streams,heads,kv,kept,recent,d,dv,p,plen", [
    (1, 1, 1, 4, 2, 8, 8, 1, None), (4, 8, 2, 30, 10, 64, 64, 200, 130), (2, 6, 2, 12, 5, 93, 77, 700, None),
    (3, 4, 4, 300, 40, 128, 128, 64, 0), (2, 6, 3, 600, 30, 128, 96, 150, 149)])
def test_steps_behind_a_prefix(streams, heads, kv, kept, recent, d, dv, p, plen, dtype):
    cache = hha.HeavyHitterStreamingAttention(d, dv, streams=streams, heads=heads, kv_heads=kv, kept=kept, recent=recent,
                                              dtype=dtype)
    want = ref.Cache(streams, kv, kept, recent)
    prefix = make(77, dtype, (kv, p, d), (kv, p, dv))
    q = make(1, dtype, (streams, heads, d))[0]
    follow(cache, want, q, prefix=prefix, plen=plen)  # the prefix alone
    for t in range(kept + recent + 6 if kept < 100 else 8):
        q, k, v = make(3000 + t, dtype, (streams, heads, d), (streams, kv, d), (streams, kv, dv))
        follow(cache, want, q, k, v, prefix=prefix, plen=plen)
    same_rows(cache, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefixes_of_groups(dtype):
    """Two prefixes, two streams each."""
    streams, heads, kv, d, p = 4, 4, 2, 32, 90
    cache = hha.HeavyHitterStreamingAttention(d, d, streams=streams, heads=heads, kv_heads=kv, kept=20, recent=4, dtype=dtype)
    pk, pv = make(3, dtype, (2, kv, p, d), (2, kv, p, d))
    q, k, v = make(4, dtype, (streams, heads, d), (streams, kv, d), (streams, kv, d))
    got = cache.step(q.to(DEV), k.to(DEV), v.to(DEV), prefix=(pk.to(DEV), pv.to(DEV)), prefix_lengths=ints([90, 33]))
    want = ref.prefix_attention(q[:, :, None], k[:, :, None], v[:, :, None], pk, pv, prefix_lengths=[90, 33])
    assert ref.over(got[:, :, None], want["out"]) <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,kept", [(4, 1, 9000), (32, 1, 3000), (8, 8, 2500), (6, 3, 560), (6, 3, 900)])
def test_caches_split_over_workgroups(heads, kv, kept, dtype):
    recent, d, dv = 100, 40, 64
    cache = hha.HeavyHitterStreamingAttention(d, dv, heads=heads, kv_heads=kv, kept=kept, recent=recent, dtype=dtype)
    want = ref.Cache(1, kv, kept, recent)
    n = kept + recent + 50
    k, v = make(8, dtype, (1, kv, n, d), (1, kv, n, dv))
    w = torch.rand(1, kv, n, generator=torch.Generator().manual_seed(1))
    cache.start(k.to(DEV), v.to(DEV), w.to(DEV))
    want.start(k, v, w)
    for t in range(3):
        q, k, v = make(4000 + t, dtype, (1, heads, d), (1, kv, d), (1, kv, dv))
        follow(cache, want, q, k, v)
    follow(cache, want, q)
    follow(cache, want, q, k, v)
    same_rows(cache, want)


@pytest.mark.parametrize("scale", [-0.7, 0.0, 3.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(dtype, scale):
    cache = hha.HeavyHitterStreamingAttention(32, 32, streams=2, heads=4, kv_heads=2, kept=10, recent=3, dtype=dtype, scale=scale)
    want = ref.Cache(2, 2, 10, 3)
    for t in range(20):
        q, k, v = make(5000 + t, dtype, (2, 4, 32), (2, 2, 32), (2, 2, 32))
        follow(cache, want, q, k, v, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_and_steps_behind_a_prefix(dtype):
    """A run as it is used: prompts of several lengths behind a shared prefix are answered and begin the streams, steps
    follow, one stream begins anew meanwhile."""
    streams, heads, kv, d, dv, p, n, kept, recent = 3, 6, 2, 64, 48, 150, 120, 40, 20
    counts, scale = [120, 1, 77], 1 / math.sqrt(d)
    q, k, v, pk, pv = make(11, dtype, (streams, heads, n, d), (streams, kv, n, d), (streams, kv, n, dv), (kv, p, d), (kv, p, dv))
    cache = hha.HeavyHitterStreamingAttention(d, dv, streams=streams, heads=heads, kv_heads=kv, kept=kept, recent=recent, dtype=dtype)
    prefix = pk.to(DEV), pv.to(DEV)
    out = cache.prefill(q.to(DEV), k.to(DEV), v.to(DEV), counts=ints(counts), prefix=prefix)
    want = ref.prefix_attention(q, k, v, pk[None], pv[None], lengths=counts, counts=counts)
    assert ref.over(out, want["out"]) <= 1.0
    lse = spa.shared_prefix_attention(q.to(DEV), k.to(DEV), v.to(DEV), *prefix, lengths=ints(counts), counts=ints(counts),
                                      with_lse=True)[1]
    weights = hha.received_attention(q.to(DEV), k.to(DEV), lengths=ints(counts), counts=ints(counts), lse=lse)
    assert ref.over(weights, ref.received(q, k, lengths=counts, counts=counts, lse=lse.cpu())) <= 1.0
    own = ref.Cache(streams, kv, kept, recent)
    own.start(k, v, weights.cpu(), counts)
    same_rows(cache, own)
    for t in range(30):
        q, k, v = make(6000 + t, dtype, (streams, heads, d), (streams, kv, d), (streams, kv, dv))
        follow(cache, own, q, k, v, prefix=(pk, pv), scale=scale)
        if t == 12:
            cache.reset([1])
            own.reset(1)
    same_rows(cache, own)
