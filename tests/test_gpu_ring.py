"""The token cache of windowed attention on the GPU (SinkWindowStreamingAttention) against a per-token float64 statement:
what it holds exactly, what queries answer element by element within the statement's bounds."""

import math

import pytest
import torch

import sink_window_attention as swa
import window_reference as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
STORAGE = [None, "fp4"]


def rand(g, dtype, *shape):
    return torch.randn(*shape, generator=g).to(dtype)


def build(streams, heads, kv, d, dv, window, sinks, dtype, storage, **kw):
    a = swa.SinkWindowStreamingAttention(d, dv, streams=streams, heads=heads, kv_heads=kv, window=window, sinks=sinks,
                                         dtype=dtype, storage=storage, device=DEV, **kw)
    return a, ref.TokenCache(streams, window, sinks, storage)


def check_items(a, cache):
    keys, values, positions = (x.cpu() for x in a.items())
    for s in range(a.streams):
        want = torch.full((a.sinks + a.window,), -1, dtype=torch.int32)
        wk, wv = torch.zeros(keys.shape[1:]), torch.zeros(values.shape[1:])
        wk, wv = wk.double(), wv.double()
        for p, (k, v) in cache.held[s].items():
            want[cache.slot(p)] = p
            wk[:, cache.slot(p)], wv[:, cache.slot(p)] = k, v
        assert torch.equal(positions[s], want)
        torch.testing.assert_close(keys[s], wk.to(a.dtype), rtol=0, atol=0, equal_nan=True)
        torch.testing.assert_close(values[s], wv.to(a.dtype), rtol=0, atol=0, equal_nan=True)
    assert a.lengths.tolist() == cache.n


def check_out(out, a, cache, q):
    for s in range(a.streams):
        want = cache.query(s, q[s], a.scale, a.dtype)
        if want is None:
            assert not out[s].any()
        else:
            assert ref.over(out[s], want) <= 1.0, (s, ref.over(out[s], want))


CASES = [  # streams heads kv d dv window sinks
    (1, 1, 1, 1, 1, 1, 0),
    (2, 2, 1, 32, 32, 5, 2),
    (1, 3, 3, 40, 24, 33, 1),
    (3, 4, 2, 64, 64, 20, 4),
    (1, 8, 1, 96, 80, 40, 16),
    (2, 2, 2, 128, 128, 31, 33),
    (1, 20, 1, 128, 64, 37, 3),
    (1, 34, 2, 33, 97, 9, 0),
]


@pytest.mark.parametrize("storage", STORAGE)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("streams,heads,kv,d,dv,window,sinks", CASES)
def test_steps(streams, heads, kv, d, dv, window, sinks, dtype, storage):
    a, cache = build(streams, heads, kv, d, dv, window, sinks, dtype, storage)
    g = torch.Generator().manual_seed(d + window)
    q = rand(g, dtype, streams, heads, d)
    assert not a.query(q.to(DEV)).any()
    for i in range(2 * (window + sinks) + 3):
        q, k, v = rand(g, dtype, streams, heads, d), rand(g, dtype, streams, kv, d), rand(g, dtype, streams, kv, dv)
        out = a.step(q.to(DEV), k.to(DEV), v.to(DEV))
        for s in range(streams):
            cache.put(s, k[s], v[s])
        check_out(out, a, cache, q)
    check_items(a, cache)
    again = a.query(q.to(DEV))
    assert torch.equal(again, out)


@pytest.mark.parametrize("storage", STORAGE)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,window,sinks", [(1, 1, 900, 4), (6, 2, 300, 40), (4, 1, 2000, 0)])
def test_extend_and_split_queries(heads, kv, window, sinks, dtype, storage):
    """Bulk prompts of several lengths, up to ones that lap the ring twice, then steps; enough tiles for a split."""
    a, cache = build(3, heads, kv, 64, 48, window, sinks, dtype, storage)
    g = torch.Generator().manual_seed(window)
    for rows, counts in ((window // 3, None), (window + 50, [window + 50, 0, 7]), (2 * window + 9, [5, 2 * window + 9, 1])):
        k, v = rand(g, dtype, 3, kv, rows, 64), rand(g, dtype, 3, kv, rows, 48)
        take = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV)
        a.extend(k.to(DEV), v.to(DEV), counts=take)
        for s in range(3):
            for i in range(rows if counts is None else counts[s]):
                cache.put(s, k[s, :, i], v[s, :, i])
        check_items(a, cache)
        for _ in range(2):
            q, k1, v1 = rand(g, dtype, 3, heads, 64), rand(g, dtype, 3, kv, 64), rand(g, dtype, 3, kv, 48)
            out = a.step(q.to(DEV), k1.to(DEV), v1.to(DEV))
            for s in range(3):
                cache.put(s, k1[s], v1[s])
            check_out(out, a, cache, q)
        a.update(k1.to(DEV), v1.to(DEV))
        for s in range(3):
            cache.put(s, k1[s], v1[s])
        check_out(a.query(q.to(DEV)), a, cache, q)
    check_items(a, cache)


def test_codes_of_borders():
    """Every border between 4-bit values, zeros, tiny and huge blocks, and blocks that are not finite."""
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.9, 0.0])
    rows = []
    for scale in (1.0, 2.0 ** -20, 2.0 ** 100, 2.0 ** -130, 2.0 ** -145):
        for eps in (-2.0 ** -20, 0.0, 2.0 ** -20):
            x = torch.zeros(64)
            x[:10] = borders * (1 + eps)
            x[10:20] = -borders * (1 + eps)
            x[32] = 6.0
            rows.append(x * scale)
    for bad in (math.inf, -math.inf, math.nan):
        x = torch.ones(64)
        x[40] = bad
        rows.append(x)
    rows.append(torch.full((64,), 3.4e38))
    rows.append(torch.zeros(64))
    k = torch.stack(rows)[None, None]
    n = k.shape[2]
    a, cache = build(1, 1, 1, 64, 64, n, 0, torch.float32, "fp4")
    a.extend(k.to(DEV), -k.to(DEV))
    b, _ = build(1, 1, 1, 64, 64, n, 0, torch.float32, "fp4")
    for i in range(n):
        cache.put(0, k[0, :, i], -k[0, :, i])
        b.step(k[:, :, i].to(DEV), k[:, :, i].to(DEV), -k[:, :, i].to(DEV))
    check_items(a, cache)
    check_items(b, cache)


@pytest.mark.parametrize("storage", STORAGE)
@pytest.mark.parametrize("dtype", DTYPES)
def test_slots_without_a_token_are_never_read(dtype, storage):
    """A stream that starts anew does not see what its slots held before, whatever that was."""
    a, cache = build(2, 2, 1, 64, 64, 50, 4, dtype, storage)
    bad = torch.full((2, 1, 54, 64), math.nan, dtype=dtype, device=DEV)
    a.extend(bad, bad)
    a.reset([1])
    assert a.lengths.tolist() == [54, 0]
    a.reset()
    g = torch.Generator().manual_seed(1)
    for _ in range(37):
        q, k, v = rand(g, dtype, 2, 2, 64), rand(g, dtype, 2, 1, 64), rand(g, dtype, 2, 1, 64)
        out = a.step(q.to(DEV), k.to(DEV), v.to(DEV))
        for s in range(2):
            cache.put(s, k[s], v[s])
        check_out(out, a, cache, q)
    check_items(a, cache)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
@pytest.mark.parametrize("storage", STORAGE)
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(dtype, storage, scale):
    a, cache = build(1, 2, 1, 32, 32, 40, 2, dtype, storage, scale=scale)
    g = torch.Generator().manual_seed(2)
    for _ in range(45):
        q, k, v = rand(g, dtype, 1, 2, 32), rand(g, dtype, 1, 1, 32), rand(g, dtype, 1, 1, 32)
        out = a.step(q.to(DEV), k.to(DEV), v.to(DEV))
        cache.put(0, k[0], v[0])
    check_out(out, a, cache, q)


def test_strided_tokens():
    g = torch.Generator().manual_seed(3)
    qkv = rand(g, torch.bfloat16, 3, 4 * 64 + 2 * 64 + 2 * 48).to(DEV)  # one projection's rows
    q = qkv[:, :256].view(3, 4, 64)
    k, v = qkv[:, 256:384].view(3, 2, 64), qkv[:, 384:].view(3, 2, 48)
    for storage in STORAGE:
        a, _ = build(3, 4, 2, 64, 48, 16, 2, torch.bfloat16, storage)
        b, _ = build(3, 4, 2, 64, 48, 16, 2, torch.bfloat16, storage)
        for _ in range(3):
            x = a.step(q, k, v)
            y = b.step(q.contiguous(), k.contiguous(), v.contiguous())
            assert torch.equal(x, y)


@pytest.mark.parametrize("storage", STORAGE)
def test_captured_steps(storage):
    """A captured step, replayed with eager steps of the same object in between, advances the state like calls do."""
    g = torch.Generator().manual_seed(4)
    shape = (2, 4, 2, 64, 64, 700, 4, torch.bfloat16, storage)
    a, _ = build(*shape)
    b, _ = build(*shape)
    k, v = rand(g, torch.bfloat16, 2, 2, 690, 64).to(DEV), rand(g, torch.bfloat16, 2, 2, 690, 64).to(DEV)
    a.extend(k, v)
    b.extend(k, v)
    q, k1, v1 = (torch.zeros(2, h, 64, dtype=torch.bfloat16, device=DEV) for h in (4, 2, 2))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a.step(q, k1, v1)
    for i in range(25):
        for x, h in ((q, 4), (k1, 2), (v1, 2)):
            x.copy_(rand(g, torch.bfloat16, 2, h, 64))
        if i % 3 == 2:
            got = a.step(q, k1, v1)
        else:
            graph.replay()
            got = out
        want = b.step(q, k1, v1)
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
    for x, y in zip(a.items(), b.items()):
        assert torch.equal(x, y)


@pytest.mark.parametrize("storage", STORAGE)
def test_state_round_trip(storage):
    g = torch.Generator().manual_seed(5)
    shape = (2, 2, 1, 40, 40, 30, 3, torch.float16, storage)
    a, _ = build(*shape)
    b, _ = build(*shape)
    a.extend(rand(g, torch.float16, 2, 1, 77, 40).to(DEV), rand(g, torch.float16, 2, 1, 77, 40).to(DEV))
    b.load_state_dict(a.state_dict())
    q, k, v = (rand(g, torch.float16, 2, h, 40).to(DEV) for h in (2, 1, 1))
    assert torch.equal(a.step(q, k, v), b.step(q, k, v))
    for x, y in zip(a.items(), b.items()):
        assert torch.equal(x, y)


@pytest.mark.parametrize("storage", STORAGE)
def test_counts_past_31_bits(storage):
    """A stream's count goes back by whole windows where it would pass 2^31 - 1, and nothing else changes."""
    g = torch.Generator().manual_seed(6)
    shape = (2, 34, 2, 32, 32, 37, 3, torch.bfloat16, storage)  # 17 query heads a key head: counted by the second launch
    for step in (True, False):
        a, _ = build(*shape)
        b, _ = build(*shape)
        k, v = rand(g, torch.bfloat16, 2, 2, 60, 32).to(DEV), rand(g, torch.bfloat16, 2, 2, 60, 32).to(DEV)
        a.extend(k, v)
        state = a.state_dict()
        state["counts"] += (2 ** 31 - 3 - 60) // 37 * 37
        b.load_state_dict(state)
        for _ in range(80):
            q, k, v = (rand(g, torch.bfloat16, 2, h, 32).to(DEV) for h in (34, 2, 2))
            if step:
                assert torch.equal(a.step(q, k, v), b.step(q, k, v))
            else:
                for x in (a, b):
                    x.update(k, v)
                assert torch.equal(a.query(q), b.query(q))
        n = b.lengths.cpu()
        assert torch.all(n >= 40) and torch.all((n - a.lengths.cpu()) % 37 == 0)
        for x, y in zip(a.items()[:2], b.items()[:2]):
            assert torch.equal(x, y)


def test_state_refusals():
    a, _ = build(2, 1, 1, 8, 8, 4, 0, torch.float32, None)
    a.extend(torch.ones(2, 1, 3, 8), torch.ones(2, 1, 3, 8))
    state = a.state_dict()
    for wrong in (dict(counts=state["counts"] - 4), dict(cache=state["cache"][:2]), dict(counts=state["counts"][:1])):
        with pytest.raises(ValueError):
            a.load_state_dict(dict(state, **wrong))
    with pytest.raises(ValueError, match="no stream"):
        a.reset([0, 2])
    assert a.lengths.tolist() == [3, 3]


def test_more_tiles_than_one_row_of_a_launch():
    """2^20 + 3 tiles of slots: the last ones are filled and read like the first."""
    window = (1 << 25) + 77
    a, _ = build(1, 1, 1, 8, 8, window, 2, torch.bfloat16, "fp4")
    a._counts.fill_(1 << 25)
    k = (torch.arange(70 * 8).remainder(3) + 1).bfloat16().reshape(1, 1, 70, 8).to(DEV)
    a.extend(k, -k)
    keys, values, positions = a.items()
    at = slice(1 << 25, (1 << 25) + 70)
    assert torch.equal(keys[:, :, at], k) and torch.equal(values[:, :, at], -k)
    assert positions[0, at].tolist() == list(range(at.start, at.stop)) and not (positions[0, at.stop:] + 1).any()
    assert not keys[:, :, :at.start].any() and not keys[:, :, at.stop:].any()


def test_scale_zero_of_huge_logits():
    """Every token held weighs the same, also in tiles that only some waves have."""
    a, _ = build(1, 1, 1, 32, 32, 40, 0, torch.float32, None, scale=0.0)
    k, v = torch.full((1, 1, 35, 32), 1e18), torch.arange(35.0)[None, None, :, None].expand(1, 1, 35, 32)
    a.extend(k, v)
    out = a.query(torch.full((1, 1, 32), 1e18)).cpu()
    # 35 weights of 1: the sum is exact, the quotient 17 too
    assert torch.equal(out, torch.full((1, 1, 32), 17.0))
