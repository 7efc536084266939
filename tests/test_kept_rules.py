"""The rule of the cache that keeps the most attended tokens on tokens whose keys are not finite, by its statement alone."""

import math

import torch

import kept_reference as ref


def held(cache):
    return [-1 if x is None else x[0] for x in cache.heads[0][0]["slots"]]


def step(cache, g, key=None, query=True):
    k, v, q = (torch.randn(1, 1, 8, generator=g) for _ in range(3))
    cache.update(k if key is None else key, v)
    return cache.query(q, 1 / math.sqrt(8))[0] if query else None


def test_two_that_come_while_the_cache_fills():
    g, cache = torch.Generator().manual_seed(1), ref.Cache(1, 1, 12, 5)
    for t in range(40):
        out = step(cache, g, torch.full((1, 1, 8), math.nan) if t in (3, 6) else None)
        assert bool(torch.isfinite(out).all()) == (t < 3 or t > 17)  # full with token 16; 17 and 18 send them away
    assert not {3, 6} & set(held(cache))


def test_no_weights_and_no_queries():
    g, cache = torch.Generator().manual_seed(2), ref.Cache(1, 1, 12, 5)
    k, v = torch.randn(1, 1, 40, 8, generator=g), torch.randn(1, 1, 40, 8, generator=g)
    k[0, 0, 3, 1] = math.nan
    cache.start(k, v, torch.full((1, 1, 40), math.nan))
    assert 3 in held(cache)
    for t in range(6):
        step(cache, g, torch.full((1, 1, 8), math.inf) if t == 2 else None, query=False)
    assert 3 in held(cache)
    assert cache.query(torch.ones(1, 1, 8), 1.0)[0].isnan().all()
    for t in range(6):
        out = step(cache, g, query=t == 5)
    assert torch.isfinite(out).all() and not {3, 42} & set(held(cache))


def test_a_query_that_is_not_finite_is_not_theirs():
    g, cache = torch.Generator().manual_seed(3), ref.Cache(1, 1, 6, 2)
    for t in range(8):
        step(cache, g)
    before = cache.state()[0]
    assert cache.query(torch.full((1, 1, 8), math.nan), 1.0)[0].isnan().all()
    assert torch.equal(cache.state()[0], before)


def test_shares_of_more_key_heads_than_half_the_compute_units():
    """float32 key heads of long caches are shared by three workgroups up to 170 of them; a workspace for partials says so."""
    import _native

    def shared(dtype, streams, kept):
        pitch = (kept + 33 + 31) // 32 * 32
        return _native.load_library().sta_heavy_attention_bytes(dtype, streams, 8, 8, 128, 128, 32, kept, 0, 0) > 4 * streams * 8 * pitch

    assert shared(0, 16, 2015) and shared(0, 17, 2015) and shared(0, 21, 2015)
    assert not shared(0, 22, 2015) and not shared(0, 32, 2015) and not shared(0, 17, 700)
    assert shared(1, 16, 2015) and not shared(1, 17, 2015) and not shared(2, 17, 16000)
