"""The cache that keeps the most attended tokens, received weights and the attention over a shared prefix as programs use
them: strides and alignments, values that are not finite, graphs, streams, saved states, long offsets."""

import math
import threading

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


def inputs(b, h, hk, n, m, sets, p, d, dv, dtype, seed=0):
    return make(seed, dtype, (b, h, n, d), (b, hk, m, d), (b, hk, m, dv), (sets, hk, p, d), (sets, hk, p, dv))


def check(got, want):
    worst = {name: ref.over(got[name], want[name]) for name in want}
    assert all(x <= 1.0 for x in worst.values()), worst


def attend(x, **kw):
    out, lse = spa.shared_prefix_attention(*x, with_lse=True, **kw)
    return {"out": out, "lse": lse}


def odd(x):
    """x with rows at an odd element, one more column apart."""
    room = torch.zeros(*x.shape[:-1], x.shape[-1] + 3, dtype=x.dtype, device=x.device)
    room[..., 1:1 + x.shape[-1]] = x
    return room[..., 1:1 + x.shape[-1]]


def rows_first(x):
    """[B,H,N,D] as a view of [B,N,H,D]."""
    return x.transpose(1, 2).contiguous().transpose(1, 2)


def spread(x):
    """Every other row of twice as many."""
    room = torch.full((*x.shape[:2], 2 * x.shape[2], x.shape[3]), math.nan, dtype=x.dtype, device=x.device)
    room[:, :, ::2] = x
    return room[:, :, ::2]


SIZES = [  # b h hk n m sets p d dv: one row, few, many; widths with and without tiles straight to LDS
    (3, 4, 2, 1, 40, 1, 300, 64, 64), (16, 16, 4, 40, 70, 2, 130, 128, 128), (9, 12, 12, 150, 150, 3, 100, 64, 64),
    (40, 8, 2, 1, 90, 1, 700, 128, 128), (2, 4, 2, 20, 33, 1, 65, 40, 24), (64, 32, 32, 20, 20, 1, 70, 64, 64),
    (24, 16, 16, 130, 150, 2, 90, 128, 128), (20, 32, 16, 140, 140, 1, 65, 64, 64),  # the last: rows that one workgroup finishes
    # prefixes and own tokens in walks of their own: tiles of 32 and of 128, many partials and few
    (3, 4, 2, 1, 40, 1, 5000, 64, 64), (16, 8, 2, 10, 40, 1, 600, 128, 128), (6, 4, 4, 33, 50, 2, 800, 64, 64),
    (12, 2, 2, 20, 33, 1, 700, 40, 24)]
WALKS = SIZES[:4] + SIZES[8:]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_strides_and_alignments(size, dtype):
    x = inputs(*size, dtype)
    want = ref.prefix_attention(*x)
    received = ref.received(*x[:2])
    y = [t.to(DEV) for t in x]
    first = attend(y)
    check(first, want)
    for view in (odd, rows_first, spread):
        got = attend([view(t) for t in y])
        check(got, want)
        assert ref.over(hha.received_attention(view(y[0]), view(y[1])), received) <= 1.0
    # one side alone off its units
    got = attend([y[0], odd(y[1]), y[2], y[3], odd(y[4])])
    check(got, want)
    again = attend(y)
    assert torch.equal(again["out"], first["out"]) and torch.equal(again["lse"], first["lse"])  # sums in a fixed order


@pytest.mark.parametrize("dtype", DTYPES)
def test_broadcast_inputs(dtype):
    """One query, one prefix head and one row for all, by strides of zero."""
    b, h, hk, n, m, p, d = 4, 4, 2, 3, 20, 90, 64
    q, k, v, pk, pv = inputs(1, 1, 1, 1, 1, 1, 1, d, d, dtype)
    x = [q.expand(b, h, n, d), k.expand(b, hk, m, d), v.expand(b, hk, m, d), pk.expand(1, hk, p, d), pv.expand(1, hk, p, d)]
    check(attend([t.to(DEV).expand(s.shape) for t, s in zip((q, k, v, pk, pv), x)]), ref.prefix_attention(*x))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_what_is_hidden_does_not_count(size, dtype):
    """Infinities and NaN behind lengths, behind prefix_lengths and in rows behind counts; later tokens hide from earlier
    rows."""
    b, h, hk, n, m, sets, p, d, dv = size
    x = inputs(*size, dtype, seed=1)
    lengths = [max(1, m - 3 * i) for i in range(b)]
    counts = [min(y, max(1, n - i)) for i, y in enumerate(lengths)]
    plens = [p - 5] * sets
    kw = dict(lengths=lengths, counts=counts, prefix_lengths=plens)
    want = ref.prefix_attention(*x, **kw)
    received = ref.received(*x[:2], lengths=lengths, counts=counts)
    y = [t.clone() for t in x]
    for i in range(b):
        y[0][i, :, counts[i]:] = math.nan
        y[1][i, :, lengths[i]:] = math.inf
        y[2][i, :, lengths[i]:] = math.nan
    y[3][:, :, p - 5:] = math.nan
    y[4][:, :, p - 5:] = math.inf
    kw = {name: ints(t) for name, t in kw.items()}
    y = [t.to(DEV) for t in y]
    check(attend(y, **kw), want)
    assert ref.over(hha.received_attention(y[0], y[1], lengths=kw["lengths"], counts=kw["counts"]), received) <= 1.0
    if n < 3:
        return
    # the last token's value and key: only the last row sees them
    z = [t.clone() for t in x]
    z[2][:, :, m - 1, 0] = math.inf
    got = attend([t.to(DEV) for t in z])
    full = ref.prefix_attention(*x)
    assert not torch.isfinite(got["out"][:, :, n - 1, 0]).any()
    check({"out": got["out"][:, :, :n - 1], "lse": got["lse"]}, {"out": tuple(t[:, :, :n - 1] for t in full["out"]), "lse": full["lse"]})
    z = [t.clone() for t in x]
    z[1][:, :, m - 1, 0] = math.nan
    got = attend([t.to(DEV) for t in z])
    assert got["out"][:, :, n - 1].isnan().all() and got["lse"][:, :, n - 1].isnan().all()
    cut = {name: tuple(t[:, :, :n - 1] for t in full[name]) for name in full}
    check({name: got[name][:, :, :n - 1] for name in got}, cut)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", WALKS)
def test_rows_of_one_key_and_lowest_values(size, dtype):
    """Keys that hide by the type's lowest value, rows whose logits are all -inf (NaN, as a softmax of them), and keys
    of -inf beside others (weights of 0)."""
    b, h, hk, n, m, sets, p, d, dv = size
    q, k, v, pk, pv = inputs(*size, dtype, seed=2)
    q = torch.zeros_like(q)
    q[..., 0] = 1.0  # logits are the keys' first column
    low = torch.finfo(dtype).min
    k, pk = torch.zeros_like(k), torch.zeros_like(pk)
    k[..., 0], pk[..., 0] = low, low
    pk[..., 7, 0] = 2.0  # the only key that counts
    got = attend([t.to(DEV) for t in (q, k, v, pk, pv)], scale=1.0)
    want = pv[:, :, 7].double()[torch.arange(b) * sets // b].repeat_interleave(h // hk, 1)[:, :, None].expand(b, h, n, dv)
    assert ref.over(got["out"], (want, 2.0 ** -7 * want.abs() if dtype == torch.bfloat16 else 2.0 ** -10 * want.abs())) <= 1.0
    k[..., 0], pk[..., 0] = -math.inf, -math.inf
    pk[..., 7, 0] = 2.0
    got = attend([t.to(DEV) for t in (q, k, v, pk, pv)], scale=1.0)
    assert ref.over(got["out"], (want, 2.0 ** -7 * want.abs() if dtype == torch.bfloat16 else 2.0 ** -10 * want.abs())) <= 1.0
    pk[..., 7, 0] = -math.inf
    got = attend([t.to(DEV) for t in (q, k, v, pk, pv)], scale=1.0)
    assert got["out"].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_logits(dtype):
    x = inputs(4, 8, 2, 5, 60, 1, 300, 64, 64, dtype, seed=3)
    x[0] *= 40
    check(attend([t.to(DEV) for t in x]), ref.prefix_attention(*x))


def test_statistics_that_are_not_finite():
    """A row whose statistic is infinite or NaN makes the weights NaN of the tokens that it sees, and of no others."""
    b, h, n, m, d = 1, 2, 300, 300, 64
    q, k = (t.to(DEV) for t in make(5, torch.bfloat16, (b, h, n, d), (b, h, m, d)))
    lse = torch.full((b, h, n), 20.0, device=DEV)
    lse[0, 1, 200] = math.inf
    got = hha.received_attention(q, k, lse=lse)
    assert got[0, 1, :201].isnan().all() and torch.isfinite(got[0, 1, 201:]).all() and torch.isfinite(got[0, 0]).all()
    got = hha.received_attention(q[:, :, 200:210], k[:, :, :210], lse=lse[:, :, 200:210].contiguous())  # few rows
    assert got[0, 1, :201].isnan().all() and torch.isfinite(got[0, 1, 201:]).all() and torch.isfinite(got[0, 0]).all()


def test_nothing_to_do():
    for b, n, m, p in ((0, 1, 4, 3), (2, 0, 4, 3)):
        out, lse = spa.shared_prefix_attention(*(t.to(DEV) for t in inputs(b, 4, 2, n, m, 1, p, 16, 8, torch.float32)), with_lse=True)
        assert out.shape == (b, 4, n, 8) and lse.shape == (b, 4, n)
    assert hha.received_attention(torch.zeros(2, 4, 0, 16, device=DEV), torch.zeros(2, 2, 5, 16, device=DEV)).eq(0).all()
    assert hha.received_attention(torch.zeros(0, 4, 1, 16, device=DEV), torch.zeros(0, 2, 5, 16, device=DEV)).shape == (0, 2, 5)


def cache_of(dtype=torch.bfloat16, streams=2, heads=4, kv=2, kept=12, recent=5, d=32, dv=24, n=40, seed=0, **kw):
    c = hha.HeavyHitterStreamingAttention(d, dv, streams=streams, heads=heads, kv_heads=kv, kept=kept, recent=recent, dtype=dtype, **kw)
    k, v = make(seed, dtype, (streams, kv, n, d), (streams, kv, n, dv))
    w = torch.rand(streams, kv, n, generator=torch.Generator().manual_seed(seed))
    c.start(k.to(DEV), v.to(DEV), w.to(DEV))
    return c


def token(c, seed):
    return [t.to(DEV) for t in make(seed, c.dtype, (c.streams, c.heads, c.dim), (c.streams, c.kv_heads, c.dim),
                                    (c.streams, c.kv_heads, c.value_dim))]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a.items(), b.items())) and torch.equal(a.lengths, b.lengths)


@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("kw", [dict(), dict(kept=3000, recent=9, n=3100), dict(heads=40, kv=1, streams=1)])
def test_captured_steps(kw, prefix):
    """Replays of captured steps, updates and queries advance the state like calls, with eager work and another graph
    of another object between them."""
    a, b, other = cache_of(**kw), cache_of(**kw), cache_of(seed=9, **kw)
    pk, pv = (t.to(DEV) for t in make(2, a.dtype, (a.kv_heads, 150, 32), (a.kv_heads, 150, 24)))
    more = dict(prefix=(pk, pv)) if prefix else {}
    q, k, v = token(a, 1)

    def work(c):
        out = c.step(q, k, v, **more)
        c.update(k, v)
        return out, c.query(q, **more)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work(cache_of(**kw))
    torch.cuda.current_stream().wait_stream(stream)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        got = work(a)
    with torch.cuda.graph(graphs[1]):
        work(other)
    for t in range(6):
        for x, y in zip((q, k, v), token(a, 100 + t)):
            x.copy_(y)
        graphs[0].replay()
        graphs[1].replay()
        torch.zeros(1 << 20, device=DEV).add_(1.0).sum().item()
        want = work(b)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), t
        assert same(a, b), t


def test_captured_prompts():
    """Prefill and start in a graph: every replay begins the streams anew."""
    a, b = cache_of(), cache_of()
    q, k, v = (t.to(DEV) for t in make(3, a.dtype, (2, 4, 30, 32), (2, 2, 30, 32), (2, 2, 30, 24)))
    pk, pv = (t.to(DEV) for t in make(2, a.dtype, (2, 50, 32), (2, 50, 24)))
    counts = ints([30, 17])
    cache_of().prefill(q, k, v, counts=counts, prefix=(pk, pv))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = a.prefill(q, k, v, counts=counts, prefix=(pk, pv))
    for t in range(4):
        q.copy_(q.roll(1, 2))
        counts.copy_(ints([30 - t, 17 + t]))
        graph.replay()
        want = b.prefill(q, k, v, counts=counts, prefix=(pk, pv))
        torch.cuda.synchronize()
        assert torch.equal(got, want) and same(a, b), t
        a.step(*token(a, t))
        b.step(*token(b, t))
        assert same(a, b), t


def test_other_streams_and_threads():
    """Calls run on the current stream, and objects of two threads do not share anything."""
    x = [t.to(DEV) for t in inputs(16, 16, 4, 1, 300, 1, 900, 64, 64, torch.bfloat16)]
    want = spa.shared_prefix_attention(*x)
    caches = [cache_of(kept=2000, n=2100), cache_of(kept=2000, n=2100)]
    single = cache_of(kept=2000, n=2100)
    expected = [single.step(*token(single, t)) for t in range(20)]
    torch.cuda.synchronize()
    errors = []

    def run(c):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for t in range(20):
                    out = c.step(*token(c, t))
                    y = spa.shared_prefix_attention(*x)
                    stream.synchronize()
                    assert torch.equal(out, expected[t]) and torch.equal(y, want)
        except BaseException as e:  # noqa: B036
            errors.append(e)

    threads = [threading.Thread(target=run, args=(c,)) for c in caches]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_saved_states():
    a = cache_of()
    for t in range(9):
        a.step(*token(a, t))
    state = a.state_dict()
    b = hha.HeavyHitterStreamingAttention(32, 24, streams=2, heads=4, kv_heads=2, kept=12, recent=5, dtype=torch.bfloat16)
    b.load_state_dict(state)
    for t in range(30):
        x = token(a, 50 + t)
        assert torch.equal(a.step(*x), b.step(*x))
    assert same(a, b) and a.state_size_bytes() == b.state_size_bytes() > 0
    other = hha.HeavyHitterStreamingAttention(32, 24, streams=2, heads=4, kv_heads=2, kept=13, recent=5, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="do not match"):
        other.load_state_dict(state)
    with pytest.raises(ValueError, match="do not match"):
        b.load_state_dict({**state, "weights": state["weights"][:1]})
    with pytest.raises(ValueError, match="must not be negative"):
        b.load_state_dict({**state, "counts": state["counts"] - 1000})
    assert same(a, b)


def test_a_token_that_is_not_finite_is_forgotten():
    c, clean = cache_of(kept=6, recent=3), cache_of(kept=6, recent=3)
    for t in range(30):
        q, k, v = token(c, t)
        clean.step(q, k, v)
        if t == 4:
            k = k.clone()
            k[0, 0, 3] = math.nan
        out = c.step(q, k, v)
        assert torch.isfinite(c.weights).all()
        assert torch.isfinite(out[1]).all() and torch.isfinite(out[0, 2:]).all()
        if 4 <= t < 7:
            assert out[0, :2].isnan().all()
    assert torch.isfinite(out).all()  # it had no weight when it passed out of the last tokens
    assert torch.equal(c.positions[1], clean.positions[1]) and torch.equal(c.weights[1], clean.weights[1])


def test_infinite_weights_keep_tokens():
    c = hha.HeavyHitterStreamingAttention(16, 16, heads=2, kv_heads=1, kept=4, recent=2)
    k, v = (t.to(DEV) for t in make(1, torch.float32, (1, 1, 10, 16), (1, 1, 10, 16)))
    w = torch.ones(1, 1, 10, device=DEV)
    w[..., [0, 5]] = math.inf
    c.start(k, v, w)
    for t in range(25):
        c.step(*token(c, t))
    assert {0, 5} <= set(c.positions[0, 0].tolist())


@pytest.mark.parametrize("dtype", DTYPES)
def test_inputs_of_steps(dtype):
    """Views, other types and rows off their units give what dense ones give."""
    a, b = cache_of(dtype, d=33, dv=40), cache_of(dtype, d=33, dv=40)
    for t in range(8):
        q, k, v = token(a, t)
        want = a.step(q, k, v)
        if t % 2:
            got = b.step(odd(q), odd(k), odd(v))
        else:
            got = b.step(q.double() if t % 4 else q.cpu(), rows_first(k[None])[0], v.float())
        assert torch.equal(got, want) and same(a, b)
    with pytest.raises(ValueError, match=r"query must be \[2, 4, 33\]"):
        a.step(q[:1], k, v)
    with pytest.raises(ValueError, match=r"key must be"):
        a.step(q, k[..., :32], v)
    assert same(a, b)  # a refused call leaves the state


def test_refusals_of_prefixes():
    c = cache_of()
    q, k, v = token(c, 0)
    good = [t.to(DEV) for t in make(1, c.dtype, (2, 9, 32), (2, 9, 24))]
    before = c.state_dict()
    for bad, message in (((good[0].float(), good[1]), "object's dtype"), ((good[0].cpu(), good[1]), "on its device"),
                         ((good[0][:, :, :31], good[1]), "must be"), ((good[0][:1], good[1][:1]), "must be"),
                         ((good[0].expand(3, 2, 9, 32), good[1].expand(3, 2, 9, 24)), "multiple of the 3 prefixes")):
        with pytest.raises(ValueError, match=message):
            c.step(q, k, v, prefix=bad)
    with pytest.raises(ValueError, match="without a prefix"):
        c.step(q, k, v, prefix_lengths=ints([3]))
    with pytest.raises(ValueError, match="prefix_lengths must be"):
        c.step(q, k, v, prefix=good, prefix_lengths=ints([3, 3]))
    small = hha.HeavyHitterStreamingAttention(4, 16, kept=4, recent=2, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="at least 16 bytes"):
        small.step(*token(small, 0), prefix=(torch.zeros(1, 3, 4, device=DEV, dtype=torch.bfloat16),
                                             torch.zeros(1, 3, 16, device=DEV, dtype=torch.bfloat16)))
    with pytest.raises(ValueError, match="weights must be a float32"):
        c.start(k[:, :, None], v[:, :, None], torch.zeros(2, 2, 2, device=DEV))
    with pytest.raises(ValueError, match="one device"):
        c.start(k[:, :, None], v[:, :, None], torch.zeros(2, 2, 1))
    with pytest.raises(ValueError, match="no stream 2"):
        c.reset([0, 2])
    after = c.state_dict()
    assert all(torch.equal(before[name], after[name]) for name in before if name != "attention")
    c.step(q, k, v, prefix=[t[None].expand(2, 2, 9, t.shape[-1]) for t in good], prefix_lengths=ints([0, 9]))


@pytest.mark.parametrize("heads,kv", [(512, 1), (272, 1), (48, 3)])
def test_many_heads_of_a_key_head(heads, kv):
    c = hha.HeavyHitterStreamingAttention(16, 16, heads=heads, kv_heads=kv, kept=40, recent=7, dtype=torch.bfloat16)
    want = ref.Cache(1, kv, 40, 7)
    for t in range(4):
        q, k, v = make(t, torch.bfloat16, (1, heads, 16), (1, kv, 16), (1, kv, 16))
        want.adopt(c.weights.cpu())
        got = c.step(q.to(DEV), k.to(DEV), v.to(DEV))
        want.update(k, v)
        out = want.query(q, 0.25)
        weights, bound, positions = want.state()
        assert ref.over(got, out) <= 1.0 and ref.over(c.weights, (weights, bound)) <= 1.0
        assert torch.equal(c.positions.cpu(), positions)


def test_offsets_past_32_bits():
    """A prefix and own tokens of more than 4 GiB: one key at either end counts, and what tokens receive at the far end."""
    p = (1 << 24) + 777
    pk = torch.zeros(1, p, 128, device=DEV, dtype=torch.bfloat16)
    pv = torch.zeros(1, p, 128, device=DEV, dtype=torch.bfloat16)
    q = torch.zeros(2, 1, 1, 128, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 8.0
    k = torch.zeros(2, 1, 3, 128, device=DEV, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    pk[0, p - 1, 0] = 50.0
    pv[0, p - 1] = 3.0
    out = spa.shared_prefix_attention(q, k, v, pk, pv)
    assert out.eq(3.0).all()
    own_out = spa.shared_prefix_attention(q[:1], pk[None], pv[None], pk[:, :0], pv[:, :0])
    assert own_out.eq(3.0).all()
    got = hha.received_attention(q[:1], pk[None])
    assert got[0, 0, p - 1].item() == pytest.approx(1.0, abs=1e-5) and got[0, 0, :-1].sum().item() < 1e-3


def test_large_caches():
    """A cache of more than 4 GiB a tensor: the last stream's tokens are its own."""
    c = hha.HeavyHitterStreamingAttention(128, 128, streams=3, heads=1, kept=(1 << 23) - 600, recent=511, dtype=torch.bfloat16)
    k, v = (t.to(DEV) for t in make(1, torch.bfloat16, (3, 1, 700, 128), (3, 1, 700, 128)))
    w = torch.rand(3, 1, 700, device=DEV)
    c.start(k, v, w)
    q = torch.zeros(3, 1, 128, device=DEV, dtype=torch.bfloat16)
    for t in range(3):
        got = c.step(q, k[:, :, t], v[:, :, t])  # equal weights
    mean = torch.cat([v[:, 0], v[:, 0, :3]], 1).double().mean(1)
    assert ref.over(got[:, 0], (mean.cpu(), 2.0 ** -8 * (mean.abs() + v.double().abs().mean()).cpu())) <= 1.0
    assert c.positions[2, 0, :512].ge(0).sum().item() == 511 and c.positions[2, 0].ge(0).sum().item() == 703


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [dict(), dict(kept=2000, recent=9, n=2100), dict(heads=40, kv=1, streams=2)])
def test_prefixes_of_nothing(kw, dtype):
    """A prefix without rows, or with none that count, is none: outputs within a rounding, and the same tokens held."""
    a, b, c = (cache_of(dtype=dtype, **kw) for _ in range(3))
    none = tuple(t.to(DEV) for t in make(3, dtype, (a.kv_heads, 0, 32), (a.kv_heads, 0, 24)))
    some = tuple(t.to(DEV) for t in make(4, dtype, (2, a.kv_heads, 77, 32), (2, a.kv_heads, 77, 24)))
    some[1][:] = math.nan
    eps = 2 * torch.finfo(dtype).eps + 64 * torch.finfo(torch.float32).eps  # two roundings of an output, fp32 sums
    for i in range(3):
        q, k, v = token(a, 20 + i)
        want = a.step(q, k, v)
        assert torch.equal(b.step(q, k, v, prefix=none), want)
        got = c.step(q, k, v, prefix=some, prefix_lengths=ints([0, -3]))
        assert ((got.double() - want.double()).abs() <= eps * v.abs().max().clamp(min=4.0)).all()
    assert same(a, b) and torch.equal(a.positions, c.positions)


@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_of_empty_caches_behind_a_prefix(dtype):
    """Before a token has come a query sees the prefix alone; without one its output is zero."""
    c = hha.HeavyHitterStreamingAttention(32, 24, streams=4, heads=8, kv_heads=2, kept=12, recent=5, dtype=dtype)
    q = token(c, 1)[0]
    pk, pv = make(2, dtype, (2, 2, 600, 32), (2, 2, 600, 24))
    got = c.query(q, prefix=(pk.to(DEV), pv.to(DEV)), prefix_lengths=ints([600, 3]))
    # the prefix's rows as own tokens of each stream, whose newest row is the query's
    k, v = (t.repeat_interleave(2, 0) for t in (pk, pv))
    want = ref.prefix_attention(q.cpu()[:, :, None], k, v, pk[:1, :, :0], pv[:1, :, :0], lengths=[600, 600, 3, 3])
    check({"out": got[:, :, None]}, {"out": want["out"]})
    assert c.query(q).eq(0).all() and c.weights.eq(0).all() and c.lengths.eq(0).all()


@pytest.mark.parametrize("streams,kv,kept,first", [(1, 1, 24, 0), (1, 1, 24, 9), (2, 2, 24, 0), (1, 1, 9000, 0)])
def test_starts_from_the_state_s_own_weights(streams, kv, kept, first):
    """`weights` is a view of what start writes."""
    slots = kept + 8
    c = cache_of(streams=streams, heads=kv, kv=kv, kept=kept, recent=7, n=slots + 5)
    own = c.weights[..., first:]
    k, v = (t.to(DEV) for t in make(6, c.dtype, (streams, kv, slots - first, 32), (streams, kv, slots - first, 24)))
    want = cache_of(streams=streams, heads=kv, kv=kv, kept=kept, recent=7, n=slots + 5)
    want.start(k, v, own.clone())
    c.start(k, v, own)
    assert same(c, want)
