"""Windowed attention with sinks on the GPU (sink_window_attention) against its float64 statement, element by element
within the bounds that the statement derives from the roundings."""

import math

import pytest
import torch

import sink_window_attention as swa
import window_reference as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(b, h, hk, n, d, dv, dtype, seed=0):
    g = torch.Generator().manual_seed(1000 * seed + 7 * n + d)
    return [torch.randn(*s, generator=g).to(dtype) for s in ((b, h, n, d), (b, hk, n, d), (b, hk, n, dv), (b, h, n, dv))]


def run(q, k, v, go, **kw):
    x = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    if kw.get("lengths") is not None:
        kw["lengths"] = torch.tensor(kw["lengths"], dtype=torch.int32, device=DEV)
    out = swa.sink_window_causal_attention(*x, **kw)
    grads = torch.autograd.grad(out, x, go.to(DEV))
    torch.cuda.synchronize()
    return dict(zip(("out", "dq", "dk", "dv"), (out, *grads)))


def check(got, want):
    worst = {name: ref.over(got[name], want[name]) for name in want}
    assert all(x <= 1.0 for x in worst.values()), worst


CASES = [  # b h hk n d dv window sinks lengths
    (1, 1, 1, 1, 1, 1, 1, 0, None),
    (1, 1, 1, 2, 8, 8, 1, 1, None),
    (1, 2, 1, 33, 16, 24, 5, 2, None),
    (1, 1, 1, 64, 32, 32, 64, 0, None),
    (2, 4, 2, 129, 64, 64, 32, 4, None),
    (1, 2, 2, 257, 64, 64, 1000, 4, None),
    (1, 1, 1, 300, 40, 33, 70, 300, None),
    (2, 2, 1, 200, 93, 77, 31, 5, [200, 77]),
    (3, 3, 1, 150, 128, 128, 64, 3, [0, 1, 149]),
    (1, 4, 1, 500, 128, 128, 100, 150, None),
    (1, 1, 1, 700, 96, 80, 128, 33, [650]),
    (1, 1, 1, 1030, 32, 64, 200, 4, None),
    (2, 1, 1, 260, 5, 3, 17, 129, [260, 131]),
    (1, 2, 2, 1400, 64, 64, 100, 4, None),
    (2, 8, 2, 700, 33, 40, 64, 70, [700, 333]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,n,d,dv,window,sinks,lengths", CASES)
def test_outputs_and_gradients(b, h, hk, n, d, dv, window, sinks, lengths, dtype):
    q, k, v, go = make(b, h, hk, n, d, dv, dtype)
    kw = dict(window=window, sinks=sinks, lengths=lengths)
    check(run(q, k, v, go, **kw), ref.window_attention(q, k, v, grad=go, **kw))


WIDE = [  # many heads: tiles of 128 rows
    (4, 32, 32, 400, 64, 64, 100, 4, None),
    (2, 32, 16, 1030, 32, 32, 1100, 0, None),
    (8, 24, 8, 513, 40, 72, 33, 140, [513, 0, 1, 512, 128, 129, 300, 511]),
    (4, 32, 32, 300, 128, 100, 90, 5, [300, 131, 299, 64]),
    (4, 64, 32, 257, 96, 96, 64, 3, None),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,n,d,dv,window,sinks,lengths", WIDE)
def test_many_heads(b, h, hk, n, d, dv, window, sinks, lengths, dtype):
    q, k, v, go = make(b, h, hk, n, d, dv, dtype)
    kw = dict(window=window, sinks=sinks, lengths=lengths)
    check(run(q, k, v, go, **kw), ref.window_attention(q, k, v, grad=go, **kw))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_heads_hide_infinities(dtype):
    """test_hidden_infinities_stay_hidden on tiles of 128 rows: one key's value, one row's gradient."""
    b, h, n, window, sinks = 8, 32, 300, 40, 3
    q, k, v, go = make(b, h, h, n, 32, 32, dtype, seed=5)
    kw = dict(window=window, sinks=sinks)
    want = ref.window_attention(q, k, v, grad=go, **kw)
    see = ref.visible(n, n, window, sinks)
    v2, g2 = v.clone(), go.clone()
    v2[3, 7, 100, 5] = math.inf
    g2[4, 9, 200, 2] = math.nan
    got = {name: x.cpu() for name, x in run(q, k, v2, g2, **kw).items()}
    rows, keys = see[:, 100], (see & see[:, 100][:, None]).any(0)
    assert not torch.isfinite(got["out"][3, 7, 100, 5]) and not torch.isfinite(got["dv"][4, 9, 190, 2])
    for name in ("out", "dq"):
        assert ref.over(got[name][3, 7][~rows], tuple(t[3, 7][~rows] for t in want[name])) <= 1.0
        other = torch.arange(n) != 200
        assert ref.over(got[name][4, 9][other], tuple(t[4, 9][other] for t in want[name])) <= 1.0
    for name in ("dk", "dv"):
        assert ref.over(got[name][3, 7][~keys], tuple(t[3, 7][~keys] for t in want[name])) <= 1.0
        assert ref.over(got[name][4, 9][~see[200]], tuple(t[4, 9][~see[200]] for t in want[name])) <= 1.0
    for name in want:
        assert ref.over(got[name][5], tuple(t[5] for t in want[name])) <= 1.0


@pytest.mark.parametrize("scale", [-0.3, 0.0, 4.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(dtype, scale):
    q, k, v, go = make(1, 2, 1, 140, 32, 32, dtype, seed=1)
    kw = dict(window=40, sinks=3, scale=scale)
    check(run(q, k, v, go, **kw), ref.window_attention(q, k, v, grad=go, **kw))


@pytest.mark.parametrize("dtype", DTYPES)
def test_full_window_is_causal_attention(dtype):
    q, k, v, go = make(1, 2, 2, 190, 64, 64, dtype, seed=2)
    out = swa.sink_window_causal_attention(q.to(DEV), k.to(DEV), v.to(DEV), window=190, sinks=0)
    see = torch.ones(190, 190, dtype=torch.bool).tril()
    x = (q.double() @ k.double().transpose(-1, -2)) / 8
    want = x.masked_fill(~see, -math.inf).softmax(-1) @ v.double()
    bound = ref.window_attention(q, k, v, window=190, sinks=0)["out"][1]
    assert ref.over(out, (want, bound)) <= 1.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_single_sequences(dtype):
    q, k, v, go = (x.to(DEV) for x in make(2, 4, 2, 131, 48, 40, dtype, seed=3))
    kw = dict(window=50, sinks=4)
    out = swa.sink_window_causal_attention(q, k, v, **kw)
    want = swa.sink_window_backward(go, q, k, v, *swa.sink_window_forward(q, k, v, **kw), **kw)

    def rows_first(x):  # [B, N, H, D] in memory
        return x.transpose(1, 2).contiguous().transpose(1, 2)

    def offset(x):  # rows that start off 16 bytes
        y = torch.empty(*x.shape[:3], x.shape[3] + 3, device=DEV, dtype=dtype)
        y[..., 1:-2] = x
        return y[..., 1:-2]

    def backwards_last(x):  # last dimension not contiguous: taken as a copy
        return x.transpose(2, 3).contiguous().transpose(2, 3)

    for f in (rows_first, offset, backwards_last):
        x = [f(t) for t in (q, k, v)]
        o, lse = swa.sink_window_forward(*x, **kw)
        assert torch.equal(o, out)
        for got, w in zip(swa.sink_window_backward(f(go), *x, f(o), lse, **kw), want):
            assert torch.equal(got, w)
    one = swa.sink_window_causal_attention(q[0, 1], k[0, 0], v[0, 0], **kw)
    assert torch.equal(one, out[0, 1])


def test_expanded_gradient_and_shared_inputs():
    # the gradient of a sum has stride 0; q, k and v may be one tensor
    x = torch.randn(1, 2, 90, 32, device=DEV, requires_grad=True)
    out = swa.sink_window_causal_attention(x, x, x, window=20, sinks=2)
    out.sum().backward()
    go = torch.ones(1, 2, 90, 32)
    y = x.detach().cpu()
    want = ref.window_attention(y, y, y, window=20, sinks=2, grad=go)
    total = tuple(sum(want[n][i] for n in ("dq", "dk", "dv")) for i in (0, 1))
    assert ref.over(x.grad, total) <= 1.0


def test_gradient_against_differences():
    q, k, v, go = (x.to(DEV) for x in make(1, 4, 2, 80, 24, 24, torch.float32, seed=4))
    kw = dict(window=30, sinks=3)
    got = run(q.cpu(), k.cpu(), v.cpu(), go.cpu(), **kw)
    g = torch.Generator().manual_seed(9)
    h = 2.0 ** -6
    for i, name in enumerate(("dq", "dk", "dv")):
        x = [q, k, v]
        step = torch.randn(x[i].shape, generator=g).to(DEV)

        def at(e):
            y = list(x)
            y[i] = x[i] + e * step
            return (swa.sink_window_causal_attention(*y, **kw).double() * go).sum().item()

        slope = (8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))) / (12 * h)
        want = (got[name].double() * step).sum().item()
        # values of about sqrt(80 4 24) = 88, each out element off by a few 1e-7: (9 / 6) 88 5e-7 / h = 4e-3; the
        # formula's remainder, h^4 f^(5) / 30, is below 1e-5 of f'
        assert abs(slope - want) <= 5e-3 + 1e-4 * abs(want), (name, slope, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_hidden_infinities_stay_hidden(dtype, value):
    """A key, value, query or gradient that is not finite reaches the results of the pairs it is part of alone."""
    n, window, sinks = 300, 40, 3
    q, k, v, go = make(1, 2, 1, n, 32, 32, dtype, seed=5)
    kw = dict(window=window, sinks=sinks)
    # what the free pairs' results are without the value; a row taken again over its visible pairs sums in another
    # order than a tile does, so the statement's bounds hold and not the bits
    want = ref.window_attention(q, k, v, grad=go, **kw)
    see = ref.visible(n, n, window, sinks)
    at = 100
    for which in range(4):
        x = [t.clone() for t in (q, k, v, go)]
        x[which][0, 0, at, 5] = value
        got = run(*x, **kw)
        if which in (1, 2):  # rows that see key `at`
            rows = see[:, at]
            heads = [0, 1]
        else:
            rows = torch.zeros(n, dtype=torch.bool)
            rows[at] = True
            heads = [0]
        keys = (see & rows[:, None]).any(0)
        for name in ("out", "dq"):
            for hi in range(2):
                free = torch.ones(n, dtype=torch.bool) if hi not in heads or (which, name) == (3, "out") else ~rows
                part = tuple(t[0, hi][free] for t in want[name])
                assert ref.over(got[name][0, hi].cpu()[free], part) <= 1.0, (which, name)
        for name in ("dk", "dv"):
            part = tuple(t[0, 0][~keys] for t in want[name])
            assert ref.over(got[name][0, 0].cpu()[~keys], part) <= 1.0, (which, name)
        # and where it is seen it is not lost
        if which == 2:
            assert not torch.isfinite(got["out"][0, 0, at, 5])
        if which == 3:
            assert not torch.isfinite(got["dv"][0, 0, at, 5])


@pytest.mark.parametrize("dtype", DTYPES)
def test_padding_is_never_read(dtype):
    q, k, v, go = make(2, 2, 1, 200, 64, 48, dtype, seed=6)
    kw = dict(window=64, sinks=4, lengths=[70, 131])
    clean = run(q, k, v, go, **kw)
    for x in (q, k, v, go):
        for i, length in enumerate(kw["lengths"]):
            x[i, :, length:] = math.nan
    got = run(q, k, v, go, **kw)
    for name in clean:
        assert torch.equal(got[name], clean[name]), name
        for i, length in enumerate(kw["lengths"]):
            assert not got[name][i, :, length:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_all_logits_at_the_lowest_value(dtype):
    """Logits of -inf everywhere: softmax is NaN there, and only there."""
    q, k, v, go = make(1, 1, 1, 100, 16, 16, dtype, seed=7)
    q[0, 0, 50] = 0
    q[0, 0, 50, 0] = 1
    k[0, 0, :, 0] = -math.inf
    q[0, 0, :50, 0] = 0.5
    q[0, 0, 51:, 0] = 0.5
    out = swa.sink_window_causal_attention(q.to(DEV), k.to(DEV), v.to(DEV), window=30, sinks=0)
    assert torch.isnan(out).all()


def test_equal_inputs_give_equal_bits():
    q, k, v, go = make(2, 4, 1, 600, 64, 64, torch.bfloat16, seed=8)
    kw = dict(window=100, sinks=20)
    a, b = run(q, k, v, go, **kw), run(q, k, v, go, **kw)
    for name in a:
        assert torch.equal(a[name], b[name])


def test_other_stream_and_captured_graph():
    q, k, v, go = (x.to(DEV) for x in make(1, 2, 1, 333, 64, 64, torch.bfloat16, seed=9))
    kw = dict(window=100, sinks=4)
    out, lse = swa.sink_window_forward(q, k, v, **kw)
    want = swa.sink_window_backward(go, q, k, v, out, lse, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, l2 = swa.sink_window_forward(q, k, v, **kw)
        g2 = swa.sink_window_backward(go, q, k, v, o2, l2, **kw)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip((o2, l2, *g2), (out, lse, *want)):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o3, l3 = swa.sink_window_forward(q, k, v, **kw)
        g3 = swa.sink_window_backward(go, q, k, v, o3, l3, **kw)
    for seed in (1, 2, 3):
        for x, y in zip((q, k, v, go), make(1, 2, 1, 333, 64, 64, torch.bfloat16, seed=20 + seed)):
            x.copy_(y)
        graph.replay()
        out, lse = swa.sink_window_forward(q, k, v, **kw)
        want = swa.sink_window_backward(go, q, k, v, out, lse, **kw)
        torch.cuda.synchronize()
        for a, b in zip((o3, l3, *g3), (out, lse, *want)):
            assert torch.equal(a, b)


def test_empty_batches():
    for shape in ((0, 2, 5, 8), (2, 2, 0, 8)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        out = swa.sink_window_causal_attention(x, x, x, window=4)
        assert out.shape == shape
        out.sum().backward()
        assert x.grad.shape == shape


def test_row_strides_of_single_rows():
    """The stride of a dimension of one element is never walked, however far it reaches."""
    q, k, v, go = make(2, 2, 1, 1, 32, 32, torch.bfloat16)
    want = run(q, k, v, go, window=3, sinks=0)

    def far(x):
        x = x.to(DEV)
        return x.as_strided(x.shape, (x.stride(0), x.stride(1), 1 << 25, 1))

    out, lse = swa.sink_window_forward(far(q), far(k), far(v), window=3, sinks=0)
    got = (out, *swa.sink_window_backward(far(go), far(q), far(k), far(v), out, lse, window=3, sinks=0))
    for x, y in zip(got, want.values()):
        assert torch.equal(x.cpu(), y.cpu())


FULL = [  # many heads whose widths fill their padded ones
    (4, 64, 32, 300, 128, 128, 70, 5, [300, 131, 1, 64]),
    (2, 64, 64, 520, 128, 128, 600, 0, None),
    (6, 32, 32, 257, 64, 64, 30, 140, [257, 129, 128, 65, 0, 200]),
    (2, 48, 48, 400, 64, 64, 399, 1, [400, 399]),
    (4, 64, 64, 129, 32, 32, 1, 0, None),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,n,d,dv,window,sinks,lengths", FULL)
def test_many_heads_of_full_width(b, h, hk, n, d, dv, window, sinks, lengths, dtype):
    q, k, v, go = make(b, h, hk, n, d, dv, dtype, seed=11)
    kw = dict(window=window, sinks=sinks, lengths=lengths)
    check(run(q, k, v, go, **kw), ref.window_attention(q, k, v, grad=go, **kw))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_many_heads_never_read_padding(dtype, d):
    q, k, v, go = make(4, 64, 32, 200, d, d, dtype, seed=12)
    kw = dict(window=64, sinks=4, lengths=[70, 131, 0, 199])
    clean = run(q, k, v, go, **kw)
    for x in (q, k, v, go):
        for i, length in enumerate(kw["lengths"]):
            x[i, :, length:] = math.nan
    got = run(q, k, v, go, **kw)
    for name in clean:
        assert torch.equal(got[name], clean[name]), name
        for i, length in enumerate(kw["lengths"]):
            assert not got[name][i, :, length:].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_heads_last_row_of_a_length(dtype):
    """A query and a gradient that are not finite in a sequence's last row reach what that row sees alone."""
    b, h, n, window, sinks, length = 4, 64, 200, 40, 3, 135
    q, k, v, go = make(b, h, h, n, 64, 64, dtype, seed=13)
    kw = dict(window=window, sinks=sinks, lengths=[length] * b)
    want = ref.window_attention(q, k, v, grad=go, **kw)
    see = ref.visible(n, n, window, sinks)[length - 1]
    q2, g2 = q.clone(), go.clone()
    q2[1, 5, length - 1, 7] = math.inf
    g2[2, 6, length - 1, 2] = math.nan
    got = {name: x.cpu() for name, x in run(q2, k, v, g2, **kw).items()}
    rows = torch.arange(n) != length - 1
    for i, head in ((1, 5), (2, 6)):
        for name in ("out", "dq"):
            assert ref.over(got[name][i, head][rows], tuple(t[i, head][rows] for t in want[name])) <= 1.0
        for name in ("dk", "dv"):
            assert ref.over(got[name][i, head][~see], tuple(t[i, head][~see] for t in want[name])) <= 1.0
    for name in want:
        assert ref.over(got[name][0], tuple(t[0] for t in want[name])) <= 1.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,h,hk,n,d,dv,window,lengths", [(1, 2, 1, 500, 64, 48, 16, None), (2, 3, 3, 200, 93, 33, 40, [200, 77]),
                                                          (4, 64, 64, 300, 64, 64, 20, None), (1, 1, 1, 70, 5, 3, 9, None)])
def test_rest_of_the_output(b, h, hk, n, d, dv, window, lengths, dtype):
    """What the output's rounding left is at most half a step of it; with it the gradients lose that rounding."""
    q, k, v, go = make(b, h, hk, n, d, dv, dtype, seed=14)
    want = ref.window_attention(q, k, v, grad=go, window=window, sinks=2, lengths=lengths)
    kw = dict(window=window, sinks=2, lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV))
    x = [t.to(DEV) for t in (q, k, v)]
    out, lse, rest = swa.sink_window_forward(*x, with_rest=True, **kw)
    assert torch.equal(out, swa.sink_window_forward(*x, **kw)[0])
    # half a step, or half the smallest step of the type
    smallest = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    half = (out.abs().double() * torch.finfo(dtype).eps / 2).clamp_min(smallest / 2)
    assert rest.dtype == dtype and torch.all(rest.double().abs() <= half * (1 + torch.finfo(dtype).eps) + smallest)
    with_rest = swa.sink_window_backward(go.to(DEV), *x, out, lse, rest=rest, **kw)
    without = swa.sink_window_backward(go.to(DEV), *x, out, lse, **kw)
    grads = dict(zip(("dq", "dk", "dv"), with_rest))
    check(grads, {name: want[name] for name in grads})
    for name, a, b_ in zip(("dq", "dk"), with_rest, without):
        error = [(t.cpu().double() - want[name][0]).norm() for t in (a, b_)]
        assert error[0] < error[1], (name, error)
    assert torch.equal(with_rest[2], without[2])
    # the differentiable call keeps it
    got = run(q, k, v, go, window=window, sinks=2, lengths=lengths)
    for name in grads:
        assert torch.equal(got[name], grads[name])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sinks", [1, 33, 64, 65])
@pytest.mark.parametrize("d,dv", [(64, 64), (128, 96)])
def test_sinks_of_many_heads_behind_short_windows(d, dv, sinks, dtype):
    """Rows behind the window of the sinks, in their own launch and in the keys' one; lengths that end before and in them."""
    q, k, v, go = make(3, 64, 64, 500, d, dv, dtype, seed=15)
    kw = dict(window=20, sinks=sinks, lengths=[500, 19, 83])
    check(run(q, k, v, go, **kw), ref.window_attention(q, k, v, grad=go, **kw))


def test_single_sequences_in_autograd():
    """[N,D] leaves of any strides, one of them used twice, under a gradient that is one expanded number."""
    base = torch.randn(48, 200, generator=torch.Generator().manual_seed(16)).to(DEV)
    x, v = base[:32].t().requires_grad_(), base[32:].t().requires_grad_()  # 200 rows, columns 200 elements apart
    out = swa.sink_window_causal_attention(x, x, v, window=30, sinks=2)
    dx, dv = torch.autograd.grad(out.sum(), (x, v))
    y, w = (t.detach().contiguous()[None, None] for t in (x, v))
    o, lse = swa.sink_window_forward(y, y, w, window=30, sinks=2)
    dq, dk, dw = swa.sink_window_backward(torch.ones_like(o), y, y, w, o, lse, window=30, sinks=2)
    assert out.shape == (200, 16) and dx.shape == x.shape and dv.shape == v.shape
    assert torch.equal(out, o[0, 0]) and torch.equal(dx, (dq + dk)[0, 0]) and torch.equal(dv, dw[0, 0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_passes_of_many_wide_heads(dtype):
    """The largest workgroups' passes captured as their first call of the process may be, replayed with eager work between."""
    q, k, v, go = (t.to(DEV) for t in make(2, 64, 32, 260, 128, 128, dtype, seed=17))
    kw = dict(window=33, sinks=3)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, lse, rest = swa.sink_window_forward(q, k, v, with_rest=True, **kw)
        grads = swa.sink_window_backward(go, q, k, v, out, lse, rest=rest, **kw)
    for i in range(4):
        for t in (q, k, v, go):
            t.copy_(t.roll(i + 1, 1) * 0.9)
        graph.replay()
        o, l, r = swa.sink_window_forward(q, k, v, with_rest=True, **kw)
        want = (o, l, *swa.sink_window_backward(go, q, k, v, o, l, rest=r, **kw))
        torch.cuda.synchronize()
        for x, y in zip((out, lse, *grads), want):
            assert torch.equal(x, y), i
