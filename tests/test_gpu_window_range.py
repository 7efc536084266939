"""Windowed attention and its cache where the element type's range counts: tiny weights of long rows, large gradients."""

import math

import pytest
import torch

import sink_window_attention as swa
import window_reference as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U16 = 2.0 ** -11  # half a step of fp16
LOGIT = 18.015625  # exp(-18.015625) = 2^-25.99: below half of fp16's smallest step


def one_large_weight(n, d, dv):
    """Keys of which the first has weight 1 and value 0, all others weight exp(-LOGIT) and value 64: row i's output is
    64 i e / (1 + i e)."""
    q, k, v = torch.zeros(1, 1, n, d), torch.zeros(1, 1, n, d), torch.full((1, 1, n, dv), 64.0)
    q[..., 0] = 1
    k[0, 0, 0, 0] = LOGIT
    v[0, 0, 0] = 0
    return [x.half().to(DEV) for x in (q, k, v)]


def wanted(i):
    e = math.exp(-LOGIT) * i.double()
    return 64 * e / (1 + e)


def bound(i, want):
    # the output's rounding (its smallest half step at least), 2^-36 of the largest weight a key, and the fp32 sums: n keys
    # and a logit of 18, twice 2^-24 of it in the weight
    return U16 * want + 2.0 ** -25 + 64 * i * 2.0 ** -36 + 2.0 ** -24 * (i + 64) * want


@pytest.mark.parametrize("heads,n", [(1, 20000), (40, 20000)])  # 32 and 128 rows a workgroup
def test_tiny_weights_of_long_fp16_rows(heads, n):
    q, k, v = (x.expand(1, heads, -1, -1) for x in one_large_weight(n, 16, 32))
    out = swa.sink_window_causal_attention(q, k, v, window=n, sinks=0, scale=1.0).cpu().double()
    i = torch.arange(n, dtype=torch.float64)[:, None]
    want = wanted(i)
    assert ((out - want).abs() <= bound(i, want)).all(), (out - want).abs().max()
    assert out[0, 0, -1, 0] > 0.01


@pytest.mark.parametrize("streams,heads", [(1, 1), (300, 2)])  # split over the slots, and not
def test_tiny_weights_of_long_fp16_caches(streams, heads):
    n = 20000
    q, k, v = one_large_weight(n, 16, 32)
    a = swa.SinkWindowStreamingAttention(16, 32, streams=streams, heads=heads, window=n, sinks=1, scale=1.0,
                                         dtype=torch.float16)
    a.extend(k.expand(streams, heads, -1, -1), v.expand(streams, heads, -1, -1))
    out = a.query(q[:, :, 0].expand(streams, heads, -1)).cpu().double()
    i = torch.tensor(n - 1.0, dtype=torch.float64)
    want = wanted(i)
    assert ((out - want).abs() <= bound(i, want)).all(), (out - want).abs().max()


def statement(q, k, v, go, *, window, sinks, lengths=None):
    """The float64 statement, and for the gradients of logits that the kernels carry lowered: an fp16 value below the
    normal range is off by up to 2^-36 of its row's (dq) or key's (dk) largest, that being 2^11 or more as it is carried."""
    want = ref.window_attention(q, k, v, grad=go, window=window, sinks=sinks, lengths=lengths)
    b, h, n, d = q.shape
    hk = k.shape[1]
    for bi in range(b):
        length = n if lengths is None else lengths[bi]
        see = ref.visible(n, length, window, sinks)
        top = torch.zeros(hk, n, dtype=torch.float64)
        size = torch.zeros(hk, n, d, dtype=torch.float64)
        for hi in range(h):
            qq, kk, vv, gg = (x.double() for x in (q[bi, hi], k[bi, hi * hk // h], v[bi, hi * hk // h], go[bi, hi]))
            p = (qq @ kk.T / math.sqrt(d)).masked_fill(~see, -math.inf).softmax(1).nan_to_num()
            ds = (p * (gg @ vv.T - (gg * (p @ vv)).sum(1, keepdim=True))).abs()
            want["dq"][1][bi, hi] += 2.0 ** -36 / math.sqrt(d) * ds.amax(1, keepdim=True) * (see.double() @ kk.abs())
            top[hi * hk // h] = torch.maximum(top[hi * hk // h], ds.amax(0))
            size[hi * hk // h] += see.double().T @ qq.abs()
        want["dk"][1][bi] += 2.0 ** -36 / math.sqrt(d) * top[..., None] * size
    return want


LARGE = [  # b h hk n d dv window sinks lengths: rows of 32 and of 128 a workgroup, sinks in the keys' launch and in their own
    (1, 2, 1, 1400, 64, 64, 1100, 4, None),
    (1, 1, 1, 1300, 128, 128, 1024, 40, None),
    (2, 4, 2, 700, 80, 72, 256, 7, [700, 401]),
    (1, 40, 40, 600, 64, 64, 260, 4, None),
    (1, 40, 20, 600, 64, 48, 260, 70, [555]),
    (1, 40, 40, 600, 128, 128, 256, 3, None),
    (1, 40, 40, 600, 96, 93, 256, 33, None),
    (4, 20, 20, 500, 32, 32, 512, 0, [500, 130, 1, 499]),
]


@pytest.mark.parametrize("b,h,hk,n,d,dv,window,sinks,lengths", LARGE)
def test_large_fp16_gradients(b, h, hk, n, d, dv, window, sinks, lengths):
    """Gradients of logits beyond fp16, whose sums are not: rows' gradients from 2^-4 to 2^9 times a unit normal, logits with
    a deviation of 2."""
    g = torch.Generator().manual_seed(n + d)
    q, k, v, go = (torch.randn(*s, generator=g) for s in ((b, h, n, d), (b, hk, n, d), (b, hk, n, dv), (b, h, n, dv)))
    q, go = 2 * q, go * 2.0 ** (13 * torch.rand(b, h, n, 1, generator=g) - 4)
    q, k, v, go = (x.half() for x in (q, k, v, go))
    kw = dict(window=window, sinks=sinks)
    want = statement(q, k, v, go, lengths=lengths, **kw)
    assert all(want[x][0].abs().max() < 60000 for x in ("dq", "dk", "dv"))
    # what a fixed lift of the window's power of two would make of them
    p = (q[0, 0].double() @ k[0, 0].double().T / math.sqrt(d)).masked_fill(~ref.visible(n, n, **kw), -math.inf).softmax(1)
    ds = (p * (go[0, 0].double() @ v[0, 0].double().T - (go[0, 0].double() * (p @ v[0, 0].double())).sum(1, keepdim=True)))
    assert 256 * ds.abs().max() > 65504
    x = [t.to(DEV) for t in (q, k, v)]
    if lengths is not None:
        kw["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out, lse, rest = swa.sink_window_forward(*x, with_rest=True, **kw)
    grads = swa.sink_window_backward(go.to(DEV), *x, out, lse, rest=rest, **kw)
    worst = {name: ref.over(y, want[name]) for name, y in zip(("dq", "dk", "dv"), grads)}
    assert all(y <= 1.0 for y in worst.values()), worst
    again = swa.sink_window_backward(go.to(DEV), *x, out, lse, rest=rest, **kw)
    assert all(torch.equal(y, z) for y, z in zip(grads, again))


def passes(go, *x, **kw):
    """Milliseconds of one backward pass, the least of five."""
    out, lse, rest = swa.sink_window_forward(*x, with_rest=True, **kw)
    best = math.inf
    for _ in range(6):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        swa.sink_window_backward(go, *x, out, lse, rest=rest, **kw)
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("heads,d", [(4, 64), (32, 64), (32, 128)])
def test_large_fp16_gradients_take_no_longer(heads, d):
    """Values choose no other way through the kernels: rows taken one by one would be 50 times as long and more."""
    g = torch.Generator().manual_seed(d)
    q, k, v, go = (torch.randn(1, heads, 2048, d, generator=g).to(DEV) for _ in range(4))
    x = [t.half() for t in (q, k, v)]
    kw = dict(window=1024, sinks=4)
    small, large = (passes((go * s).half(), *x, **kw) for s in (1.0, 1024.0))
    assert large < 4 * small, (small, large)
