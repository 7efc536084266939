"""Windowed attention with infinities and NaN: which results they reach, element by element, and what they cost."""

import math

import pytest
import torch

import sink_window_attention as swa
import window_reference as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def reached(bad_q, bad_k, bad_v, bad_go, window, sinks, lengths):
    """Which results values that are not finite reach, by the formulas: truth values like out, dq, dk and dv."""
    b, h, n, d = bad_q.shape
    hk = bad_k.shape[1]
    out, dq = torch.zeros_like(bad_go), torch.zeros_like(bad_q)
    dk, dv = torch.zeros_like(bad_k), torch.zeros_like(bad_v)
    for bi in range(b):
        see = ref.visible(n, n if lengths is None else lengths[bi], window, sinks)
        rows = see.any(1)
        for hi in range(h):
            ki = hi * hk // h
            count = lambda x: (see.double() @ x.double()) > 0
            row = rows & (bad_q[bi, hi].any(1) | count(bad_k[bi, ki].any(1)))  # a logit is not finite: all of the row's weights
            out[bi, hi] = row[:, None] | count(bad_v[bi, ki])
            delta = rows & (out[bi, hi].any(1) | bad_go[bi, hi].any(1))
            dq[bi, hi] = (row | delta)[:, None]
            back = lambda x: (see.T.double() @ x.double()) > 0
            dk[bi, ki] |= back(row | delta)[:, None]
            dv[bi, ki] |= back(row[:, None] | bad_go[bi, hi])
    return dict(out=out, dq=dq, dk=dk, dv=dv)


SHAPES = [  # b h hk n d dv window sinks lengths: every padded width, rows of 32 and of 128 a workgroup, sinks of both kinds
    (1, 2, 1, 300, 64, 64, 70, 5, None),
    (1, 2, 2, 400, 128, 128, 100, 40, [377]),
    (2, 2, 1, 260, 80, 93, 600, 0, [260, 131]),
    (4, 64, 64, 300, 32, 32, 64, 4, [300, 131, 299, 0]),
    (2, 64, 32, 400, 64, 48, 90, 3, None),
    (2, 64, 64, 300, 96, 96, 70, 33, [300, 200]),
    (2, 64, 64, 300, 128, 128, 60, 5, [290, 300]),
    (2, 64, 64, 300, 120, 100, 400, 0, None),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,n,d,dv,window,sinks,lengths", SHAPES)
def test_values_that_are_not_finite_reach_what_sees_them(b, h, hk, n, d, dv, window, sinks, lengths, dtype):
    g = torch.Generator().manual_seed(n + d)
    x = [torch.randn(*s, generator=g).to(dtype) for s in ((b, h, n, d), (b, hk, n, d), (b, hk, n, dv), (b, h, n, dv))]
    kw = dict(window=window, sinks=sinks)
    want = ref.window_attention(*x[:3], grad=x[3], lengths=lengths, **kw)
    # a few heads get a few such values each; every head has rows and keys that see none
    bad = [torch.zeros(t.shape, dtype=torch.bool) for t in x]
    values = [math.inf, -math.inf, math.nan]
    for i in range(6):
        for which in (2, 3) if i % 2 else (i // 2,):
            t = x[which]
            at = [int(torch.randint(0, s, (1,), generator=g)) for s in t.shape]
            at[1] = (7 * i + which) % t.shape[1]
            t[tuple(at)] = values[i % 3]
            bad[which][tuple(at)] = True
    reach = reached(*bad, window, sinks, lengths)
    x = [t.to(DEV) for t in x]
    if lengths is not None:
        kw["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out, lse, rest = swa.sink_window_forward(*x[:3], with_rest=True, **kw)
    grads = swa.sink_window_backward(x[3], *x[:3], out, lse, rest=rest, **kw)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        got = got.double().cpu()
        hit = reach[name]
        assert hit.any() and not hit.all()
        assert not torch.isfinite(got[hit]).any(), name
        assert ref.over(got[~hit], tuple(t[~hit] for t in want[name])) <= 1.0, name
    again = swa.sink_window_backward(x[3], *x[:3], out, lse, rest=rest, **kw)
    for y, z in zip(grads, again):
        assert torch.equal(y.nan_to_num(), z.nan_to_num())


@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_one_infinite_value_keeps_its_sign(value):
    """sum_j p_ij v_j with one infinite v_j is that infinity."""
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(1, 64, 300, 64, generator=g).bfloat16() for _ in range(3))
    v[0, 5, 100, 7] = value
    out = swa.sink_window_causal_attention(q.to(DEV), k.to(DEV), v.to(DEV), window=90, sinks=2).cpu()
    assert (out[0, 5, 100:190, 7] == value).all()
    assert torch.isfinite(out[0, 5, :100]).all() and torch.isfinite(out[0, 5, 190:]).all()


def least(f):
    best = math.inf
    for _ in range(4):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        f()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("where", ["one", "all"])
@pytest.mark.parametrize("d", [64, 128])
def test_cost_of_values_that_are_not_finite(d, where):
    """Ten times an ordinary call at most: a step whose gradient overflowed must not hold the device (rows and keys taken one
    after another would be a hundred times as long and more)."""
    g = torch.Generator().manual_seed(d)
    q, k, v, go = (torch.randn(4, 8, 4096, d, generator=g).bfloat16().to(DEV) for _ in range(4))
    kw = dict(window=1024, sinks=4)

    def passes(q, k, v, go):
        out, lse, rest = swa.sink_window_forward(q, k, v, with_rest=True, **kw)
        swa.sink_window_backward(go, q, k, v, out, lse, rest=rest, **kw)

    plain = least(lambda: passes(q, k, v, go))
    bad_v, bad_go = v.clone(), go.clone()
    if where == "one":
        bad_v[0, 0, 2000, 3], bad_go[1, 1, 2100, 5] = math.inf, math.nan
    else:
        bad_go.fill_(math.nan)
    assert least(lambda: passes(q, k, bad_v, bad_go)) < 10 * plain
    if where == "all":
        bad_v.fill_(math.nan)
        assert least(lambda: passes(q, k, bad_v, go)) < 10 * plain


@pytest.mark.parametrize("heads", [2, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("logit", [1e8, -1e8, 1e11, -1e11, 1e25, -1e31])
def test_finite_logits_of_any_size(logit, dtype, heads):
    """Equal logits give the mean of what is seen, one that is larger gives its value."""
    n, window = 200, 70
    g = torch.Generator().manual_seed(5)
    v = torch.randn(1, heads, n, 32, generator=g).to(dtype)
    q, k = torch.zeros(1, heads, n, 16), torch.zeros(1, heads, n, 16)
    q[..., 0], k[..., 0] = abs(logit) ** 0.5, math.copysign(abs(logit) ** 0.5, logit)
    kw = dict(window=window, sinks=0, scale=1.0)
    out = swa.sink_window_causal_attention(*(x.to(dtype).to(DEV) for x in (q, k, v)), **kw).cpu().double()
    see = ref.visible(n, n, window, 0).double()
    mean = see @ v.double() / see.sum(1, keepdim=True)
    size = see @ v.double().abs() / see.sum(1, keepdim=True)
    # the output's rounding, 16-bit weights' half a step, and 200 fp32 operations
    u = ref.half_step(dtype)
    assert ((out - mean).abs() <= u * mean.abs() + (ref.weight_step(dtype) + 200 * ref.F24) * size).all()
    k[:, :, 50, 0] += k[:, :, 50, 0].abs() / 4  # apart by far more than an exponent holds
    out = swa.sink_window_causal_attention(*(x.to(dtype).to(DEV) for x in (q, k, v)), **kw).cpu().double()
    # w v / w with a weight w that is not 1 (its exponent's argument is rounded): the weight as the sum takes it, three fp32
    # roundings (w v, 1 / w, their product) and the output's
    one = v[:, :, 50:51].double()
    off = (out[:, :, 50:120] - one).abs()
    assert (off <= (u + ref.weight_step(dtype) + 4 * ref.F24) * one.abs()).all()
