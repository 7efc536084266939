"""Refusals of the windowed attention, the head norm with rotation and the token cache, which need no GPU, and the
float64 statements' own checks."""

import ctypes
import math

import pytest
import torch

import _native
import qk_rotary as qkr
import sink_window_attention as swa
import window_reference as ref


def x(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("q,k,v,kw,message", [
    (x(4, 8), x(4, 8), x(4, 8), dict(window=0), "window"),
    (x(4, 8), x(4, 8), x(4, 8), dict(window=2.0), "window"),
    (x(4, 8), x(4, 8), x(4, 8), dict(window=True), "window"),
    (x(4, 8), x(4, 8), x(4, 8), dict(window=2, sinks=-1), "sinks"),
    (x(1, 4, 8), x(1, 4, 8), x(1, 4, 8), dict(window=2), r"\[N,D\]"),
    (x(4, 8), x(1, 1, 4, 8), x(4, 8), dict(window=2), r"\[N,D\]"),
    (x(4, 8), x(5, 8), x(5, 8), dict(window=2), "k must be"),
    (x(4, 8), x(4, 9), x(4, 8), dict(window=2), "k must be"),
    (x(4, 8), x(4, 8), x(5, 8), dict(window=2), "v must be"),
    (x(1, 3, 4, 8), x(1, 2, 4, 8), x(1, 2, 4, 8), dict(window=2), "multiple"),
    (x(1, 2, 4, 8), x(1, 0, 4, 8), x(1, 0, 4, 8), dict(window=2), "multiple"),
    (x(4, 129), x(4, 129), x(4, 8), dict(window=2), "widths"),
    (x(4, 8), x(4, 8), x(4, 129), dict(window=2), "widths"),
    (x(4, 8), x(4, 8), x(4, 8, dtype=torch.float16), dict(window=2), "one dtype"),
    (*(x(4, 8, dtype=torch.float64) for _ in range(3)), dict(window=2), "not supported"),
    (x(2, 1, 4, 8), x(2, 1, 4, 8), x(2, 1, 4, 8), dict(window=2, lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (x(2, 1, 4, 8), x(2, 1, 4, 8), x(2, 1, 4, 8), dict(window=2, lengths=torch.zeros(2, dtype=torch.int64)), "lengths"),
    (x(4, 8), x(4, 8), x(4, 8), dict(window=2), "GPU"),
])
def test_attention_refuses(q, k, v, kw, message):
    with pytest.raises(ValueError, match=message):
        swa.sink_window_causal_attention(q, k, v, **kw)
    with pytest.raises(ValueError, match=message):
        swa.sink_window_forward(q, k, v, **kw)


def test_scales_must_be_finite():
    for bad in (math.inf, math.nan):
        with pytest.raises(ValueError, match="finite"):
            swa._attention_scale(bad, 8)


def test_differentiable_calls_refuse_capture(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for f, args in ((swa._SinkWindow, (x(1, 1, 4, 8).requires_grad_(), x(1, 1, 4, 8), x(1, 1, 4, 8), 2, 0, 1.0, None)),
                    (qkr._NormRotary, (x(1, 1, 4, 8).requires_grad_(), x(1, 1, 4, 8), None, None, x(4, 8), None, None))):
        with pytest.raises(RuntimeError, match="captured"):
            f.apply(*args)


@pytest.mark.parametrize("kw,message", [
    (dict(streams=0), "positive"), (dict(heads=3, kv_heads=2), "multiple"), (dict(kv_heads=0), "positive"),
    (dict(window=0), "window"), (dict(sinks=-1), "sinks"), (dict(dim=129), "widths"), (dict(value_dim=0), "widths"),
    (dict(dtype=torch.float64), "not supported"), (dict(storage="int4"), "storage"), (dict(device="cpu"), "GPU"),
    (dict(window=1 << 30, sinks=1), "at most"), (dict(scale=math.nan), "finite"),
])
def test_cache_refuses(kw, message):
    args = dict(dim=8, value_dim=8, streams=1, heads=1, window=4, sinks=1)
    args.update(kw)
    with pytest.raises(ValueError, match=message):
        swa.SinkWindowStreamingAttention(args.pop("dim"), args.pop("value_dim"), **args)


@pytest.mark.parametrize("q,k,kw,message", [
    (x(8), x(8), {}, "q and k must be"),
    (x(2, 3, 8), x(2, 8), {}, "q and k must be"),
    (x(1, 2, 3, 8), x(1, 2, 4, 8), {}, "match"),
    (x(1, 2, 3, 8), x(1, 2, 3, 7), {}, "match"),
    (x(3, 257), x(3, 257), {}, "widths"),
    (x(3, 8), x(3, 8, dtype=torch.float16), {}, "one dtype"),
    (x(3, 8, dtype=torch.float64), x(3, 8, dtype=torch.float64), {}, "one dtype"),
    (x(3, 8), x(3, 8), dict(table=x(4, 7)), "table"),
    (x(3, 8), x(3, 8), dict(table=x(4, 10)), "table"),
    (x(3, 8), x(3, 8), dict(table=x(0, 8)), "positions"),
    (x(3, 8), x(3, 8), dict(table=x(4, 8, dtype=torch.float16)), "table"),
    (x(3, 8), x(3, 8), dict(q_weight=x(7)), "weights"),
    (x(3, 8), x(3, 8), dict(q_weight=x(8, dtype=torch.float16)), "weights"),
    (x(3, 8, dtype=torch.float16), x(3, 8, dtype=torch.float16),
     dict(q_weight=x(8, dtype=torch.float16), k_weight=x(8)), "weights"),
    (x(3, 8), x(3, 8), dict(positions=torch.zeros(3)), "int32 or int64"),
    (x(3, 8), x(3, 8), dict(positions=torch.zeros(4, dtype=torch.int32)), "positions must be"),
    (x(2, 1, 8), x(2, 1, 8), dict(positions=torch.zeros(1, dtype=torch.int32)), "positions must be"),
    (x(3, 8), x(3, 8), dict(eps=-1.0), "eps"),
    (x(3, 8), x(3, 8), dict(eps=math.nan), "eps"),
    (x(3, 8), x(3, 8), {}, "GPU"),
])
def test_rotary_refuses(q, k, kw, message):
    kw = dict(kw)
    table = kw.pop("table", x(4, 8))
    with pytest.raises(ValueError, match=message):
        qkr.qk_norm_rotary(q, k, table, **kw)


def test_rotary_table_takes_no_gradient(monkeypatch):
    monkeypatch.setattr(qkr, "_check_gpu", lambda *a: None)
    with pytest.raises(ValueError, match="table takes no gradient"):
        qkr.qk_norm_rotary(x(3, 8), x(3, 8), x(4, 8).requires_grad_())


def test_rotary_table():
    t = qkr.rotary_table(100, 8, base=100.0)
    assert t.shape == (100, 8) and t.dtype == torch.float32
    assert abs(t[7, 1].item() - math.cos(7 * 100.0 ** -0.25)) < 1e-7
    assert abs(t[7, 5].item() - math.sin(7 * 100.0 ** -0.25)) < 1e-7
    assert qkr.rotary_table(3, 0).shape == (3, 0)
    for bad in ((0, 8, 1e4), (3, 7, 1e4), (3, 8, 0.0)):
        with pytest.raises(ValueError):
            qkr.rotary_table(bad[0], bad[1], base=bad[2])


def test_library_refuses_without_touching_a_device():
    lib = _native.load_library()
    st = (ctypes.c_int64 * 12)(*([64] * 12))
    E = _native

    def fwd(q=16, k=16, v=16, dt=0, b=1, h=2, hk=1, n=8, d=8, dv=8, s=st, scale=1.0, w=4, sinks=1, out=16, rest=None):
        return lib.sta_window_attention(q, k, v, dt, b, h, hk, n, d, dv, s, scale, w, sinks, None, out, rest, None, None)

    for kw, want in [(dict(q=None), E.STA_ERR_ARG), (dict(out=None), E.STA_ERR_ARG), (dict(out=8), E.STA_ERR_ARG), (dict(rest=8), E.STA_ERR_ARG),
                     (dict(s=None), E.STA_ERR_ARG), (dict(dt=3), E.STA_ERR_DTYPE), (dict(b=0), E.STA_ERR_SHAPE),
                     (dict(h=3, hk=2), E.STA_ERR_SHAPE), (dict(n=0), E.STA_ERR_SHAPE), (dict(d=129), E.STA_ERR_UNSUPPORTED),
                     (dict(dv=129), E.STA_ERR_UNSUPPORTED), (dict(d=3), E.STA_ERR_UNSUPPORTED),
                     (dict(dt=1, dv=7), E.STA_ERR_UNSUPPORTED), (dict(n=(1 << 30) + 1), E.STA_ERR_UNSUPPORTED),
                     (dict(w=0), E.STA_ERR_ARG), (dict(sinks=-1), E.STA_ERR_ARG), (dict(scale=math.inf), E.STA_ERR_ARG),
                     (dict(b=1 << 31), E.STA_ERR_UNSUPPORTED), (dict(b=1 << 30, n=1 << 20), E.STA_ERR_SHAPE),
                     (dict(b=1 << 23, n=1), E.STA_ERR_SHAPE)]:  # 2^24 workgroups
        assert fwd(**kw) == want, kw
    assert lib.sta_window_backward_bytes(0, 1, 2, 1, 8, 8, 8, 0, 1) == -1
    need = lib.sta_window_backward_bytes(0, 1, 2, 1, 1000, 8, 8, 100, 4)
    assert need >= 4 * 2 * 1000
    back = [16] * 5 + [None, 16, 0, 1, 2, 1, 1000, 8, 8, st, 1.0, 100, 4, None, 16, 16, 16, 16]
    assert lib.sta_window_attention_backward(*back, need - 1, None) == E.STA_ERR_SCRATCH
    assert lib.sta_window_attention_backward(None, *back[1:], need, None) == E.STA_ERR_ARG
    wide = [16] * 5 + [None, 16, 0, 1 << 23, 2, 1, 1, 8, 8, st, 1.0, 100, 4, None, 16, 16, 16, 16]
    assert lib.sta_window_attention_backward(*wide, 1 << 40, None) == E.STA_ERR_SHAPE

    rot = dict(q=16, k=16, dt=0, b=1, h=2, hk=1, n=8, d=8, s=st, qw=None, kw=None, wt=0, table=16, limit=8, r=8, i=0,
               pos=None, p64=0, psb=0, psn=0, eps=1e-6, qo=16, ko=16)
    for kw, want in [(dict(q=None), E.STA_ERR_ARG), (dict(ko=8), E.STA_ERR_ARG), (dict(dt=5), E.STA_ERR_DTYPE),
                     (dict(wt=5), E.STA_ERR_DTYPE), (dict(r=7), E.STA_ERR_SHAPE), (dict(r=10), E.STA_ERR_SHAPE),
                     (dict(d=257), E.STA_ERR_UNSUPPORTED), (dict(limit=0), E.STA_ERR_ARG), (dict(eps=-1.0), E.STA_ERR_ARG),
                     (dict(b=1 << 30), E.STA_ERR_UNSUPPORTED), (dict(h=20000), E.STA_ERR_UNSUPPORTED),
                     (dict(h=0, hk=0), E.STA_ERR_SHAPE), (dict(table=None), E.STA_ERR_ARG)]:
        a = dict(rot, **kw)
        assert lib.sta_head_rotary(*a.values(), None) == want, kw
    assert lib.sta_head_rotary_backward_bytes(0, 1, 1, 1, 8) == -1

    sizes = (ctypes.c_int64 * 4)()
    assert lib.sta_ring_layout(1, 1, 2, 3, 64, 48, 60, 4, sizes) == E.STA_OK
    assert list(sizes) == [2 * 3 * 2 * 32 * 64 * 2, 2 * 3 * 2 * 32 * 64 * 2, 0, 0]
    assert lib.sta_ring_layout(1, 3, 2, 3, 70, 48, 61, 4, sizes) == E.STA_OK
    assert list(sizes) == [2 * 3 * 3 * 32 * 48, 2 * 3 * 3 * 32 * 32, 2 * 3 * 3 * 32 * 4, 2 * 3 * 3 * 32 * 2]
    assert lib.sta_ring_layout(1, 2, 2, 3, 64, 48, 60, 4, sizes) == E.STA_ERR_DTYPE  # fp16 storage of bf16
    assert lib.sta_ring_layout(0, 0, 1, 1, 8, 8, (1 << 30), 1, sizes) == E.STA_ERR_UNSUPPORTED
    assert lib.sta_ring_attention_bytes(1, 3, 2, 8, 8, 4, 0) == -1
    ring = dict(q=16, k=16, v=16, dt=1, store=3, s=1, h=2, hk=1, d=8, dv=8, st=st, scale=1.0, w=4000, sinks=1, ck=16, cv=16,
                ek=16, ev=16, counts=16, out=16, ws=None, wb=0)
    for kw, want in [(dict(q=None), E.STA_ERR_ARG), (dict(k=None), E.STA_ERR_ARG), (dict(counts=None), E.STA_ERR_ARG),
                     (dict(ek=None), E.STA_ERR_ARG), (dict(ck=8), E.STA_ERR_ARG), (dict(store=2), E.STA_ERR_DTYPE),
                     (dict(h=3, hk=2), E.STA_ERR_SHAPE), (dict(w=0), E.STA_ERR_ARG), (dict(scale=math.nan), E.STA_ERR_ARG),
                     (dict(), E.STA_ERR_SCRATCH), (dict(s=1 << 24, w=4), E.STA_ERR_SHAPE)]:
        a = dict(ring, **kw)
        assert lib.sta_ring_attention(*a.values(), None) == want, kw
    fill = dict(k=16, v=16, dt=1, store=1, s=1, hk=1, rows=4, d=8, dv=8, st=st, w=4, sinks=1, take=None, ck=16, cv=16,
                ek=None, ev=None, counts=16)
    for kw, want in [(dict(k=None), E.STA_ERR_ARG), (dict(rows=0), E.STA_ERR_SHAPE), (dict(rows=1 << 31), E.STA_ERR_UNSUPPORTED),
                     (dict(d=129), E.STA_ERR_UNSUPPORTED), (dict(s=0), E.STA_ERR_SHAPE)]:
        a = dict(fill, **kw)
        assert lib.sta_ring_extend(*a.values(), None) == want, kw


def test_statement_of_attention_against_autograd():
    g = torch.Generator().manual_seed(0)
    q, k, v, go = (torch.randn(*s, generator=g, dtype=torch.float64) for s in
                   ((2, 4, 30, 6), (2, 2, 30, 6), (2, 2, 30, 5), (2, 4, 30, 5)))
    lengths = [30, 17]
    for t in (q, k, v):
        t.requires_grad_()
    see = torch.stack([ref.visible(30, n, 7, 3) for n in lengths])[:, None]
    kk, vv = k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
    s = (q @ kk.transpose(-1, -2) / math.sqrt(6)).masked_fill(~see, -math.inf)
    p = torch.where(see, s.softmax(-1).nan_to_num(), 0.0)
    out = p @ vv
    grads = torch.autograd.grad((out * go).sum(), (q, k, v))
    want = ref.window_attention(q.detach(), k.detach(), v.detach(), window=7, sinks=3, lengths=lengths, grad=go)
    for name, t in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert (want[name][0] - t).abs().max() < 1e-12, name


def test_statement_catches_planted_mistakes():
    """The bounds are tight enough to see a key too many, a sink too few and a weight left out."""
    g = torch.Generator().manual_seed(1)
    q, k, v, go = (torch.randn(1, 1, 60, 32, generator=g).bfloat16() for _ in range(4))
    want = ref.window_attention(q, k, v, window=20, sinks=3, grad=go)
    for wrong in (dict(window=21, sinks=3), dict(window=20, sinks=2), dict(window=20, sinks=3, lengths=[59])):
        got = ref.window_attention(q, k, v, grad=go, **wrong)
        assert all(ref.over(got[name][0], want[name]) > 1.5 for name in want), wrong


def test_statement_of_the_norm_against_autograd():
    g = torch.Generator().manual_seed(2)
    x_, w, go = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 3, 5, 10), (10,), (2, 3, 5, 10)))
    table = qkr.rotary_table(9, 6).double()[torch.tensor([[0, 3, 8, 2, 1], [5, 5, 4, 7, 6]])]
    cos, sin = table.chunk(2, -1)
    for interleaved in (False, True):
        x_.requires_grad_()
        w.requires_grad_()
        h = x_ / (x_.square().mean(-1, keepdim=True) + 1e-3).sqrt() * w
        z = (torch.complex(h[..., 0:6:2], h[..., 1:6:2]) if interleaved else torch.complex(h[..., :3], h[..., 3:6]))
        z = z * torch.complex(cos, sin)[:, None]
        parts = torch.stack([z.real, z.imag], -1).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1)
        y = torch.cat([parts, h[..., 6:]], -1)
        dx, dw = torch.autograd.grad((y * go).sum(), (x_, w))
        want = ref.norm_rotary(x_.detach(), w.detach(), cos, sin, eps=1e-3, interleaved=interleaved, grad=go)
        for name, t in (("y", y), ("dx", dx), ("dw", dw)):
            assert (want[name][0] - t).abs().max() < 1e-12, (interleaved, name)


def test_held_values():
    """Known 4-bit roundings: ties go to the even code, magnitudes above 6 units down to 6."""
    row = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.1, -0.3, 7.9])
    assert ref.as_held(row, "fp4").tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, -0.5, 6.0]
    assert ref.as_held(row * 2.0 ** 20, "fp4").tolist() == [x * 2.0 ** 20 for x in ref.as_held(row, "fp4").tolist()]


@pytest.mark.parametrize("dtype,rest", [(torch.float32, x(3, 8)), (torch.float16, x(3, 8)), (torch.float16, x(3, 7, dtype=torch.float16))])
def test_backward_refuses_another_rest(monkeypatch, dtype, rest):
    monkeypatch.setattr(swa, "_check_gpu", lambda *a: None)
    t = x(3, 8, dtype=dtype)
    with pytest.raises(ValueError, match="rest must be like out"):
        swa.sink_window_backward(t, t, t, t, t, x(3), window=2, rest=rest)
