"""Head norm with rotation on the GPU (qk_rotary) against its float64 statement, element by element within the bounds
that the statement derives from the roundings."""

import math

import pytest
import torch

import qk_rotary as qkr
import window_reference as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(b, h, hk, n, d, dtype, wdtype, seed=0):
    g = torch.Generator().manual_seed(100 * seed + n + d)
    rows = [torch.randn(b, x, n, d, generator=g).mul(2).to(dtype) for x in (h, hk, h, hk)]
    weights = [(torch.randn(d, generator=g) * 0.3 + 1).to(wdtype) for _ in range(2)]
    return rows, weights


def check(got, want):
    worst = {name: ref.over(got[name], want[name]) for name in want}
    assert all(x <= 1.0 for x in worst.values()), worst


def statement(x, w, table, positions, go, eps, interleaved):
    rows = table.double()[positions.long()]
    cos, sin = rows.chunk(2, -1)
    if positions.ndim == 1:
        cos, sin = (t[None].expand(x.shape[0], -1, -1) for t in (cos, sin))
    want = ref.norm_rotary(x, w, cos, sin, eps=eps, interleaved=interleaved, grad=go)
    if w is not None:
        value, bound = want["dw"]
        want["dw"] = value, bound + ref.half_step(w.dtype) * value.abs() + (2.0 ** -25 if w.dtype == torch.float16 else 0)
    else:
        del want["dw"]
    return want


CASES = [  # b h hk n d rotary
    (1, 1, 1, 1, 1, 0),
    (1, 1, 1, 1, 2, 2),
    (2, 3, 1, 5, 8, 8),
    (1, 4, 2, 33, 64, 64),
    (3, 2, 2, 130, 72, 48),
    (2, 5, 1, 77, 128, 32),
    (1, 2, 1, 300, 96, 80),
    (2, 2, 1, 19, 93, 30),
    (1, 1, 1, 40, 256, 256),
    (1, 40, 8, 3, 64, 16),
    (2, 1, 1, 70, 130, 128),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,h,hk,n,d,rotary", CASES)
def test_results_and_gradients(b, h, hk, n, d, rotary, interleaved, dtype):
    for wdtype in {dtype, torch.float32}:
        (q, k, gq, gk), (qw, kw) = make(b, h, hk, n, d, dtype, wdtype)
        table = qkr.rotary_table(50 + n, rotary)
        positions = torch.arange(n)[None] + 3 * torch.arange(b)[:, None] + 11
        x = [t.to(DEV).requires_grad_() for t in (q, k, qw, kw)]
        yq, yk = qkr.qk_norm_rotary(x[0], x[1], table.to(DEV), q_weight=x[2], k_weight=x[3],
                                    positions=positions.to(DEV), eps=1e-5, interleaved=interleaved)
        grads = torch.autograd.grad((yq, yk), x, (gq.to(DEV), gk.to(DEV)))
        for y, dx, dw, t, w, g in ((yq, grads[0], grads[2], q, qw, gq), (yk, grads[1], grads[3], k, kw, gk)):
            check({"y": y, "dx": dx, "dw": dw}, statement(t, w, table, positions, g, 1e-5, interleaved))


def test_many_rows():
    (q, k, gq, gk), (qw, kw) = make(3, 12, 3, 3000, 64, torch.bfloat16, torch.float32, seed=1)
    table = qkr.rotary_table(3000, 64)
    x = [t.to(DEV).requires_grad_() for t in (q, k, qw, kw)]
    yq, yk = qkr.qk_norm_rotary(x[0], x[1], table.to(DEV), q_weight=x[2], k_weight=x[3])
    grads = torch.autograd.grad((yq, yk), x, (gq.to(DEV), gk.to(DEV)))
    for y, dx, dw, t, w, g in ((yq, grads[0], grads[2], q, qw, gq), (yk, grads[1], grads[3], k, kw, gk)):
        check({"y": y, "dx": dx, "dw": dw}, statement(t, w, table, torch.arange(3000), g, 1e-6, False))
    again = torch.autograd.grad(qkr.qk_norm_rotary(x[0], x[1], table.to(DEV), q_weight=x[2], k_weight=x[3]), x,
                                (gq.to(DEV), gk.to(DEV)))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("interleaved", [False, True])
def test_layouts_give_equal_bits(interleaved):
    (q, k, gq, gk), (qw, kw) = make(4, 6, 2, 21, 64, torch.bfloat16, torch.bfloat16, seed=2)
    q, k, gq, gk, qw, kw = (t.to(DEV) for t in (q, k, gq, gk, qw, kw))
    table = qkr.rotary_table(64, 64).to(DEV)
    positions = torch.randint(0, 64, (4, 21), device=DEV)
    kwargs = dict(q_weight=qw, k_weight=kw, interleaved=interleaved)
    y = qkr.qk_norm_rotary(q, k, table, positions=positions, **kwargs)
    dy = qkr.qk_norm_rotary_backward(gq, gk, q, k, table, positions=positions, **kwargs)
    swap = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, gq, gk)]
    for p in (positions, positions.int(), positions.t().contiguous().t()):
        for a, b in zip(qkr.qk_norm_rotary(*swap[:2], table, positions=p, **kwargs), y):
            assert torch.equal(a, b)
        for a, b in zip(qkr.qk_norm_rotary_backward(*swap[2:], *swap[:2], table, positions=p, **kwargs), dy):
            assert torch.equal(a, b)
    # one token of every stream
    one = qkr.qk_norm_rotary(q[:, :, 7], k[:, :, 7], table, positions=positions[:, 7], **kwargs)
    assert torch.equal(one[0], y[0][:, :, 7]) and torch.equal(one[1], y[1][:, :, 7])
    # a sequence without batch and heads
    single = qkr.qk_norm_rotary(q[1, 1], k[1, 1], table, positions=positions[1], **kwargs)
    assert torch.equal(single[0], y[0][1, 1]) and torch.equal(single[1], y[1][1, 1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_off_sixteen_bytes(dtype):
    (q, k, gq, gk), (qw, kw) = make(2, 3, 1, 17, 64, dtype, torch.float32, seed=3)
    table = qkr.rotary_table(20, 32)

    def off(x):
        y = torch.empty(*x.shape[:3], 67, dtype=dtype, device=DEV)
        y[..., 1:65] = x.to(DEV)
        return y[..., 1:65]

    x = [off(t) for t in (q, k, gq, gk)]
    y = qkr.qk_norm_rotary(x[0], x[1], table.to(DEV), q_weight=qw.to(DEV), k_weight=kw.to(DEV))
    dy = qkr.qk_norm_rotary_backward(x[2], x[3], x[0], x[1], table.to(DEV), q_weight=qw.to(DEV), k_weight=kw.to(DEV))
    for i, (t, w, g) in enumerate(((q, qw, gq), (k, kw, gk))):
        check({"y": y[i], "dx": dy[i], "dw": dy[2 + i]}, statement(t, w, table, torch.arange(17), g, 1e-6, False))


@pytest.mark.parametrize("d,rotary", [(64, 32), (93, 30)])
def test_positions_outside_the_table(d, rotary):
    (q, k, gq, gk), _ = make(1, 2, 1, 6, d, torch.float32, torch.float32, seed=4)
    table = qkr.rotary_table(10, rotary).to(DEV)
    positions = torch.tensor([0, 9, 10, -1, 2 ** 40, 3], device=DEV)
    y = qkr.qk_norm_rotary(q.to(DEV), k.to(DEV), table, positions=positions)
    bad = torch.tensor([False, False, True, True, True, False], device=DEV)
    for t in y:
        assert torch.isnan(t[:, :, bad]).all() and torch.isfinite(t[:, :, ~bad]).all()
    dq, dk, _, _ = qkr.qk_norm_rotary_backward(gq.to(DEV), gk.to(DEV), q.to(DEV), k.to(DEV), table, positions=positions)
    for t in (dq, dk):
        assert torch.isnan(t[:, :, bad]).all() and torch.isfinite(t[:, :, ~bad]).all()


def test_far_positions_keep_their_angles():
    table = qkr.rotary_table(1 << 20, 64, device=DEV)
    p = (1 << 20) - 1
    for i in (0, 1, 31):
        angle = p * 10000.0 ** (-2.0 * i / 64)
        assert abs(table[p, i].item() - math.cos(angle)) < 1e-7 and abs(table[p, 32 + i].item() - math.sin(angle)) < 1e-7


def test_captured_graph_and_stream():
    (q, k, gq, gk), (qw, kw) = make(2, 4, 2, 50, 64, torch.bfloat16, torch.bfloat16, seed=5)
    q, k, gq, gk, qw, kw = (t.to(DEV) for t in (q, k, gq, gk, qw, kw))
    table = qkr.rotary_table(64, 64).to(DEV)
    kwargs = dict(q_weight=qw, k_weight=kw)
    qkr.qk_norm_rotary_backward(gq, gk, q, k, table, **kwargs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = qkr.qk_norm_rotary(q, k, table, **kwargs)
        dy = qkr.qk_norm_rotary_backward(gq, gk, q, k, table, **kwargs)
    for seed in (6, 7, 8):
        rows, _ = make(2, 4, 2, 50, 64, torch.bfloat16, torch.bfloat16, seed=seed)
        for x, new in zip((q, k, gq, gk), rows):
            x.copy_(new)
        graph.replay()
        want = (*qkr.qk_norm_rotary(q, k, table, **kwargs), *qkr.qk_norm_rotary_backward(gq, gk, q, k, table, **kwargs))
        torch.cuda.synchronize()
        for a, b in zip((*y, *dy), want):
            assert torch.equal(a, b)


def test_empty_tensors():
    w = torch.ones(8, device=DEV, requires_grad=True)
    q = torch.empty(0, 2, 5, 8, device=DEV, requires_grad=True)
    y = qkr.qk_norm_rotary(q, q, qkr.rotary_table(8, 8).to(DEV), q_weight=w, k_weight=w)
    (y[0].sum() + y[1].sum()).backward()
    assert q.grad.shape == q.shape and not w.grad.any()
