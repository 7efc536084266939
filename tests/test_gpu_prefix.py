"""Attention over a shared prefix and received weights on the GPU against their float64 statements, element by element
within the bounds that the statements derive from the roundings."""

import math

import pytest
import torch

import heavy_hitter_attention as hha
import kept_reference as ref
import shared_prefix_attention as spa

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(b, h, hk, n, m, sets, p, d, dv, dtype, seed=0):
    g = torch.Generator().manual_seed(1000 * seed + 7 * n + d + p)
    return [torch.randn(*s, generator=g).to(dtype) for s in
            ((b, h, n, d), (b, hk, m, d), (b, hk, m, dv), (sets, hk, p, d), (sets, hk, p, dv))]


def ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)


def attend(x, **kw):
    kw = {k: ints(y) if k in ("lengths", "counts", "prefix_lengths") else y for k, y in kw.items()}
    out, lse = spa.shared_prefix_attention(*(t.to(DEV) for t in x), with_lse=True, **kw)
    torch.cuda.synchronize()
    return {"out": out.cpu(), "lse": lse.cpu()}


def check(got, want):
    worst = {name: ref.over(got[name], want[name]) for name in want}
    assert all(x <= 1.0 for x in worst.values()), worst


CASES = [  # b h hk n m sets p d dv lengths counts prefix_lengths
    (1, 1, 1, 1, 1, 1, 0, 8, 8, None, None, None),
    (1, 1, 1, 1, 1, 1, 1, 1, 1, None, None, None),
    (2, 2, 1, 1, 5, 1, 3, 16, 24, [5, 0], None, None),
    (2, 1, 1, 2, 5, 2, 7, 5, 3, [5, 1], None, [7, 0]),
    (4, 8, 2, 1, 70, 1, 130, 64, 64, [70, 1, 64, 33], None, None),
    (3, 6, 2, 9, 40, 3, 65, 93, 77, [40, 17, 3], [9, 5, 9], [65, 1, 40]),
    (6, 4, 4, 33, 33, 2, 200, 128, 128, [33, 1, 0, 32, 5, 33], [33, 1, 0, 32, 5, 33], None),
    (2, 4, 1, 40, 300, 1, 513, 40, 32, None, None, None),
    (1, 2, 2, 257, 257, 1, 100, 64, 64, None, None, [99]),
    (1, 3, 1, 130, 900, 1, 700, 96, 80, [777], [129], None),
    (5, 40, 1, 1, 100, 1, 600, 32, 64, [100, 99, 3, 0, 64], None, None),
    (1, 2, 1, 300, 300, 1, 0, 32, 32, [290], [290], None),
    (2, 1, 1, 70, 100, 1, 64, 33, 40, [-5, 200], [90, 7], [77]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,n,m,sets,p,d,dv,lengths,counts,plens", CASES)
def test_outputs_and_statistics(b, h, hk, n, m, sets, p, d, dv, lengths, counts, plens, dtype):
    x = make(b, h, hk, n, m, sets, p, d, dv, dtype)
    kw = dict(lengths=lengths, counts=counts, prefix_lengths=plens)
    check(attend(x, **kw), ref.prefix_attention(*x, **kw))


WALKS = [  # keys enough for the prefix and the own tokens to be walked apart
    (2, 2, 1, 1, 5, 1, 600, 16, 24, [5, 0], None, None),
    (4, 1, 1, 2, 5, 2, 700, 5, 3, [5, 1, 0, 2], None, [700, 0]),
    (6, 6, 2, 9, 40, 3, 600, 93, 77, [40, 17, 3, 40, 0, 1], [9, 5, 9, 1, 0, 1], [600, 1, 333]),
    (6, 4, 4, 33, 33, 2, 900, 128, 128, [33, 1, 0, 32, 5, 33], [33, 1, 0, 32, 5, 33], None),
    (8, 64, 32, 60, 70, 1, 500, 32, 32, [70, 66, 1, 0, 33, 64, 65, 70], [60, 60, 1, 0, 33, 60, 60, 2], None),
    (6, 2, 2, 64, 64, 1, 520, 64, 64, None, None, [519]),
    (2, 3, 1, 30, 60, 1, 600, 96, 80, [60, 31], [30, 29], None),
    (3, 1, 1, 1, 1, 1, 9000, 32, 32, None, None, None),
    (1, 2, 2, 1, 9000, 1, 0, 32, 64, [8999], None, None),
    (2, 1, 1, 1, 4500, 1, 700, 64, 32, [4500, 1], None, [640]),
    (16, 8, 8, 32, 40, 1, 8200, 64, 32, None, None, None),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,n,m,sets,p,d,dv,lengths,counts,plens", WALKS)
def test_walks_that_are_joined(b, h, hk, n, m, sets, p, d, dv, lengths, counts, plens, dtype):
    x = make(b, h, hk, n, m, sets, p, d, dv, dtype, seed=2)
    kw = dict(lengths=lengths, counts=counts, prefix_lengths=plens)
    check(attend(x, **kw), ref.prefix_attention(*x, **kw))


MANY = [  # enough rows for tiles of 128, and for workgroups that finish their rows
    (16, 32, 8, 5, 64, 1, 300, 64, 64, None, None, None),
    (24, 16, 16, 130, 130, 2, 90, 64, 32, None, None, [90, 61]),
    (32, 32, 8, 1, 300, 4, 400, 128, 128, None, None, None),
    (8, 64, 32, 66, 70, 1, 64, 32, 32, [70, 66, 1, 0, 33, 64, 65, 70], [66, 60, 1, 5, 33, 64, 65, 2], None),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,n,m,sets,p,d,dv,lengths,counts,plens", MANY)
def test_many_rows(b, h, hk, n, m, sets, p, d, dv, lengths, counts, plens, dtype):
    x = make(b, h, hk, n, m, sets, p, d, dv, dtype, seed=1)
    kw = dict(lengths=lengths, counts=counts, prefix_lengths=plens)
    check(attend(x, **kw), ref.prefix_attention(*x, **kw))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,n,m,sets,p,d,dv,lengths,counts,plens", CASES[1:])
def test_received_weights(b, h, hk, n, m, sets, p, d, dv, lengths, counts, plens, dtype):
    x = make(b, h, hk, n, m, sets, p, d, dv, dtype, seed=2)
    kw = dict(lengths=lengths, counts=counts)
    q, k = x[0].to(DEV), x[1].to(DEV)
    got = hha.received_attention(q, k, lengths=ints(lengths), counts=ints(counts))
    assert ref.over(got.cpu(), ref.received(*x[:2], **kw)) <= 1.0
    # behind a prefix: the statistics take its weights in
    lse = attend(x, prefix_lengths=plens, **kw)["lse"]
    got = hha.received_attention(q, k, lengths=ints(lengths), counts=ints(counts), lse=lse.to(DEV))
    assert ref.over(got.cpu(), ref.received(*x[:2], lse=lse, **kw)) <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
def test_received_weights_of_many_keys(dtype):
    x = make(2, 16, 8, 900, 1100, 1, 1, 64, 64, dtype, seed=3)
    got = hha.received_attention(x[0].to(DEV), x[1].to(DEV))
    assert ref.over(got.cpu(), ref.received(*x[:2])) <= 1.0


@pytest.mark.parametrize("scale", [-0.3, 0.0, 4.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(dtype, scale):
    x = make(2, 4, 2, 20, 50, 1, 90, 32, 32, dtype, seed=4)
    check(attend(x, scale=scale), ref.prefix_attention(*x, scale=scale))
    got = hha.received_attention(x[0].to(DEV), x[1].to(DEV), scale=scale)
    assert ref.over(got.cpu(), ref.received(*x[:2], scale=scale)) <= 1.0
