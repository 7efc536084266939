"""The cache that keeps the most attended tokens and received weights where keys, values or logits are infinite or NaN."""

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


def odd(x):
    """x with rows at an odd element, off their units."""
    room = torch.zeros(*x.shape[:-1], x.shape[-1] + 3, dtype=x.dtype, device=x.device)
    room[..., 1:1 + x.shape[-1]] = x
    return room[..., 1:1 + x.shape[-1]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,n,m,d,counts", [
    # rows that stay in LDS, a block of 32 not full
    (1, 1, 1, 5, 64, 64, None), (2, 4, 2, 9, 70, 64, [9, 4]), (1, 6, 2, 33, 150, 93, None), (3, 2, 2, 100, 300, 128, [99, 1, 64]),
    # tiles of rows, the last not full
    (1, 2, 2, 257, 257, 64, None), (2, 4, 1, 130, 200, 128, [130, 77]), (2, 2, 1, 190, 333, 40, [3, 190]),
    (1, 3, 3, 200, 200, 93, [131])])
def test_received_weights_of_keys_that_hide(b, h, hk, n, m, d, counts, dtype):
    """Keys whose logits are -inf for every row receive 0, whatever fills up a block of rows; the others what they do."""
    q, k, pk = make(b + n + m + d, dtype, (b, h, n, d), (b, hk, m, d), (1, hk, 50, d))
    q[..., 0] = 1.0
    hide = torch.zeros(m, dtype=torch.bool)
    hide[2::7] = True
    finite = k.clone()
    k[:, :, hide, 0] = -math.inf
    want = ref.received(q, finite, counts=counts, hide=hide)
    assert (want[0][:, :, hide] == 0).all()
    lse = spa.shared_prefix_attention(q.to(DEV), k.to(DEV), k.to(DEV).nan_to_num(0.0, 0.0, 0.0), pk.to(DEV), pk.to(DEV),
                                      counts=ints(counts), with_lse=True)[1]
    given = ref.received(q, finite, counts=counts, hide=hide, lse=lse.cpu())
    for view in (lambda x: x, odd):
        got = hha.received_attention(view(q.to(DEV)), view(k.to(DEV)), counts=ints(counts))
        assert got[:, :, hide.to(DEV)].eq(0).all()
        assert ref.over(got, want) <= 1.0
        got = hha.received_attention(view(q.to(DEV)), view(k.to(DEV)), counts=ints(counts), lse=lse)
        assert ref.over(got, given) <= 1.0
