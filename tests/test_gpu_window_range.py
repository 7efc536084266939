"""Windowed attention and its cache where the element type's range counts: tiny weights of long rows, large gradients."""

import math

import pytest
import torch

import sink_window_attention as swa

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
