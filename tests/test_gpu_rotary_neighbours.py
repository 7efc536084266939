"""Columns that do not turn take nothing of the columns next to them, infinities and NaN included."""

import math

import pytest
import torch

import qk_rotary as qkr

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [0, 32])
@pytest.mark.parametrize("d", [64, 93])  # rows in 16-byte units, and not
def test_infinities_stay_in_their_column(d, rotary, interleaved):
    """x / inf: NaN at an infinity that does not turn, 0 elsewhere; a NaN makes its row NaN."""
    x = torch.ones(1, 1, 4, d, device=DEV)
    for row, col in enumerate((d - 1, d - 10)):
        x[0, 0, row, col] = math.inf
    x[0, 0, 2, d - 1] = math.nan
    y = qkr.qk_norm_rotary(x, x, qkr.rotary_table(4, rotary, device=DEV), interleaved=interleaved)[0][0, 0]
    for row, col in enumerate((d - 1, d - 10)):
        others = torch.arange(d, device=DEV) != col
        assert torch.isnan(y[row, col]) and not y[row, others].any()
    assert torch.isnan(y[2]).all() and torch.isfinite(y[3]).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d", [64, 93])
def test_gradients_stay_in_their_column(d, interleaved):
    """The weights' gradient sums every column's own."""
    g = torch.Generator().manual_seed(d)
    x, go = (torch.randn(1, 2, 5, d, generator=g).to(DEV) for _ in range(2))
    w = torch.ones(d, device=DEV)
    table = qkr.rotary_table(5, 32, device=DEV)
    args = dict(q_weight=w, k_weight=w, interleaved=interleaved)
    want = qkr.qk_norm_rotary_backward(go, go, x, x, table, **args)[2]
    bad = go.clone()
    bad[0, 1, 3, d - 2] = math.nan
    got = qkr.qk_norm_rotary_backward(bad, go, x, x, table, **args)[2]
    others = torch.arange(d, device=DEV) != d - 2
    assert torch.isnan(got[d - 2]) and torch.equal(got[others], want[others])
