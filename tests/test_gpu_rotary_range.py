"""Head norm with rotation of rows whose squares leave fp32."""

import pytest
import torch

import qk_rotary as qkr
import window_reference as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotary", [(64, 32), (93, 30), (256, 256)])  # rows in 16-byte units, and not
@pytest.mark.parametrize("scale", [1e19, 1e25, 1e30])
def test_large_rows(scale, d, rotary, interleaved, dtype):
    """sqrt(mean(x^2)) of finite rows is finite, and so are the rows over it."""
    g = torch.Generator().manual_seed(d)
    x, go = torch.randn(2, 3, 40, d, generator=g), torch.randn(2, 3, 40, d, generator=g)
    x[:, :, ::2] *= scale  # next to ordinary rows
    x, go = x.to(dtype), go.to(dtype)
    w = torch.rand(d, generator=g) + 0.5
    table = qkr.rotary_table(40, rotary)
    cos, sin = (t[None].expand(2, -1, -1) for t in table.chunk(2, -1))
    want = ref.norm_rotary(x, w, cos, sin, eps=1e-6, interleaved=interleaved, grad=go)
    value, bound = want["dw"]
    want["dw"] = value, bound + ref.half_step(torch.float32) * value.abs()
    want["dx"] = want["dx"][0], want["dx"][1] + 2.0 ** -149  # fp32's smallest step
    args = dict(q_weight=w.to(DEV), k_weight=w.to(DEV), interleaved=interleaved)
    x, go, table = x.to(DEV), go.to(DEV), table.to(DEV)
    y, _ = qkr.qk_norm_rotary(x, x[:, :1], table, **args)
    dx, _, dw, _ = qkr.qk_norm_rotary_backward(go, go[:, :1], x, x[:, :1], table, **args)
    for name, got in (("y", y), ("dx", dx), ("dw", dw)):
        assert ref.over(got, want[name]) <= 1.0, name
