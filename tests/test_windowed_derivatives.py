"""Forward-mode tangents at the windowed operators: refused, and not dropped."""

import pytest
import torch
from torch.autograd import forward_ad

import qk_rotary as qkr
import sink_window_attention as swa


def x(*shape):
    return torch.zeros(*shape)


@pytest.mark.parametrize("which", range(3))
def test_attention_refuses_tangents(which):
    args = [x(4, 8), x(4, 8), x(4, 8)]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], x(4, 8))
        for f in (swa.sink_window_causal_attention, swa.sink_window_forward):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(*args, window=2)


@pytest.mark.parametrize("which", range(6))
def test_backward_refuses_tangents(monkeypatch, which):
    monkeypatch.setattr(swa, "_check_gpu", lambda *a: None)
    args = [x(4, 8), x(4, 8), x(4, 8), x(4, 8), x(4, 8), x(4)]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], x(*args[which].shape))
        with pytest.raises(RuntimeError, match="forward-mode"):
            swa.sink_window_backward(*args, window=2)


@pytest.mark.parametrize("which", range(5))
def test_rotary_refuses_tangents(which):
    args = [x(4, 8), x(4, 8), x(4, 8), x(8), x(8)]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], x(*args[which].shape))
        q, k, table, qw, kw = args
        with pytest.raises(RuntimeError, match="forward-mode"):
            qkr.qk_norm_rotary(q, k, table, q_weight=qw, k_weight=kw)
        with pytest.raises(RuntimeError, match="forward-mode"):
            qkr.qk_norm_rotary_backward(x(4, 8), x(4, 8), q, k, table, q_weight=qw, k_weight=kw)


@pytest.mark.parametrize("which", range(2))
def test_rotary_backward_refuses_tangents_of_gradients(monkeypatch, which):
    monkeypatch.setattr(qkr, "_check_gpu", lambda *a: None)
    grads = [x(4, 8), x(4, 8)]
    with forward_ad.dual_level():
        grads[which] = forward_ad.make_dual(grads[which], x(4, 8))
        with pytest.raises(RuntimeError, match="forward-mode"):
            qkr.qk_norm_rotary_backward(*grads, x(4, 8), x(4, 8), x(4, 8))
