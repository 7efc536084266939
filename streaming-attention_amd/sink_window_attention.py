"""Exact causal attention over a sliding window and the first tokens ("sinks"), next to the Taylor + coreset attention
of the other modules: the same bounded state, exact weights, and no view of what the window has passed.

    sink_window_causal_attention   [N,D] or [B,H,N,D] sequences, differentiable in q, k and v
    sink_window_forward, sink_window_backward
                                   the two passes by themselves, for captured graphs and programs without autograd

Row i sees the keys j <= i with i - j < window or j < sinks; window >= N is exact causal attention.  Key heads may be
shared: k and v may have fewer heads than q (a divisor).  Computed by hand-written HIP kernels on the inputs'
ROCm device and its current stream; there is no CPU path.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

import _native

Tensor = torch.Tensor

__all__ = ["sink_window_causal_attention", "sink_window_forward", "sink_window_backward"]

MAX_DIM = 128  # key and value widths of the kernels
MAX_ROWS = 1 << 30


def _attention_scale(scale: Optional[float], dim: int) -> float:
    s = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not math.isfinite(s):
        raise ValueError("scale must be finite")
    return s


def _check_tokens(window: int, sinks: int) -> Tuple[int, int]:
    for name, x in (("window", window), ("sinks", sinks)):
        if isinstance(x, bool) or not isinstance(x, int):
            raise ValueError(f"{name} must be an int, got {x!r}")
    if window < 1:
        raise ValueError("window must be at least 1")
    if sinks < 0:
        raise ValueError("sinks must be non-negative")
    return min(window, MAX_ROWS), min(sinks, MAX_ROWS)


def _check_gpu(**tensors: Optional[Tensor]) -> None:
    dev = None
    for name, x in tensors.items():
        if x is None:
            continue
        if not x.is_cuda:
            raise ValueError(f"HIP kernels require GPU (cuda/ROCm) tensors: {name} is on {x.device}")
        if dev is not None and x.device != dev:
            raise ValueError("all tensors must be on one device")
        dev = x.device


def _check_dtype(*tensors: Tensor) -> None:
    t = tensors[0].dtype
    if t not in _native.DTYPE_CODES:
        raise ValueError(f"dtype {t} is not supported (use float32, bfloat16 or float16)")
    if any(x.dtype != t for x in tensors):
        raise ValueError("all of q, k and v (and their gradients) must have one dtype")


def _heads_first(q: Tensor, k: Tensor, v: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    """[N,D] sequences as [1,1,N,D]; shapes checked."""
    if q.ndim != k.ndim or q.ndim != v.ndim or q.ndim not in (2, 4):
        raise ValueError("q/k/v must be [N,D] or [B,H,N,D]")
    if q.ndim == 2:
        q, k, v = q[None, None], k[None, None], v[None, None]
    b, h, n, d = q.shape
    if k.shape[0] != b or k.shape[2:] != (n, d):
        raise ValueError(f"k must be [B,Hkv,N,D] like q [B,H,N,D], got {tuple(k.shape)} and {tuple(q.shape)}")
    if v.shape[:3] != k.shape[:3]:
        raise ValueError(f"v must be [B,Hkv,N,Dv] like k, got {tuple(v.shape)} and {tuple(k.shape)}")
    if h != k.shape[1] and (k.shape[1] == 0 or h % k.shape[1] != 0):
        raise ValueError(f"the query heads ({h}) must be a multiple of the key heads ({k.shape[1]})")
    if not 1 <= d <= MAX_DIM or not 1 <= v.shape[3] <= MAX_DIM:
        raise ValueError(f"key and value widths must be 1 .. {MAX_DIM}, got {d} and {v.shape[3]}")
    if n > MAX_ROWS:
        raise ValueError(f"sequences of at most {MAX_ROWS} rows are supported")
    return q, k, v


def _check_lengths(lengths: Optional[Tensor], batch: int) -> Optional[Tensor]:
    if lengths is None:
        return None
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (batch,):
        raise ValueError(f"lengths must be an int32 tensor [{batch}]")
    return lengths.contiguous()


def _rows(x: Tensor) -> Tensor:
    """x itself where the kernels can walk its rows (contiguous last dimension), else a dense copy."""
    return x if x.stride(3) == 1 or x.shape[3] == 1 else x.contiguous()


def _dense(x: Tensor) -> Tensor:
    """x dense and on 16 bytes."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _strides(*tensors: Tensor):
    flat = [s for x in tensors for s in x.stride()[:3]]
    return (ctypes.c_int64 * len(flat))(*flat)


def _forward(q: Tensor, k: Tensor, v: Tensor, window: int, sinks: int, scale: float, lengths: Optional[Tensor],
             with_lse: bool) -> Tuple[Tensor, Optional[Tensor]]:
    b, h, n, d = q.shape
    dv = v.shape[3]
    out = torch.empty((b, h, n, dv), device=q.device, dtype=q.dtype)
    lse = torch.empty((b, h, n), device=q.device, dtype=torch.float32) if with_lse else None
    if out.numel() == 0:
        return out, lse
    q, k, v = _rows(q), _rows(k), _rows(v)
    with torch.cuda.device(q.device):
        st = _native.lib().sta_window_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _native.DTYPE_CODES[q.dtype], b, h, k.shape[1], n, d, dv,
            _strides(q, k, v), scale, window, sinks, _native.ptr(lengths), out.data_ptr(), _native.ptr(lse),
            _native.stream_handle(q.device))
    _native.check(st, "sta_window_attention")
    return out, lse


def _backward(grad: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, window: int, sinks: int,
              scale: float, lengths: Optional[Tensor]) -> Tuple[Tensor, Tensor, Tensor]:
    b, h, n, d = q.shape
    hk, dv = k.shape[1], v.shape[3]
    dq = torch.empty((b, h, n, d), device=q.device, dtype=q.dtype)
    dk = torch.empty((b, hk, n, d), device=q.device, dtype=q.dtype)
    dvo = torch.empty((b, hk, n, dv), device=q.device, dtype=q.dtype)
    if dq.numel() == 0:
        return dq, dk.zero_(), dvo.zero_()
    grad, q, k, v, out, lse = _rows(grad), _rows(q), _rows(k), _rows(v), _dense(out), lse.contiguous()
    lib = _native.lib()
    with torch.cuda.device(q.device):
        nbytes = lib.sta_window_backward_bytes(b, h, hk, n, d, dv, window, sinks)
        if nbytes < 0:
            raise _native.NativeError("sta_window_backward_bytes refused the shape")
        ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8)
        st = lib.sta_window_attention_backward(
            grad.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
            _native.DTYPE_CODES[q.dtype], b, h, hk, n, d, dv, _strides(q, k, v, grad), scale, window, sinks,
            _native.ptr(lengths), dq.data_ptr(), dk.data_ptr(), dvo.data_ptr(), ws.data_ptr(), nbytes,
            _native.stream_handle(q.device))
    _native.check(st, "sta_window_attention_backward")
    return dq, dk, dvo


def _refuse_capture() -> None:
    """The gradient of a leaf that also belongs to an eager graph joins that graph's stream; under capture that ends
    the process, so differentiable calls are refused there."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("differentiable calls cannot be captured into a graph: call the forward and backward "
                           "functions by themselves, or run under torch.no_grad()")


class _SinkWindow(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, lengths):
        _refuse_capture()
        out, lse = _forward(q, k, v, window, sinks, scale, lengths, True)
        ctx.save_for_backward(q, k, v, out, lse, lengths)
        ctx.settings = window, sinks, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _refuse_capture()
        q, k, v, out, lse, lengths = ctx.saved_tensors
        dq, dk, dv = _backward(grad, q, k, v, out, lse, *ctx.settings, lengths)
        return dq, dk, dv, None, None, None, None


def _checked(q, k, v, window, sinks, scale, lengths):
    window, sinks = _check_tokens(window, sinks)
    q4, k4, v4 = _heads_first(q, k, v)
    _check_dtype(q4, k4, v4)
    lengths = _check_lengths(lengths, q4.shape[0])
    _check_gpu(q=q4, k=k4, v=v4, lengths=lengths)
    return q4, k4, v4, window, sinks, _attention_scale(scale, q4.shape[3]), lengths


def sink_window_causal_attention(q: Tensor, k: Tensor, v: Tensor, *, window: int, sinks: int = 4,
                                 scale: Optional[float] = None, lengths: Optional[Tensor] = None) -> Tensor:
    """Exact causal attention of every row over the last `window` tokens (its own among them) and the first `sinks`
    ones, for [N,D] and [B,H,N,D] tensors (any strides); differentiable in q, k and v.

    q [B,H,N,D], k [B,Hkv,N,D], v [B,Hkv,N,Dv], H a multiple of Hkv; float32, bfloat16 or float16, widths up to 128.
    scale: 1/sqrt(D) when None.  lengths: int32 [B] on the device, the rows of every sequence of a padded batch;
    output rows behind them are zero and take no part in the gradients, whatever the padding holds.
    The output has q's dtype.  Differentiable calls cannot be captured into a graph (RuntimeError); use
    sink_window_forward and sink_window_backward there."""
    q4, k4, v4, window, sinks, s, lengths = _checked(q, k, v, window, sinks, scale, lengths)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out = _SinkWindow.apply(q4, k4, v4, window, sinks, s, lengths)
    else:
        out = _forward(q4, k4, v4, window, sinks, s, lengths, False)[0]
    return out[0, 0] if q.ndim == 2 else out


@torch.no_grad()
def sink_window_forward(q: Tensor, k: Tensor, v: Tensor, *, window: int, sinks: int = 4,
                        scale: Optional[float] = None, lengths: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """sink_window_causal_attention's output and its row statistics [B,H,N] ([N] for [N,D] tensors): log2 of every
    row's sum of weights, float32, as sink_window_backward takes them.  May be captured into a graph."""
    q4, k4, v4, window, sinks, s, lengths = _checked(q, k, v, window, sinks, scale, lengths)
    out, lse = _forward(q4, k4, v4, window, sinks, s, lengths, True)
    return (out[0, 0], lse[0, 0]) if q.ndim == 2 else (out, lse)


@torch.no_grad()
def sink_window_backward(grad: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, *, window: int,
                         sinks: int = 4, scale: Optional[float] = None,
                         lengths: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """(dq, dk, dv) of sink_window_causal_attention for the output's gradient `grad`, from the inputs and results of
    sink_window_forward with the same settings.  May be captured into a graph."""
    q4, k4, v4, window, sinks, s, lengths = _checked(q, k, v, window, sinks, scale, lengths)
    if q.ndim == 2:
        if grad.ndim != 2 or out.ndim != 2 or lse.ndim != 1:
            raise ValueError("for [N,D] inputs grad and out must be [N,Dv] and lse [N]")
        grad, out, lse = grad[None, None], out[None, None], lse[None, None]
    want = (*q4.shape[:3], v4.shape[3])
    if tuple(grad.shape) != want or tuple(out.shape) != want or tuple(lse.shape) != want[:3]:
        raise ValueError(f"grad and out must be {want} and lse {want[:3]}")
    _check_dtype(q4, grad, out)
    if lse.dtype != torch.float32:
        raise ValueError("lse must be float32")
    _check_gpu(q=q4, grad=grad, out=out, lse=lse)
    dq, dk, dv = _backward(grad, q4, k4, v4, out, lse, window, sinks, s, lengths)
    return (dq[0, 0], dk[0, 0], dv[0, 0]) if q.ndim == 2 else (dq, dk, dv)
