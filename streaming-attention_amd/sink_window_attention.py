"""Exact causal attention over a sliding window and the first tokens ("sinks"), next to the Taylor + coreset attention
of the other modules: the same bounded state, exact weights, and no view of what the window has passed.

    sink_window_causal_attention   [N,D] or [B,H,N,D] sequences, differentiable in q, k and v
    sink_window_forward, sink_window_backward
                                   the two passes by themselves, for captured graphs and programs without autograd
    SinkWindowStreamingAttention   its serving form: a cache of sinks and a ring of `window` tokens for streams in
                                   lockstep, in the element type or in 4 bits, and one query a head at a time

Row i sees the keys j <= i with i - j < window or j < sinks; window >= N is exact causal attention.  Key heads may be
shared: k and v may have fewer heads than q (a divisor).  Computed by hand-written HIP kernels on the inputs'
ROCm device and its current stream; there is no CPU path.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
from typing import Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad

import _native

Tensor = torch.Tensor

__all__ = ["SinkWindowStreamingAttention", "sink_window_backward", "sink_window_causal_attention",
           "sink_window_forward"]

MAX_DIM = 128  # key and value widths of the kernels
MAX_ROWS = 1 << 30


def _attention_scale(scale: Optional[float], dim: int) -> float:
    s = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not math.isfinite(s):
        raise ValueError("scale must be finite")
    return s


def _check_tokens(window: int, sinks: int) -> Tuple[int, int]:
    if type(window) is not int or type(sinks) is not int:
        for name, x in (("window", window), ("sinks", sinks)):
            if isinstance(x, bool) or not isinstance(x, int):
                raise ValueError(f"{name} must be an int, got {x!r}")
    if window < 1:
        raise ValueError("window must be at least 1")
    if sinks < 0:
        raise ValueError("sinks must be non-negative")
    return min(window, MAX_ROWS), min(sinks, MAX_ROWS)


def _check_gpu(*tensors: Optional[Tensor]) -> None:
    dev = tensors[0].device
    if dev.type != "cuda":
        raise ValueError(f"HIP kernels require GPU (cuda/ROCm) tensors, got one on {dev}")
    for x in tensors:
        if x is not None and x.device != dev:
            raise ValueError(f"all tensors must be on one device, got {x.device} and {dev}")


def _check_dtype(*tensors: Tensor) -> None:
    t = tensors[0].dtype
    if t not in _native.DTYPE_CODES:
        raise ValueError(f"dtype {t} is not supported (use float32, bfloat16 or float16)")
    for x in tensors:
        if x.dtype != t:
            raise ValueError("all of q, k and v (and their gradients) must have one dtype")


def _four(x: Tensor) -> Tensor:
    """[N,D] as [1,1,N,D]."""
    return x.view(1, 1, *x.shape)


def _heads_first(q: Tensor, k: Tensor, v: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    """[N,D] sequences as [1,1,N,D]; shapes checked."""
    if q.ndim != k.ndim or q.ndim != v.ndim or q.ndim not in (2, 4):
        raise ValueError("q/k/v must be [N,D] or [B,H,N,D]")
    if q.ndim == 2:
        q, k, v = _four(q), _four(k), _four(v)
    (b, h, n, d), (kb, hk, kn, kd), (vb, vh, vn, dv) = q.shape, k.shape, v.shape
    if kb != b or kn != n or kd != d:
        raise ValueError(f"k must be [B,Hkv,N,D] like q [B,H,N,D], got {tuple(k.shape)} and {tuple(q.shape)}")
    if vb != kb or vh != hk or vn != kn:
        raise ValueError(f"v must be [B,Hkv,N,Dv] like k, got {tuple(v.shape)} and {tuple(k.shape)}")
    if h != hk and (hk == 0 or h % hk != 0):
        raise ValueError(f"the query heads ({h}) must be a multiple of the key heads ({hk})")
    if not 1 <= d <= MAX_DIM or not 1 <= dv <= MAX_DIM:
        raise ValueError(f"key and value widths must be 1 .. {MAX_DIM}, got {d} and {dv}")
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
    """x itself where the kernels can walk its rows (contiguous last dimension, rows at most 2^24 bytes apart), else a
    dense copy."""
    strides = x.stride()
    if strides[2] * x.element_size() <= 1 << 24 and (strides[3] == 1 or x.shape[3] == 1):
        return x
    return x.clone(memory_format=torch.contiguous_format)  # strides of dimensions of one element too


def _dense(x: Tensor) -> Tensor:
    """x dense and on 16 bytes."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _like(x: Tensor) -> Tensor:
    """A dense tensor like x, its values not set (half the host time of torch.empty)."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


_STRIDES = {n: ctypes.c_int64 * n for n in (6, 9, 12)}


def _strides(*tensors: Tensor):
    """The element strides of batch, head and row of every tensor, for the C ABI."""
    flat = ()
    for x in tensors:
        flat += x.stride()[:3]
    return _STRIDES[len(flat)](*flat)


_here = contextlib.nullcontext()


def _on(device: torch.device):
    """The device as the current one (nothing to do where it is: 5 us of a small call's host time)."""
    return _here if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _widen(x: Tensor) -> Tensor:
    """x with zero columns up to the 16 bytes that the kernels' rows have at least."""
    short = 16 // x.element_size() - x.shape[3]
    return torch.nn.functional.pad(x, (0, short)) if short > 0 else x


def _forward(q: Tensor, k: Tensor, v: Tensor, window: int, sinks: int, scale: float, lengths: Optional[Tensor],
             with_lse: bool, with_rest: bool) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor]]:
    b, h, n, d = q.shape
    dv = v.shape[3]
    out = _like(q) if d == dv else q.new_empty((b, h, n, dv))
    rest = _like(out) if with_rest and q.dtype != torch.float32 else None
    lse = q.new_empty((b, h, n), dtype=torch.float32) if with_lse else None
    if out.numel() == 0:
        return out, rest, lse
    if min(d, dv) * q.element_size() < 16:
        wide = _forward(_widen(q), _widen(k), _widen(v), window, sinks, scale, lengths, with_lse, with_rest)
        return out.copy_(wide[0][..., :dv]), None if rest is None else rest.copy_(wide[1][..., :dv]), wide[2]
    q, k, v = _rows(q), _rows(k), _rows(v)
    with _on(q.device):
        st = _native.lib().sta_window_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _native.DTYPE_CODES[q.dtype], b, h, k.shape[1], n, d, dv,
            _strides(q, k, v), scale, window, sinks, _native.ptr(lengths), out.data_ptr(), _native.ptr(rest),
            _native.ptr(lse), _native.stream_handle(q.device))
    _native.check(st, "sta_window_attention")
    return out, rest, lse


def _backward(grad: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, rest: Optional[Tensor], lse: Tensor,
              window: int, sinks: int, scale: float, lengths: Optional[Tensor]) -> Tuple[Tensor, Tensor, Tensor]:
    b, h, n, d = q.shape
    hk, dv = k.shape[1], v.shape[3]
    dq, dk, dvo = _like(q), _like(k), _like(v)
    if dq.numel() == 0:
        return dq, dk.zero_(), dvo.zero_()
    if min(d, dv) * q.element_size() < 16:
        wide = _backward(*(_widen(x) for x in (grad, q, k, v, out)), None if rest is None else _widen(rest), lse, window,
                         sinks, scale, lengths)
        return dq.copy_(wide[0][..., :d]), dk.copy_(wide[1][..., :d]), dvo.copy_(wide[2][..., :dv])
    grad, q, k, v, out, lse = _rows(grad), _rows(q), _rows(k), _rows(v), _dense(out), lse.contiguous()
    rest = None if rest is None else _dense(rest)
    lib = _native.lib()
    with _on(q.device):
        nbytes = lib.sta_window_backward_bytes(_native.DTYPE_CODES[q.dtype], b, h, hk, n, d, dv, window, sinks)
        if nbytes < 0:
            raise _native.NativeError("sta_window_backward_bytes refused the shape")
        ws = q.new_empty(nbytes, dtype=torch.uint8)
        st = lib.sta_window_attention_backward(
            grad.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _native.ptr(rest), lse.data_ptr(),
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


def _refuse_tangents(*tensors: Optional[Tensor]) -> None:
    """The operators have no forward-mode derivative; a result without one would be taken for a constant."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # no tangents anywhere (five tensors' looks take 0.7 us)
        return
    for x in tensors:
        if x is not None and forward_ad.unpack_dual(x).tangent is not None:
            raise RuntimeError("forward-mode derivatives are not supported: use the backward pass")


def _differentiable_once(backward):
    """once_differentiable where a graph of the gradients is asked for; without one its wrapping costs 5 us a call."""
    once = torch.autograd.function.once_differentiable(backward)
    return lambda ctx, *grads: once(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)


class _SinkWindow(torch.autograd.Function):
    """[N,D] tensors become [1,1,N,D] in here: the gradients of views taken outside are launches of their own (100 us of
    a small training step)."""

    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, lengths):
        _refuse_capture()
        ctx.flat = q.ndim == 2
        q4, k4, v4 = (_four(q), _four(k), _four(v)) if ctx.flat else (q, k, v)
        out, rest, lse = _forward(q4, k4, v4, window, sinks, scale, lengths, True, True)
        if ctx.flat:
            out = out.view(out.shape[2:])
        ctx.save_for_backward(q, k, v, out, rest, lse, lengths)
        ctx.settings = window, sinks, scale
        return out

    @staticmethod
    @_differentiable_once
    def backward(ctx, grad):
        _refuse_capture()
        q, k, v, out, rest, lse, lengths = ctx.saved_tensors
        if ctx.flat:
            grad, q, k, v, out = (_four(x) for x in (grad, q, k, v, out))
        grads = _backward(grad, q, k, v, out, rest, lse, *ctx.settings, lengths)
        if ctx.flat:
            grads = (x.view(x.shape[2:]) for x in grads)
        return *grads, None, None, None, None


def _checked(q, k, v, window, sinks, scale, lengths):
    window, sinks = _check_tokens(window, sinks)
    _refuse_tangents(q, k, v)
    q4, k4, v4 = _heads_first(q, k, v)
    _check_dtype(q4, k4, v4)
    lengths = _check_lengths(lengths, q4.shape[0])
    _check_gpu(q4, k4, v4, lengths)
    return q4, k4, v4, window, sinks, _attention_scale(scale, q4.shape[3]), lengths


def sink_window_causal_attention(q: Tensor, k: Tensor, v: Tensor, *, window: int, sinks: int = 4,
                                 scale: Optional[float] = None, lengths: Optional[Tensor] = None) -> Tensor:
    """Exact causal attention of every row over the last `window` tokens (its own among them) and the first `sinks`
    ones, for [N,D] and [B,H,N,D] tensors (any strides); differentiable in q, k and v.

    q [B,H,N,D], k [B,Hkv,N,D], v [B,Hkv,N,Dv], H a multiple of Hkv; float32, bfloat16 or float16, widths up to 128.
    scale: 1/sqrt(D) when None.  lengths: int32 [B] on the device, the rows of every sequence of a padded batch
    (values outside 0 .. N are taken as the nearest of them); output rows behind them are zero and take no part in the
    gradients, whatever the padding holds.
    The output has q's dtype; with gradients a 16-bit call also keeps what the output's rounding left.  Differentiable
    calls cannot be captured into a graph (RuntimeError); use sink_window_forward and sink_window_backward there.  Second
    and forward-mode derivatives are refused (RuntimeError)."""
    q4, k4, v4, window, sinks, s, lengths = _checked(q, k, v, window, sinks, scale, lengths)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _SinkWindow.apply(q, k, v, window, sinks, s, lengths)
    out = _forward(q4, k4, v4, window, sinks, s, lengths, False, False)[0]
    return out[0, 0] if q.ndim == 2 else out


@torch.no_grad()
def sink_window_forward(q: Tensor, k: Tensor, v: Tensor, *, window: int, sinks: int = 4,
                        scale: Optional[float] = None, lengths: Optional[Tensor] = None,
                        with_rest: bool = False) -> Tuple[Tensor, ...]:
    """sink_window_causal_attention's output and its row statistics [B,H,N] ([N] for [N,D] tensors): log2 of every
    row's sum of weights, float32, as sink_window_backward takes them.  with_rest: also what the output's rounding left,
    like the output (None for float32), which keeps that rounding out of the gradients.  May be captured into a graph."""
    q4, k4, v4, window, sinks, s, lengths = _checked(q, k, v, window, sinks, scale, lengths)
    out, rest, lse = _forward(q4, k4, v4, window, sinks, s, lengths, True, with_rest)
    if q.ndim == 2:
        out, rest, lse = out[0, 0], None if rest is None else rest[0, 0], lse[0, 0]
    return (out, lse, rest) if with_rest else (out, lse)


@torch.no_grad()
def sink_window_backward(grad: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, *, window: int,
                         sinks: int = 4, scale: Optional[float] = None, lengths: Optional[Tensor] = None,
                         rest: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """(dq, dk, dv) of sink_window_causal_attention for the output's gradient `grad`, from the inputs and results of
    sink_window_forward with the same settings (rest: its third result, if it was asked for).  May be captured into a
    graph."""
    q4, k4, v4, window, sinks, s, lengths = _checked(q, k, v, window, sinks, scale, lengths)
    if q.ndim == 2:
        if grad.ndim != 2 or out.ndim != 2 or lse.ndim != 1:
            raise ValueError("for [N,D] inputs grad and out must be [N,Dv] and lse [N]")
        grad, out, lse = grad[None, None], out[None, None], lse[None, None]
        rest = None if rest is None else rest[None, None]
    want = (*q4.shape[:3], v4.shape[3])
    if tuple(grad.shape) != want or tuple(out.shape) != want or tuple(lse.shape) != want[:3]:
        raise ValueError(f"grad and out must be {want} and lse {want[:3]}")
    _check_dtype(q4, grad, out)
    _refuse_tangents(grad, out, lse, rest)
    if rest is not None and (q4.dtype == torch.float32 or rest.shape != out.shape or rest.dtype != out.dtype):
        raise ValueError("rest must be like out, and None for float32")
    if lse.dtype != torch.float32:
        raise ValueError("lse must be float32")
    _check_gpu(q4, grad, out, lse, rest)
    dq, dk, dv = _backward(grad, q4, k4, v4, out, rest, lse, window, sinks, s, lengths)
    return (dq[0, 0], dk[0, 0], dv[0, 0]) if q.ndim == 2 else (dq, dk, dv)


class SinkWindowStreamingAttention:
    """Exact streaming attention over the last `window` tokens and the first `sinks` ones of every stream: a cache
    of sinks + window tokens a stream and key head, whatever the streams' length.

    `step(q, k, v)` takes one token of every stream: keys [S,Hkv,dim], values [S,Hkv,value_dim], queries [S,H,dim] ->
    [S,H,value_dim], H a multiple of Hkv; `update` and `query` are its two halves, `extend` takes prompts in bulk and
    `prefill` answers them too.  Queries see every token held, their own step's among them.

    dtype (float32, bfloat16, float16) is that of inputs and outputs; storage None keeps the cache in it, "fp4" in 4
    bits: blocks of 32 columns of a token as 4-bit floats (0, 0.5, 1, 1.5, 2, 3, 4, 6 and signs) times a power of two,
    4.25 bits a value (a block with a value that is not finite becomes NaN).  Sums and softmax statistics are fp32.
    A token held with an infinity or NaN makes the outputs that it reaches NaN or infinite until it leaves.

    Calls run on the device's current stream and may be captured into graphs (replays advance the state like
    calls); calls on one object have to be ordered, by one stream or by events.  Results take no part in derivatives."""

    def __init__(self, dim: int, value_dim: int, *, streams: int = 1, heads: int = 1, kv_heads: Optional[int] = None,
                 window: int, sinks: int = 4, scale: Optional[float] = None,
                 dtype: torch.dtype = torch.float32, storage: Optional[str] = None,
                 device: Optional[Union[str, torch.device]] = None) -> None:
        kv_heads = heads if kv_heads is None else kv_heads
        if streams < 1 or heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError("streams and heads must be positive and heads a multiple of kv_heads")
        if not 1 <= dim <= MAX_DIM or not 1 <= value_dim <= MAX_DIM:
            raise ValueError(f"key and value widths must be 1 .. {MAX_DIM}, got {dim} and {value_dim}")
        self.window, self.sinks = _check_tokens(window, sinks)
        if window + sinks > MAX_ROWS:
            raise ValueError(f"a cache of at most {MAX_ROWS} tokens is supported")
        if dtype not in _native.DTYPE_CODES:
            raise ValueError(f"dtype {dtype} is not supported (use float32, bfloat16 or float16)")
        if storage not in (None, "fp4"):
            raise ValueError("storage must be None or 'fp4'")
        self.scale = _attention_scale(scale, dim)
        self.dim, self.value_dim, self.streams, self.heads, self.kv_heads = dim, value_dim, streams, heads, kv_heads
        self.dtype, self.storage = dtype, storage
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise ValueError(f"HIP kernels require a GPU (cuda/ROCm) device, got {dev}")
        if not torch.cuda.is_available():
            raise RuntimeError("streaming-attention HIP kernels need a ROCm GPU; none is visible")
        self.device = torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)
        self._code = _native.DTYPE_CODES[dtype]
        self._store = self._code if storage is None else _native.STORAGE_FP4
        sizes = (ctypes.c_int64 * 4)()
        _native.check(_native.lib().sta_ring_layout(self._code, self._store, streams, kv_heads, dim, value_dim,
                                                    self.window, self.sinks, sizes), "sta_ring_layout")
        self._cache = [torch.zeros(n, device=self.device, dtype=torch.uint8) if n else None for n in sizes]
        self._counts = torch.zeros((streams, kv_heads), device=self.device, dtype=torch.int32)
        self._state = (*(_native.ptr(x) for x in self._cache), self._counts.data_ptr())
        self._shapes = {"query": (streams, heads, dim), "key": (streams, kv_heads, dim),
                        "value": (streams, kv_heads, value_dim)}
        self._dense = _STRIDES[6](heads * dim, dim, kv_heads * dim, dim, kv_heads * value_dim, value_dim)
        self._bytes = _native.lib().sta_ring_attention_bytes(streams, heads, kv_heads, dim, value_dim, self.window,
                                                             self.sinks)
        self._used = False  # a call has changed the state, or has been captured to

    @property
    def lengths(self) -> Tensor:
        """int32 [S] on the device: tokens that each stream has taken, a view of the state to be read only.  A count
        that would pass 2^31 - 1 goes back by whole windows; outputs do not depend on that."""
        return self._counts[:, 0]

    def _rows(self, x: Tensor, want: Tuple[int, ...], what: str) -> Tensor:
        if x.shape != want:
            raise ValueError(f"{what} must be {list(want)}, got {list(x.shape)}")
        if x.dtype != self.dtype or x.device != self.device:
            x = x.detach().to(device=self.device, dtype=self.dtype)
        return x if x.is_contiguous() or x.stride(-1) == 1 or x.shape[-1] == 1 else x.detach().contiguous()

    def _attend(self, q: Tensor, k: Optional[Tensor], v: Optional[Tensor]) -> Tensor:
        out = _like(q) if self.dim == self.value_dim else q.new_empty((self.streams, self.heads, self.value_dim))
        ws = q.new_empty(self._bytes, dtype=torch.uint8) if self._bytes else None
        if q.is_contiguous() and (k is None or (k.is_contiguous() and v.is_contiguous())):
            strides = self._dense
        else:
            none = (0, 0)
            strides = _STRIDES[6](*q.stride()[:2], *(none if k is None else k.stride()[:2]),
                                  *(none if v is None else v.stride()[:2]))
        with _on(self.device):
            st = _native.lib().sta_ring_attention(
                q.data_ptr(), _native.ptr(k), _native.ptr(v), self._code, self._store, self.streams, self.heads,
                self.kv_heads, self.dim, self.value_dim, strides, self.scale, self.window, self.sinks,
                *self._state, out.data_ptr(), _native.ptr(ws), self._bytes, _native.stream_handle(self.device))
        _native.check(st, "sta_ring_attention")
        return out

    def step(self, query: Tensor, key: Tensor, value: Tensor) -> Tensor:
        """One token of every stream into the cache, then one query a head: update(key, value); query(query)."""
        shapes = self._shapes
        q = self._rows(query, shapes["query"], "query")
        k = self._rows(key, shapes["key"], "key")
        v = self._rows(value, shapes["value"], "value")
        self._used = True
        return self._attend(q, k, v)

    def query(self, query: Tensor) -> Tensor:
        """Attention of one query a head over the tokens held; zero for a stream that holds none."""
        return self._attend(self._rows(query, self._shapes["query"], "query"), None, None)

    def update(self, key: Tensor, value: Tensor) -> None:
        """One token of every stream into the cache."""
        k = self._rows(key, self._shapes["key"], "key")
        v = self._rows(value, self._shapes["value"], "value")
        self._extend(k[:, :, None], v[:, :, None], None)

    def _extend(self, k: Tensor, v: Tensor, counts: Optional[Tensor]) -> None:
        if k.shape[2] == 0:
            return
        self._used = True
        with _on(self.device):
            st = _native.lib().sta_ring_extend(
                k.data_ptr(), v.data_ptr(), self._code, self._store, self.streams, self.kv_heads, k.shape[2], self.dim,
                self.value_dim, _strides(k, v), self.window, self.sinks, _native.ptr(counts),
                *self._state, _native.stream_handle(self.device))
        _native.check(st, "sta_ring_extend")

    def _prompt(self, keys: Tensor, values: Tensor, counts: Optional[Tensor]):
        rows = keys.shape[2] if keys.ndim == 4 else 0
        if rows > MAX_ROWS:
            raise ValueError(f"at most {MAX_ROWS} rows at a time are supported")
        k = self._rows(keys, (self.streams, self.kv_heads, rows, self.dim), "keys")
        v = self._rows(values, (self.streams, self.kv_heads, rows, self.value_dim), "values")
        if counts is not None:
            counts = _check_lengths(counts, self.streams)
            if counts.device != self.device:
                raise ValueError("counts must be on the object's device")
        return k, v, counts

    def extend(self, keys: Tensor, values: Tensor, *, counts: Optional[Tensor] = None) -> None:
        """update() with the rows of keys [S,Hkv,P,dim] and values [S,Hkv,P,value_dim] in bulk; counts: int32 [S] on
        the device, the rows of every stream that are tokens (None: all P; values outside 0 .. P are taken as the
        nearest of them)."""
        self._extend(*self._prompt(keys, values, counts))

    @torch.no_grad()
    def prefill(self, q: Tensor, k: Tensor, v: Tensor, *, counts: Optional[Tensor] = None) -> Tensor:
        """Outputs [S,H,P,value_dim] of a prompt's rows (sink_window_causal_attention, on the rows as given), leaving
        the state after it.  Only on an empty state: on an object that has been used the call waits for the device to
        see that it is.  A captured call cannot see that; it empties the state itself, so that every replay starts there."""
        with _on(self.device):
            captured = torch.cuda.is_current_stream_capturing()
        # the device's counts decide: replays of captured calls change them unseen
        if not captured and self._used and bool(self._counts.any()):
            raise ValueError("prefill starts from an empty state; use step() / extend() afterwards")
        k, v, counts = self._prompt(k, v, counts)
        q = self._rows(q, (self.streams, self.heads, k.shape[2], self.dim), "q")
        out = sink_window_causal_attention(q, k, v, window=self.window, sinks=self.sinks, scale=self.scale,
                                           lengths=counts)
        if captured:
            self._counts.zero_()
        self._extend(k, v, counts)
        return out

    def reset(self, streams: Optional[Sequence[int]] = None) -> None:
        """Forgets every token of all streams, or of the given ones (new sequences start there)."""
        if streams is None:
            self._counts.zero_()
            return
        streams = list(streams)
        for i in streams:
            if not 0 <= i < self.streams:
                raise ValueError(f"there is no stream {i}")
        for i in streams:
            self._counts[i].zero_()

    def items(self) -> Tuple[Tensor, Tensor, Tensor]:
        """(keys [S,Hkv,sinks + window,dim], values [S,Hkv,sinks + window,value_dim], positions int32
        [S,sinks + window]) as the cache holds them, in the order of its slots; zero and -1 where no token is."""
        slots = self.sinks + self.window
        positions = self._counts.new_empty((self.streams, slots))
        keys = positions.new_empty((self.streams, self.kv_heads, slots, self.dim), dtype=self.dtype)
        values = (_like(keys) if self.dim == self.value_dim else
                  keys.new_empty((self.streams, self.kv_heads, slots, self.value_dim)))
        with _on(self.device):
            st = _native.lib().sta_ring_items(
                self._code, self._store, self.streams, self.kv_heads, self.dim, self.value_dim, self.window, self.sinks,
                *self._state, keys.data_ptr(), values.data_ptr(), positions.data_ptr(),
                _native.stream_handle(self.device))
        _native.check(st, "sta_ring_items")
        return keys, values, positions

    def state_size_bytes(self) -> int:
        """Device bytes of the cache."""
        return sum(x.numel() for x in self._cache if x is not None) + 4 * self._counts.numel()

    def state_dict_settings(self) -> dict:
        return {"dim": self.dim, "value_dim": self.value_dim, "streams": self.streams, "heads": self.heads,
                "kv_heads": self.kv_heads, "window": self.window, "sinks": self.sinks, "scale": self.scale,
                "dtype": str(self.dtype), "storage": self.storage}

    def state_dict(self) -> dict:
        """The state for a later resume: plain tensors on the host and Python scalars."""
        return {"attention": self.state_dict_settings(), "counts": self._counts.cpu(),
                "cache": [None if x is None else x.cpu() for x in self._cache]}

    def load_state_dict(self, state: dict) -> None:
        """Resume from state_dict() of an object built with the same settings (the device may differ)."""
        mine = self.state_dict_settings()
        if state["attention"] != mine:
            raise ValueError(f"state settings {state['attention']} do not match this object's {mine}")
        if len(state["cache"]) != len(self._cache):
            raise ValueError("the state's tensors do not match this object's")
        for x, y in zip((self._counts, *self._cache), (state["counts"], *state["cache"])):
            if (x is None) != (y is None) or (x is not None and (x.shape != y.shape or x.dtype != y.dtype)):
                raise ValueError("the state's tensors do not match this object's")
        if bool((state["counts"] < 0).any()):
            raise ValueError("the state's counts must not be negative")
        for x, y in zip((self._counts, *self._cache), (state["counts"], *state["cache"])):
            if x is not None:
                x.copy_(y)
        self._used = True
