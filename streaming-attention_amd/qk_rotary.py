"""RMS norm of every head's queries and keys and their position rotation in one pass: what goes in front of the
attention functions of this package, and keeps the logits bounded that their Taylor part needs small.

    qk_norm_rotary    q and k of [N,D], [B,H,N,D] or (one token of every stream) [S,H,D], differentiable
    rotary_table      cos and sin of a position's angles

Computed by hand-written HIP kernels on the inputs' ROCm device and its current stream; there is no CPU path.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

import _native
from sink_window_attention import (_STRIDES, _check_gpu, _differentiable_once, _like, _on, _refuse_capture, _refuse_tangents,
                                   _strides)

Tensor = torch.Tensor

__all__ = ["qk_norm_rotary", "qk_norm_rotary_backward", "rotary_table"]

MAX_DIM = 256
MAX_ROWS = 1 << 30
MAX_HEADS = 16384


def rotary_table(limit: int, rotary_dim: int, *, base: float = 10000.0,
                 device: Optional[Union[str, torch.device]] = None) -> Tensor:
    """float32 [limit, rotary_dim] for qk_norm_rotary: row p holds cos(p f_i), then sin(p f_i), for the rotary_dim / 2
    frequencies f_i = base^(-2 i / rotary_dim).  The angles are taken in float64: those of far positions keep their
    accuracy."""
    if limit < 1 or rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("limit must be positive and rotary_dim even")
    if not base > 0:
        raise ValueError("base must be positive")
    i = torch.arange(rotary_dim // 2, device=device, dtype=torch.float64)
    angle = torch.arange(limit, device=device, dtype=torch.float64)[:, None] * float(base) ** (-2.0 * i / max(rotary_dim, 1))
    return torch.cat([angle.cos(), angle.sin()], 1).float()


class _Call:
    """The checked arguments of a call, as the kernels take them."""

    def __init__(self, q, k, table, q_weight, k_weight, positions, eps, interleaved):
        _refuse_tangents(q, k, table, q_weight, k_weight)
        if q.ndim != k.ndim or q.ndim not in (2, 3, 4):
            raise ValueError("q and k must be [N,D], [S,H,D] or [B,H,N,D]")
        self.ndim = q.ndim
        (b, h, n, d), (kb, hk, kn, kd) = self.shape_of(q), self.shape_of(k)
        if kb != b or kn != n or kd != d:
            raise ValueError(f"k must match q but for its heads, got {tuple(k.shape)} and {tuple(q.shape)}")
        if q.dtype not in _native.DTYPE_CODES or k.dtype != q.dtype:
            raise ValueError("q and k must have one dtype of float32, bfloat16 and float16")
        if not 1 <= d <= MAX_DIM:
            raise ValueError(f"head widths must be 1 .. {MAX_DIM}, got {d}")
        if h > MAX_HEADS or hk > MAX_HEADS or b * n > MAX_ROWS:
            raise ValueError(f"at most {MAX_HEADS} heads and {MAX_ROWS} rows of a head are supported")
        if table.ndim != 2 or table.dtype != torch.float32 or table.shape[1] % 2 or table.shape[1] > d:
            raise ValueError(f"table must be float32 [limit, rotary_dim], rotary_dim even and at most {d}")
        if not 1 <= table.shape[0] <= 0x7FFFFFFF:
            raise ValueError("table must have 1 .. 2^31 - 1 positions")
        weights = [w for w in (q_weight, k_weight) if w is not None]
        for w in weights:
            if tuple(w.shape) != (d,) or w.dtype not in (q.dtype, torch.float32) or w.dtype != weights[0].dtype:
                raise ValueError(f"weights must be [{d}] of one dtype, q's or float32")
        if not (math.isfinite(eps) and eps >= 0):
            raise ValueError("eps must be finite and non-negative")
        if positions is not None:
            if positions.dtype not in (torch.int32, torch.int64):
                raise ValueError("positions must be int32 or int64")
            want = ((b,),) if self.ndim == 3 else ((n,), (b, n))
            if tuple(positions.shape) not in want:
                raise ValueError(f"positions must be {' or '.join(map(str, want))}, got {tuple(positions.shape)}")
            # element strides of batch and row
            if self.ndim == 3:
                self.pos_strides = (positions.stride(0), 0)
            elif positions.ndim == 1:
                self.pos_strides = (0, positions.stride(0))
            else:
                self.pos_strides = tuple(positions.stride())
        else:
            self.pos_strides = (0, 0)
        _check_gpu(q, k, table, q_weight, k_weight, positions)
        self.table = table.contiguous()
        self.positions, self.eps, self.interleaved = positions, float(eps), bool(interleaved)
        self.weight_code = _native.DTYPE_CODES[weights[0].dtype if weights else q.dtype]
        self.shape = (b, h, hk, n, d)

    def shape_of(self, x: Tensor) -> Tuple[int, int, int, int]:
        """x's shape as [B,H,N,D]."""
        s = x.shape
        return s if self.ndim == 4 else ((1, 1, *s) if self.ndim == 2 else (s[0], s[1], 1, s[2]))

    def strides(self, *tensors: Tensor):
        """The element strides of batch, head and row of every tensor, for the C ABI."""
        if self.ndim == 4:
            return _strides(*tensors)
        flat = ()
        for x in tensors:
            s = x.stride()
            flat += (0, 0, s[0]) if self.ndim == 2 else (s[0], s[1], 0)
        return _STRIDES[len(flat)](*flat)

    def tail(self, q_weight, k_weight):
        b, h, hk, n, d = self.shape
        pos = self.positions
        return (None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(),
                self.weight_code, self.table.data_ptr(), self.table.shape[0], self.table.shape[1], int(self.interleaved),
                _native.ptr(pos), int(pos is not None and pos.dtype == torch.int64), *self.pos_strides, self.eps)

    def forward(self, q, k, q_weight, k_weight):
        b, h, hk, n, d = self.shape
        q, k = _walkable(q), _walkable(k)
        qw, kw = (None if w is None else w.contiguous() for w in (q_weight, k_weight))
        yq, yk = _like(q), _like(k)
        if b * n and h + hk:
            with _on(q.device):
                st = _native.lib().sta_head_rotary(
                    q.data_ptr(), k.data_ptr(), _native.DTYPE_CODES[q.dtype], b, h, hk, n, d, self.strides(q, k),
                    *self.tail(qw, kw), yq.data_ptr(), yk.data_ptr(), _native.stream_handle(q.device))
            _native.check(st, "sta_head_rotary")
        return yq, yk

    def backward(self, gq, gk, q, k, q_weight, k_weight):
        b, h, hk, n, d = self.shape
        q, k, gq, gk = _walkable(q), _walkable(k), _walkable(gq), _walkable(gk)
        qw, kw = (None if w is None else w.contiguous() for w in (q_weight, k_weight))
        dq, dk = _like(q), _like(k)
        empty = not (b * n and h + hk)
        dw = [None if w is None else (torch.zeros_like(w) if empty or not heads else torch.empty_like(w))
              for w, heads in ((qw, h), (kw, hk))]
        if not empty:
            lib = _native.lib()
            nbytes = lib.sta_head_rotary_backward_bytes(b, h, hk, n, d)
            ws = q.new_empty(nbytes, dtype=torch.uint8)
            with _on(q.device):
                st = lib.sta_head_rotary_backward(
                    gq.data_ptr(), gk.data_ptr(), q.data_ptr(), k.data_ptr(), _native.DTYPE_CODES[q.dtype], b, h, hk,
                    n, d, self.strides(q, k, gq, gk), *self.tail(qw, kw), dq.data_ptr(), dk.data_ptr(),
                    _native.ptr(dw[0]), _native.ptr(dw[1]), ws.data_ptr(), nbytes, _native.stream_handle(q.device))
            _native.check(st, "sta_head_rotary_backward")
        return dq, dk, dw[0], dw[1]


def _walkable(x: Tensor) -> Tensor:
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


class _NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, positions, call):
        _refuse_capture()
        ctx.save_for_backward(q, k, q_weight, k_weight, table, positions)
        ctx.call = call
        return call.forward(q, k, q_weight, k_weight)

    @staticmethod
    @_differentiable_once
    def backward(ctx, gq, gk):
        _refuse_capture()
        q, k, q_weight, k_weight, _, _ = ctx.saved_tensors  # table and positions: checked to be as they were
        return (*ctx.call.backward(gq, gk, q, k, q_weight, k_weight), None, None, None)


def qk_norm_rotary(q: Tensor, k: Tensor, table: Tensor, *, q_weight: Optional[Tensor] = None,
                   k_weight: Optional[Tensor] = None, positions: Optional[Tensor] = None, eps: float = 1e-6,
                   interleaved: bool = False) -> Tuple[Tensor, Tensor]:
    """(q', k'): every head's row x becomes R(p) (x / sqrt(mean(x^2) + eps) * weight), R(p) turning the first
    table.shape[1] columns by the angles of the row's position, in pairs (i, i + R/2), or (2 i, 2 i + 1) if
    interleaved.  Differentiable in q, k and the weights.

    q [B,H,N,D] and k [B,Hkv,N,D] (any strides), [N,D] each, or one token of every stream, [S,H,D] and [S,Hkv,D];
    float32, bfloat16 or float16, D up to 256.  Weights [D] in that dtype or float32 (None: 1).
    positions: int32 or int64, [N] or [B,N] ([S] for [S,H,D]); None: 0 .. N-1.  A position outside the table makes its
    rows (and gradients) NaN; the table takes no gradient.  The results are dense in q's dtype.  Differentiable calls
    cannot be captured into a graph (RuntimeError); qk_norm_rotary_backward can.  Second and forward-mode derivatives are
    refused (RuntimeError)."""
    call = _Call(q, k, table, q_weight, k_weight, positions, eps, interleaved)
    if torch.is_grad_enabled() and table.requires_grad:
        raise ValueError("table takes no gradient: pass table.detach()")
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, q_weight, k_weight)):
        return _NormRotary.apply(q, k, q_weight, k_weight, table, positions, call)
    return call.forward(q, k, q_weight, k_weight)


@torch.no_grad()
def qk_norm_rotary_backward(q_grad: Tensor, k_grad: Tensor, q: Tensor, k: Tensor, table: Tensor, *,
                            q_weight: Optional[Tensor] = None, k_weight: Optional[Tensor] = None,
                            positions: Optional[Tensor] = None, eps: float = 1e-6, interleaved: bool = False
                            ) -> Tuple[Tensor, Tensor, Optional[Tensor], Optional[Tensor]]:
    """(dq, dk, dq_weight, dk_weight) of qk_norm_rotary's inputs from the gradients of its results, with the same
    settings; None for a weight that is None."""
    if q_grad.shape != q.shape or k_grad.shape != k.shape:
        raise ValueError("gradients must have their results' shapes")
    if q_grad.dtype != q.dtype or k_grad.dtype != q.dtype:
        raise ValueError("gradients must have q's dtype")
    call = _Call(q, k, table, q_weight, k_weight, positions, eps, interleaved)
    _refuse_tangents(q_grad, k_grad)
    _check_gpu(q, q_grad, k_grad)
    return call.backward(q_grad, k_grad, q, k, q_weight, k_weight)
