"""Exact attention for a batch whose sequences begin with one long prefix (a system prompt, a common document): the
prefix's keys and values are held and read once, and the sequences' own tokens follow them.

    shared_prefix_attention   the newest rows of every sequence, one (decode) or many (prefill), over the shared prefix
                              and the sequence's own tokens

Computed by hand-written HIP kernels on the inputs' ROCm device and its current stream; there is no CPU path.  Serving
only: results take no part in derivatives, and inputs that ask for one are refused.
"""

from __future__ import annotations

import struct
from typing import Optional, Tuple, Union

import torch

import _native
from sink_window_attention import (MAX_DIM, MAX_ROWS, _attention_scale, _check_dtype, _check_gpu, _check_lengths, _like, _on,
                                   _refuse_tangents, _widen)

Tensor = torch.Tensor

__all__ = ["shared_prefix_attention"]

_STRIDES = {n: struct.Struct(f"{3 * n}q").pack for n in (2, 5)}  # a third of a ctypes array's host time


def _walkable(*tensors: Tensor):
    """The tensors, those whose rows the kernels cannot walk as dense copies, and the element strides of batch (0 for a
    prefix [Hkv,P,D]), head and row of each, for the C ABI."""
    rows, strides = [], ()
    for x in tensors:
        s = x.stride()
        # rows of contiguous elements, at most 2^24 bytes apart
        if (s[-1] != 1 and x.shape[-1] != 1) or (s[-2] > 1 << 22 and s[-2] * x.element_size() > 1 << 24):
            x = x.clone(memory_format=torch.contiguous_format)  # strides of dimensions of one element too
            s = x.stride()
        rows.append(x)
        strides += s[:3] if len(s) == 4 else (0, *s[:2])
    return rows, _STRIDES[len(rows)](*strides)


def _refuse_gradients(*tensors: Tensor) -> None:
    """There is no backward pass; a result without one would be taken for a constant."""
    _refuse_tangents(*tensors)
    if torch.is_grad_enabled():
        for x in tensors:
            if x.requires_grad:
                raise RuntimeError("there is no backward pass: call under torch.no_grad(), or detach the inputs")


def _check_rows(q: Tensor, k: Tensor, names: str) -> None:
    """q [B,H,N,D] with own keys k [B,Hkv,M,D], N <= M."""
    if q.ndim != 4 or k.ndim != 4:
        raise ValueError(f"{names} must be [B,H,N,D]")
    (b, h, n, d), (kb, hk, m, kd) = q.shape, k.shape
    if kb != b or kd != d:
        raise ValueError(f"k must be [B,Hkv,M,D] like q [B,H,N,D], got {tuple(k.shape)} and {tuple(q.shape)}")
    if h != hk and (hk == 0 or h % hk != 0):
        raise ValueError(f"the query heads ({h}) must be a multiple of the key heads ({hk})")
    if not 1 <= d <= MAX_DIM:
        raise ValueError(f"key and value widths must be 1 .. {MAX_DIM}, got {d}")
    if n > m:
        raise ValueError(f"the {n} query rows are the last of the own tokens, of which there are {m}")
    if m > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows are supported")


def _check_prefix(prefix_k: Tensor, prefix_v: Tensor, batch: int, kv_heads: int, d: int, dv: int) -> Tuple[int, int]:
    """(prefixes, rows of each) of [G,Hkv,P,D], or of [Hkv,P,D]; shapes checked."""
    shape, values = prefix_k.shape, prefix_v.shape
    if len(shape) != len(values) or len(shape) not in (3, 4):
        raise ValueError("prefix_k and prefix_v must be [Hkv,P,D] or [G,Hkv,P,D]")
    sets, hk, p, pd = shape if len(shape) == 4 else (1, *shape)
    if hk != kv_heads or pd != d or values[-1] != dv or values[:-1] != shape[:-1]:
        raise ValueError(f"prefix_k and prefix_v must be [G,{kv_heads},P,{d}] and [G,{kv_heads},P,{dv}], got "
                         f"{tuple(prefix_k.shape)} and {tuple(prefix_v.shape)}")
    if sets == 0 or batch % sets != 0:
        raise ValueError(f"the {batch} sequences must be a multiple of the {sets} prefixes")
    if p > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows are supported")
    return sets, p


_workspaces: dict = {}  # bytes by shape, of the last few shapes


def _workspace(*shape) -> int:
    nbytes = _workspaces.get(shape)
    if nbytes is None:
        nbytes = _native.lib().sta_prefix_attention_bytes(*shape)
        if nbytes < 0:
            raise _native.NativeError("sta_prefix_attention_bytes refused the shape")
        if len(_workspaces) >= 64:
            _workspaces.clear()
        _workspaces[shape] = nbytes
    return nbytes


def _attention(q: Tensor, k: Tensor, v: Tensor, pk: Tensor, pv: Tensor, sets: int, p: int, lengths: Optional[Tensor],
               counts: Optional[Tensor], prefix_lengths: Optional[Tensor], scale: float,
               with_lse: bool) -> Tuple[Tensor, Optional[Tensor]]:
    b, h, n, d = q.shape
    hk, m, dv = k.shape[1], k.shape[2], v.shape[3]
    out = _like(q) if d == dv else q.new_empty((b, h, n, dv))
    lse = q.new_empty((b, h, n), dtype=torch.float32) if with_lse else None
    if out.numel() == 0:
        return out, lse
    if min(d, dv) * q.element_size() < 16:
        wide = _attention(*(_widen(x) for x in (q, k, v, pk, pv)), sets, p, lengths, counts, prefix_lengths, scale, with_lse)
        return out.copy_(wide[0][..., :dv]), wide[1]
    (q, k, v, pk, pv), strides = _walkable(q, k, v, pk, pv)
    code = _native.DTYPE_CODES[q.dtype]
    nbytes = _workspace(code, b, h, hk, sets, n, m, p, d, dv)
    with _on(q.device):
        ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        st = _native.lib().sta_prefix_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), pk.data_ptr(), pv.data_ptr(), code, b, h, hk, sets, n, m, p, d,
            dv, strides, scale, _native.ptr(lengths), _native.ptr(counts),
            _native.ptr(prefix_lengths), out.data_ptr(), _native.ptr(lse), _native.ptr(ws), nbytes,
            _native.stream_handle(q.device))
    _native.check(st, "sta_prefix_attention")
    return out, lse


def shared_prefix_attention(q: Tensor, k: Tensor, v: Tensor, prefix_k: Tensor, prefix_v: Tensor, *,
                            lengths: Optional[Tensor] = None, counts: Optional[Tensor] = None,
                            prefix_lengths: Optional[Tensor] = None, scale: Optional[float] = None,
                            with_lse: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Exact attention [B,H,N,Dv] of the newest rows of every sequence: each row sees the whole prefix and, causally, its
    sequence's own tokens.

    q [B,H,N,D]; own tokens k [B,Hkv,M,D], v [B,Hkv,M,Dv], the queries' among them (N <= M), H a multiple of Hkv; prefix_k
    [Hkv,P,D], prefix_v [Hkv,P,Dv] for all sequences, or [G,Hkv,P,D] and [G,Hkv,P,Dv] with sequence b reading prefix
    b // (B / G) (sequences of one prompt are neighbours); P may be 0.  float32, bfloat16 or float16, any strides, widths up
    to 128.  scale: 1/sqrt(D) when None.
    lengths: int32 [B] on the device, the own tokens of every sequence (None: M; values outside 0 .. M are taken as the
    nearest of them), whatever k and v hold behind them.  counts: int32 [B], the query rows of every sequence (None: N; at
    most its length): row i < counts[b] belongs to own token lengths[b] - counts[b] + i, so a decode step gives the
    lengths alone (counts of 1) and a padded batch of prompts the same tensor for both.  Output rows behind counts are zero.
    prefix_lengths: int32 [G], the rows of every prefix that count (None: P).
    with_lse: also log2 of every row's sum of weights, float32 [B,H,N] (0 behind counts), as received_attention takes
    them.  May be captured into a graph.  Inputs that ask for derivatives are refused (RuntimeError)."""
    _refuse_gradients(q, k, v, prefix_k, prefix_v)
    _check_rows(q, k, "q, k and v")
    b, _, _, d = q.shape
    if v.ndim != 4 or v.shape[:3] != k.shape[:3]:
        raise ValueError(f"v must be [B,Hkv,M,Dv] like k, got {tuple(v.shape)} and {tuple(k.shape)}")
    if not 1 <= v.shape[3] <= MAX_DIM:
        raise ValueError(f"key and value widths must be 1 .. {MAX_DIM}, got {v.shape[3]}")
    sets, p = _check_prefix(prefix_k, prefix_v, b, k.shape[1], d, v.shape[3])
    _check_dtype(q, k, v, prefix_k, prefix_v)
    lengths, counts = _check_lengths(lengths, b), _check_lengths(counts, b, "counts")
    prefix_lengths = _check_lengths(prefix_lengths, sets, "prefix_lengths")
    _check_gpu(q, k, v, prefix_k, prefix_v, lengths, counts, prefix_lengths)
    out, lse = _attention(q, k, v, prefix_k, prefix_v, sets, p, lengths, counts, prefix_lengths,
                          _attention_scale(scale, d), with_lse)
    return (out, lse) if with_lse else out
