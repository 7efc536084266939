"""Exact attention over a bounded cache that keeps the tokens which received the most attention, next to the Taylor +
coreset state and the window with sinks of the other modules: the last tokens, and of the older ones those whose
accumulated attention weights are the largest.

    HeavyHitterStreamingAttention   the cache of streams in lockstep, one query a head at a time; may stand behind a prefix
                                    that the streams share
    received_attention              the weights that a prompt's tokens receive from its rows, which the cache starts from

Computed by hand-written HIP kernels on the inputs' ROCm device and its current stream; there is no CPU path.  Serving
only: results take no part in derivatives.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple, Union

import torch

import _native
from shared_prefix_attention import _check_prefix, _check_rows, _refuse_gradients, _walkable, shared_prefix_attention
from sink_window_attention import (MAX_DIM, MAX_ROWS, _attention_scale, _check_dtype, _check_gpu, _check_lengths, _like, _on,
                                   _widen)

Tensor = torch.Tensor

__all__ = ["HeavyHitterStreamingAttention", "received_attention"]

MAX_GROUP = 512  # query heads of a key head

_PAIRS = {n: ctypes.c_int64 * n for n in (4, 6)}


def received_attention(q: Tensor, k: Tensor, *, lengths: Optional[Tensor] = None, counts: Optional[Tensor] = None,
                       lse: Optional[Tensor] = None, scale: Optional[float] = None) -> Tensor:
    """The attention weights that tokens receive, float32 [B,Hkv,M]: for every own token the sum, over the query rows that
    see it and the query heads of its key head, of exp(scale q.k) over the row's sum of them.

    q [B,H,N,D] (the newest rows, or only the last of a prompt: its window of observation), k [B,Hkv,M,D]; lengths and
    counts as shared_prefix_attention takes them.  lse: float32 [B,H,N], the rows' statistics as shared_prefix_attention
    gives them with_lse (a prefix's tokens then have their share of every row), or None: computed here, over the own
    tokens alone.  Zero behind the lengths; NaN for tokens that a row with an infinite or NaN statistic sees.  May be
    captured into a graph; inputs that ask for derivatives are refused (RuntimeError)."""
    _refuse_gradients(*((q, k) if lse is None else (q, k, lse)))
    _check_rows(q, k, "q and k")
    b, h, n, d = q.shape
    hk, m = k.shape[1], k.shape[2]
    _check_dtype(q, k)
    lengths, counts = _check_lengths(lengths, b), _check_lengths(counts, b, "counts")
    if lse is not None:
        if lse.dtype != torch.float32 or tuple(lse.shape) != (b, h, n):
            raise ValueError(f"lse must be a float32 tensor {[b, h, n]}")
        lse = lse.detach().contiguous()
    _check_gpu(q, k, lengths, counts, lse)
    s = _attention_scale(scale, d)
    weights = q.new_empty((b, hk, m), dtype=torch.float32)
    if weights.numel() == 0 or n == 0 or h == 0:
        return weights.zero_()
    (q, k), strides = _walkable(_widen(q.detach()), _widen(k.detach()))
    code, lib = _native.DTYPE_CODES[q.dtype], _native.lib()
    with _on(q.device):
        nbytes = lib.sta_received_attention_bytes(code, b, h, hk, n, m, q.shape[3], lse is not None)
        if nbytes < 0:
            raise _native.NativeError("sta_received_attention_bytes refused the shape")
        ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        st = lib.sta_received_attention(
            q.data_ptr(), k.data_ptr(), code, b, h, hk, n, m, q.shape[3], strides, s, _native.ptr(lengths),
            _native.ptr(counts), _native.ptr(lse), weights.data_ptr(), _native.ptr(ws), nbytes,
            _native.stream_handle(q.device))
    _native.check(st, "sta_received_attention")
    return weights


class HeavyHitterStreamingAttention:
    """Exact streaming attention over a bounded cache of every stream and key head: the last `recent` tokens and `kept` older
    ones, those that received the most attention.

    Each token held has a weight, the sum of the attention weights that the queries gave it, over the query heads of its
    key head.  When a token comes and the cache is full, the token that passes out of the last `recent` takes the place
    of the kept one of the lowest weight (of equal ones that of the first slot), unless its own is lower still; then it
    is the one that is forgotten.

    `step(q, k, v)` takes one token of every stream: keys [S,Hkv,dim], values [S,Hkv,value_dim], queries [S,H,dim] ->
    [S,H,value_dim], H a multiple of Hkv (at most 512 times); `update` and `query` are its two halves.  `start` begins
    streams from prompts whose tokens' weights are known, `prefill` from prompts that it answers.  With `prefix` queries
    also see keys and values that the streams share and that never leave; their share counts in every weight.

    dtype (float32, bfloat16, float16) is that of inputs, outputs and the cache; weights, sums and softmax statistics are
    fp32.  A weight is a plain fp32 sum: what a query adds to it is rounded at 2^-24 of the weight, so that weights order what
    differs by more than n 2^-24 of them after n queries, and one does not grow past 2^24 times what each query adds.
    Increments that are infinite or NaN are left out of the weights.  A token whose key gives a logit of +infinity
    (or beyond fp32) or NaN with a finite query makes the outputs that it reaches NaN while it is held; its weight is the
    lowest finite one from then on, whatever it was, so it is the first that another token takes the place of.  One whose
    value alone is infinite or NaN is forgotten like others.

    Calls run on the device's current stream and may be captured into graphs (replays advance the state like
    calls); calls on one object have to be ordered, by one stream or by events.  Results take no part in derivatives."""

    def __init__(self, dim: int, value_dim: int, *, streams: int = 1, heads: int = 1, kv_heads: Optional[int] = None,
                 kept: int, recent: int, scale: Optional[float] = None, dtype: torch.dtype = torch.float32,
                 device: Optional[Union[str, torch.device]] = None) -> None:
        kv_heads = heads if kv_heads is None else kv_heads
        if streams < 1 or heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError("streams and heads must be positive and heads a multiple of kv_heads")
        if heads // kv_heads > MAX_GROUP:
            raise ValueError(f"at most {MAX_GROUP} query heads of a key head are supported")
        if not 1 <= dim <= MAX_DIM or not 1 <= value_dim <= MAX_DIM:
            raise ValueError(f"key and value widths must be 1 .. {MAX_DIM}, got {dim} and {value_dim}")
        for name, x in (("kept", kept), ("recent", recent)):
            if isinstance(x, bool) or not isinstance(x, int):
                raise ValueError(f"{name} must be an int, got {x!r}")
            if x < 1:
                raise ValueError(f"{name} must be at least 1")
        if kept + recent > MAX_ROWS:
            raise ValueError(f"a cache of at most {MAX_ROWS} tokens is supported")
        if dtype not in _native.DTYPE_CODES:
            raise ValueError(f"dtype {dtype} is not supported (use float32, bfloat16 or float16)")
        self.scale = _attention_scale(scale, dim)
        self.dim, self.value_dim, self.streams, self.heads, self.kv_heads = dim, value_dim, streams, heads, kv_heads
        self.kept, self.recent, self.dtype = kept, recent, dtype
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise ValueError(f"HIP kernels require a GPU (cuda/ROCm) device, got {dev}")
        if not torch.cuda.is_available():
            raise RuntimeError("streaming-attention HIP kernels need a ROCm GPU; none is visible")
        self.device = torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)
        self._code = _native.DTYPE_CODES[dtype]
        sizes = (ctypes.c_int64 * 3)()
        _native.check(_native.lib().sta_heavy_layout(self._code, streams, kv_heads, dim, value_dim, recent, kept, sizes),
                      "sta_heavy_layout")

        def room(*shape, dtype, value=0):
            return torch.full(shape, value, device=self.device, dtype=dtype)

        self._slots = recent + 1 + kept
        self._keys, self._values = (room(n, dtype=torch.uint8) for n in sizes[:2])
        self._counts = room(streams, kv_heads, dtype=torch.int64)
        self._weights = room(streams, kv_heads, sizes[2], dtype=torch.float32)
        self._positions = room(streams, kv_heads, sizes[2], dtype=torch.int64, value=-1)
        self._lowest = room(streams, kv_heads, 2, dtype=torch.int64, value=-1)
        self._tensors = {"keys": self._keys, "values": self._values, "counts": self._counts, "weights": self._weights,
                         "positions": self._positions, "lowest": self._lowest}
        self._state = tuple(x.data_ptr() for x in self._tensors.values())
        self._views = self._weights[..., :self._slots], self._positions[..., :self._slots]
        shape = (streams, kv_heads, self._slots)  # of the items' rows, without memory of their own
        self._items = tuple(torch.empty(1, dtype=t, device=self.device).expand(size) for size, t in (
            ((*shape, dim), dtype), ((*shape, value_dim), dtype), (shape, torch.int64), (shape, torch.float32)))
        self._shapes = {"query": (streams, heads, dim), "key": (streams, kv_heads, dim),
                        "value": (streams, kv_heads, value_dim)}
        self._dense = _PAIRS[6](heads * dim, dim, kv_heads * dim, dim, kv_heads * value_dim, value_dim)
        self._bytes: dict = {}
        self._start_bytes = _native.lib().sta_heavy_start_bytes(streams, kv_heads, recent, kept)

    @property
    def lengths(self) -> Tensor:
        """int64 [S] on the device: tokens that each stream has taken, a view of the state to be read only."""
        return self._counts[:, 0]

    @property
    def weights(self) -> Tensor:
        """float32 [S,Hkv,recent + 1 + kept]: the slots' weights (0 where no token is), a view of the state to be read only.
        Token p is in slot p % (recent + 1) while it is one of the last `recent`; the slots behind are those of kept
        tokens, taken in turn by the first that pass out."""
        return self._views[0]

    @property
    def positions(self) -> Tensor:
        """int64 [S,Hkv,recent + 1 + kept]: the slots' tokens (-1 where none is), a view of the state to be read only."""
        return self._views[1]

    def _rows(self, x: Tensor, want: Tuple[int, ...], what: str) -> Tensor:
        if x.shape != want:
            raise ValueError(f"{what} must be {list(want)}, got {list(x.shape)}")
        if x.dtype != self.dtype or x.device != self.device:
            x = x.detach().to(device=self.device, dtype=self.dtype)
        return x if x.is_contiguous() or x.stride(-1) == 1 or x.shape[-1] == 1 else x.detach().contiguous()

    def _check_shared(self, prefix, prefix_lengths) -> tuple:
        pk, pv = prefix
        if self.dim * pk.element_size() < 16 or self.value_dim * pk.element_size() < 16:
            raise ValueError("a shared prefix needs keys and values of at least 16 bytes")
        sets, p = _check_prefix(pk, pv, self.streams, self.kv_heads, self.dim, self.value_dim)
        for x in (pk, pv):
            if x.dtype != self.dtype or x.device != self.device:
                raise ValueError("the prefix must have the object's dtype and be on its device")
        prefix_lengths = _check_lengths(prefix_lengths, sets, "prefix_lengths")
        if prefix_lengths is not None and prefix_lengths.device != self.device:
            raise ValueError("prefix_lengths must be on the object's device")
        return *_walkable(pk.detach(), pv.detach()), sets, p, prefix_lengths

    def _attend(self, q: Tensor, k: Optional[Tensor], v: Optional[Tensor], prefix, prefix_lengths) -> Tensor:
        sets = p = 0
        pk = pv = prefix_strides = None
        if prefix is not None:
            (pk, pv), prefix_strides, sets, p, prefix_lengths = self._check_shared(prefix, prefix_lengths)
        elif prefix_lengths is not None:
            raise ValueError("prefix_lengths without a prefix")
        nbytes = self._bytes.get((sets, p))
        if nbytes is None:  # another prefix than the last call's
            nbytes = _native.lib().sta_heavy_attention_bytes(
                self._code, self.streams, self.heads, self.kv_heads, self.dim, self.value_dim, self.recent, self.kept,
                sets, p)
            if nbytes < 0:
                raise _native.NativeError("sta_heavy_attention_bytes refused the shape")
            self._bytes = {(sets, p): nbytes}
        out = _like(q) if self.dim == self.value_dim else q.new_empty((self.streams, self.heads, self.value_dim))
        ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        if q.is_contiguous() and (k is None or (k.is_contiguous() and v.is_contiguous())):
            strides = self._dense
        else:
            none = (0, 0)
            strides = _PAIRS[6](*q.stride()[:2], *(none if k is None else k.stride()[:2]),
                                *(none if v is None else v.stride()[:2]))
        with _on(self.device):
            st = _native.lib().sta_heavy_attention(
                q.data_ptr(), _native.ptr(k), _native.ptr(v), self._code, self.streams, self.heads, self.kv_heads,
                self.dim, self.value_dim, strides, self.scale, self.recent, self.kept, _native.ptr(pk), _native.ptr(pv),
                sets, p, prefix_strides, _native.ptr(prefix_lengths), *self._state, out.data_ptr(), _native.ptr(ws),
                nbytes, _native.stream_handle(self.device))
        _native.check(st, "sta_heavy_attention")
        return out

    def step(self, query: Tensor, key: Tensor, value: Tensor, *, prefix: Optional[Tuple[Tensor, Tensor]] = None,
             prefix_lengths: Optional[Tensor] = None) -> Tensor:
        """One token of every stream into the cache, then one query a head: update(key, value); query(query).

        prefix: (keys [Hkv,P,dim], values [Hkv,P,value_dim]) that all streams see in front of their own tokens, or
        ([G,Hkv,P,dim], [G,Hkv,P,value_dim]) with stream s seeing prefix s // (S / G), in the object's dtype; prefix_lengths:
        int32 [G] on the device, the rows of each that count (None: P)."""
        shapes = self._shapes
        q = self._rows(query, shapes["query"], "query")
        k = self._rows(key, shapes["key"], "key")
        v = self._rows(value, shapes["value"], "value")
        return self._attend(q, k, v, prefix, prefix_lengths)

    def query(self, query: Tensor, *, prefix: Optional[Tuple[Tensor, Tensor]] = None,
              prefix_lengths: Optional[Tensor] = None) -> Tensor:
        """Attention of one query a head over the tokens held (and the prefix), whose weights grow by it; zero for a stream
        that has nothing to see."""
        return self._attend(self._rows(query, self._shapes["query"], "query"), None, None, prefix, prefix_lengths)

    def update(self, key: Tensor, value: Tensor) -> None:
        """One token of every stream into the cache."""
        k = self._rows(key, self._shapes["key"], "key")
        v = self._rows(value, self._shapes["value"], "value")
        with _on(self.device):
            st = _native.lib().sta_heavy_update(
                k.data_ptr(), v.data_ptr(), self._code, self.streams, self.kv_heads, self.dim, self.value_dim,
                _PAIRS[4](*k.stride()[:2], *v.stride()[:2]), self.recent, self.kept, *self._state,
                _native.stream_handle(self.device))
        _native.check(st, "sta_heavy_update")

    @torch.no_grad()
    def start(self, keys: Tensor, values: Tensor, weights: Tensor, *, counts: Optional[Tensor] = None) -> None:
        """Streams begin anew from prompts: keys [S,Hkv,P,dim], values [S,Hkv,P,value_dim] and the weights that their
        tokens have received, float32 [S,Hkv,P] (received_attention's; an infinite one keeps a token with a finite key
        for good, NaN counts as 0).  The last `recent` tokens stay, and of the others the `kept` of the largest weights (of
        equal ones the first), in the order of their positions.  counts: int32 [S] on the device, the rows of every stream
        that are tokens (None: all P; values above P are taken as P); a stream with none, 0 or less, keeps what it holds."""
        rows = keys.shape[2] if keys.ndim == 4 else 0
        if rows > MAX_ROWS:
            raise ValueError(f"at most {MAX_ROWS} rows at a time are supported")
        k = self._rows(keys, (self.streams, self.kv_heads, rows, self.dim), "keys")
        v = self._rows(values, (self.streams, self.kv_heads, rows, self.value_dim), "values")
        if weights.dtype != torch.float32 or tuple(weights.shape) != (self.streams, self.kv_heads, rows):
            raise ValueError(f"weights must be a float32 tensor {[self.streams, self.kv_heads, rows]}")
        counts = _check_lengths(counts, self.streams, "counts")
        _check_gpu(k, v, weights, counts)
        if rows == 0:
            return
        weights = weights.detach().contiguous()
        if 0 <= weights.data_ptr() - self._state[3] < 4 * self._weights.numel():  # the state's own, which the call writes
            weights = weights.clone()
        (k, v), strides = _walkable(k, v)
        lib = _native.lib()
        with _on(self.device):
            ws = k.new_empty(self._start_bytes, dtype=torch.uint8)
            st = lib.sta_heavy_start(
                k.data_ptr(), v.data_ptr(), weights.data_ptr(), self._code, self.streams, self.kv_heads, rows, self.dim,
                self.value_dim, strides, self.recent, self.kept, _native.ptr(counts), *self._state,
                ws.data_ptr(), self._start_bytes, _native.stream_handle(self.device))
        _native.check(st, "sta_heavy_start")

    @torch.no_grad()
    def prefill(self, q: Tensor, k: Tensor, v: Tensor, *, counts: Optional[Tensor] = None,
                prefix: Optional[Tuple[Tensor, Tensor]] = None, prefix_lengths: Optional[Tensor] = None) -> Tensor:
        """Exact causal outputs [S,H,P,value_dim] of prompts' rows, behind the prefix if there is one, from which the streams
        then begin: shared_prefix_attention, received_attention and start in one.  counts as start takes them; output rows
        behind them are zero."""
        rows = k.shape[2] if k.ndim == 4 else 0
        q = self._rows(q, (self.streams, self.heads, rows, self.dim), "q")
        k = self._rows(k, (self.streams, self.kv_heads, rows, self.dim), "k")
        v = self._rows(v, (self.streams, self.kv_heads, rows, self.value_dim), "v")
        if prefix is None:
            if prefix_lengths is not None:
                raise ValueError("prefix_lengths without a prefix")
            prefix = k.new_empty((self.kv_heads, 0, self.dim)), k.new_empty((self.kv_heads, 0, self.value_dim))
        out, lse = shared_prefix_attention(q.detach(), k.detach(), v.detach(), *(x.detach() for x in prefix),
                                           lengths=counts, counts=counts, prefix_lengths=prefix_lengths,
                                           scale=self.scale, with_lse=True)
        weights = received_attention(q, k, lengths=counts, counts=counts, lse=lse, scale=self.scale)
        self.start(k, v, weights, counts=counts)
        return out

    def reset(self, streams: Optional[Sequence[int]] = None) -> None:
        """Forgets every token of all streams, or of the given ones."""
        chosen = [slice(None)] if streams is None else list(streams)
        for i in chosen if streams is not None else ():
            if not 0 <= i < self.streams:
                raise ValueError(f"there is no stream {i}")
        for i in chosen:
            self._counts[i].zero_()
            self._weights[i].zero_()
            self._positions[i].fill_(-1)
            self._lowest[i].fill_(-1)

    def items(self) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
        """(keys [S,Hkv,recent + 1 + kept,dim], values [S,Hkv,recent + 1 + kept,value_dim], positions int64, weights
        float32 [S,Hkv,recent + 1 + kept]) as the cache holds them, in the order of its slots; zero, and position -1,
        where no token is."""
        keys, values, positions, weights = (_like(x) for x in self._items)
        with _on(self.device):
            st = _native.lib().sta_heavy_items(
                self._code, self.streams, self.kv_heads, self.dim, self.value_dim, self.recent, self.kept,
                self._keys.data_ptr(), self._values.data_ptr(), self._weights.data_ptr(), self._positions.data_ptr(),
                keys.data_ptr(), values.data_ptr(), weights.data_ptr(), positions.data_ptr(),
                _native.stream_handle(self.device))
        _native.check(st, "sta_heavy_items")
        return keys, values, positions, weights

    def state_size_bytes(self) -> int:
        """Device bytes of the cache."""
        return sum(x.numel() * x.element_size() for x in self._tensors.values())

    def state_dict_settings(self) -> dict:
        return {"dim": self.dim, "value_dim": self.value_dim, "streams": self.streams, "heads": self.heads,
                "kv_heads": self.kv_heads, "kept": self.kept, "recent": self.recent, "scale": self.scale,
                "dtype": str(self.dtype)}

    def state_dict(self) -> dict:
        """The state for a later resume: plain tensors on the host and Python scalars."""
        return {"attention": self.state_dict_settings(), **{name: x.cpu() for name, x in self._tensors.items()}}

    def load_state_dict(self, state: dict) -> None:
        """Resume from state_dict() of an object built with the same settings (the device may differ)."""
        mine = self.state_dict_settings()
        if state["attention"] != mine:
            raise ValueError(f"state settings {state['attention']} do not match this object's {mine}")
        for name, x in self._tensors.items():
            if state[name].shape != x.shape or state[name].dtype != x.dtype:
                raise ValueError("the state's tensors do not match this object's")
        if bool((state["counts"] < 0).any()):
            raise ValueError("the state's counts must not be negative")
        for name, x in self._tensors.items():
            x.copy_(state[name])
