"""Refusals of the cache that keeps the most attended tokens, of received weights and of the attention over a shared prefix
that need no GPU: arguments are checked before any kernel is asked for."""

import pathlib
import re

import pytest
import torch

import _native
import heavy_hitter_attention as hha
import kept_reference as ref
import shared_prefix_attention as spa

B, H, HK, N, M, P, D, DV = 4, 6, 2, 3, 9, 7, 16, 24


def attend(q=(B, H, N, D), k=(B, HK, M, D), v=(B, HK, M, DV), pk=(HK, P, D), pv=(HK, P, DV), dtype=torch.float32, **kw):
    return spa.shared_prefix_attention(*(torch.zeros(*s, dtype=dtype) for s in (q, k, v, pk, pv)), **kw)


@pytest.mark.parametrize("kw,message", [
    (dict(q=(H, N, D)), r"must be \[B,H,N,D\]"),
    (dict(k=(B, HK, M, D + 1)), r"k must be \[B,Hkv,M,D\]"),
    (dict(k=(B + 1, HK, M, D)), r"k must be \[B,Hkv,M,D\]"),
    (dict(k=(B, 4, M, D), v=(B, 4, M, DV)), "multiple of the key heads"),
    (dict(v=(B, HK, M + 1, DV)), r"v must be \[B,Hkv,M,Dv\]"),
    (dict(v=(HK, M, DV)), r"v must be \[B,Hkv,M,Dv\]"),
    (dict(v=(B, HK, M, 129), pv=(HK, P, 129)), "widths must be 1 .. 128"),
    (dict(q=(B, H, N, 129), k=(B, HK, M, 129), pk=(HK, P, 129)), "widths must be 1 .. 128"),
    (dict(q=(B, H, M + 1, D)), "query rows are the last of the own tokens"),
    (dict(pk=(P, D), pv=(P, DV)), r"must be \[Hkv,P,D\] or \[G,Hkv,P,D\]"),
    (dict(pk=(HK, P, D), pv=(1, HK, P, DV)), r"must be \[Hkv,P,D\] or \[G,Hkv,P,D\]"),
    (dict(pk=(HK, P, D), pv=(HK, P + 1, DV)), "prefix_k and prefix_v must be"),
    (dict(pk=(3, P, D), pv=(3, P, DV)), "prefix_k and prefix_v must be"),
    (dict(pk=(3, HK, P, D), pv=(3, HK, P, DV)), "multiple of the 3 prefixes"),
    (dict(pk=(0, HK, P, D), pv=(0, HK, P, DV)), "multiple of the 0 prefixes"),
    (dict(dtype=torch.float64), "dtype torch.float64 is not supported"),
    (dict(lengths=torch.zeros(B)), r"lengths must be an int32 tensor \[4\]"),
    (dict(counts=torch.zeros(B + 1, dtype=torch.int32)), r"counts must be an int32 tensor \[4\]"),
    (dict(prefix_lengths=torch.zeros(2, dtype=torch.int32)), r"prefix_lengths must be an int32 tensor \[1\]"),
    (dict(scale=float("nan")), "HIP kernels require GPU"),
    ({}, "HIP kernels require GPU"),
])
def test_prefix_refusals(kw, message):
    with pytest.raises(ValueError, match=message):
        attend(**kw)


def test_mixed_types_and_derivatives():
    x = [torch.zeros(*s) for s in ((B, H, N, D), (B, HK, M, D), (B, HK, M, DV), (HK, P, D), (HK, P, DV))]
    with pytest.raises(ValueError, match="one dtype"):
        spa.shared_prefix_attention(*x[:4], x[4].bfloat16())
    with pytest.raises(ValueError, match="one dtype"):
        hha.received_attention(x[0], x[1].half())
    for i in range(5):
        y = [t.clone().requires_grad_(j == i) for j, t in enumerate(x)]
        with pytest.raises(RuntimeError, match="no backward pass"):
            spa.shared_prefix_attention(*y)
        with torch.no_grad(), pytest.raises(ValueError, match="require GPU"):
            spa.shared_prefix_attention(*y)
    with pytest.raises(RuntimeError, match="no backward pass"):
        hha.received_attention(x[0].requires_grad_(), x[1])
    with pytest.raises(RuntimeError, match="no backward pass"):
        hha.received_attention(x[0].detach(), x[1], lse=torch.zeros(B, H, N, requires_grad=True))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x[1], torch.ones_like(x[1]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            hha.received_attention(x[0].detach(), dual)


@pytest.mark.parametrize("kw,message", [
    (dict(lse=torch.zeros(B, H, N + 1)), "lse must be a float32 tensor"),
    (dict(lse=torch.zeros(B, H, N, dtype=torch.float64)), "lse must be a float32 tensor"),
    (dict(lengths=torch.zeros(B, 1, dtype=torch.int32)), "lengths must be an int32 tensor"),
    (dict(counts=torch.zeros(B, dtype=torch.int64)), "counts must be an int32 tensor"),
    ({}, "HIP kernels require GPU"),
])
def test_received_refusals(kw, message):
    with pytest.raises(ValueError, match=message):
        hha.received_attention(torch.zeros(B, H, N, D), torch.zeros(B, HK, M, D), **kw)


@pytest.mark.parametrize("kw,message", [
    (dict(kept=0), "kept must be at least 1"),
    (dict(recent=0), "recent must be at least 1"),
    (dict(kept=True), "kept must be an int"),
    (dict(recent=2.0), "recent must be an int"),
    (dict(kept=1 << 30, recent=1), "at most 1073741824 tokens"),
    (dict(heads=3, kv_heads=2), "heads a multiple of kv_heads"),
    (dict(streams=0), "must be positive"),
    (dict(heads=513, kv_heads=1), "at most 512 query heads"),
    (dict(dim=0), "widths must be 1 .. 128"),
    (dict(value_dim=129), "widths must be 1 .. 128"),
    (dict(dtype=torch.float64), "is not supported"),
    (dict(scale=float("inf")), "scale must be finite"),
    (dict(device="cpu"), "require a GPU"),
])
def test_cache_refusals(kw, message):
    args = dict(dim=16, value_dim=16, kept=8, recent=4)
    args.update(kw)
    with pytest.raises(ValueError, match=message):
        hha.HeavyHitterStreamingAttention(**args)


def lib():
    return _native.load_library()


def test_workspaces_refuse_what_the_calls_refuse():
    f = lib().sta_prefix_attention_bytes
    good = (1, 4, 8, 2, 2, 1, 64, 1280, 64, 64)  # type batch heads kv sets n m p d dv
    assert f(*good) > 0
    for i, x in ((0, 3), (1, 0), (1, 3), (2, 7), (3, 0), (4, 0), (5, 0), (6, 0), (7, -1), (8, 129), (8, 7), (9, 0), (9, 129),
                 (7, (1 << 30) + 1), (5, 1 << 31)):
        bad = list(good)
        bad[i] = x
        assert f(*bad) == -1, (i, x)
    g = lib().sta_received_attention_bytes
    good = (1, 2, 8, 2, 64, 256, 64, 0)
    assert g(*good) > 0
    for i, x in ((0, 9), (1, 0), (2, 3), (4, 0), (5, 0), (6, 4), (6, 200)):
        bad = list(good)
        bad[i] = x
        assert g(*bad) == -1, (i, x)
    h = lib().sta_heavy_attention_bytes
    good = (1, 2, 8, 2, 64, 64, 16, 100, 1, 50)  # type streams heads kv d dv recent kept sets p
    assert h(*good) > 0
    for i, x in ((0, 3), (1, 0), (2, 7), (2, 2048), (4, 0), (5, 129), (6, 0), (7, 0), (7, 1 << 30), (8, 3), (9, -1)):
        bad = list(good)
        bad[i] = x
        assert h(*bad) == -1, (i, x)
    assert lib().sta_heavy_start_bytes(2, 2, 0, 4) == -1
    assert lib().sta_heavy_start_bytes(2, 2, 3, 4) == 4 * 2 * 2 * 32


def test_null_pointers_are_refused():
    """Entry points look at their arguments before they touch the device."""
    l = lib()
    strides = (_native.ctypes.c_int64 * 15)()
    some = 4096  # never read: the call ends before
    arg = _native.STA_ERR_ARG
    prefix = [some, some, some, some, some, 1, 4, 8, 2, 2, 1, 64, 1280, 64, 64, strides, 0.125, None, None, None, some, None, None,
              0, None]
    for i in (0, 1, 2, 3, 4, 15, 20):
        bad = list(prefix)
        bad[i] = None
        assert l.sta_prefix_attention(*bad) == arg, i
    assert l.sta_prefix_attention(*prefix) == _native.STA_ERR_SCRATCH  # no workspace
    assert l.sta_prefix_attention(*prefix[:16], float("nan"), *prefix[17:]) == arg
    far = (_native.ctypes.c_int64 * 15)(*([0, 0, 1 << 24] * 5))
    assert l.sta_prefix_attention(*prefix[:15], far, *prefix[16:]) == _native.STA_ERR_UNSUPPORTED
    received = [some, some, 1, 2, 8, 2, 64, 256, 64, strides, 0.125, None, None, None, some, None, 0, None]
    for i in (0, 1, 9, 14):
        bad = list(received)
        bad[i] = None
        assert l.sta_received_attention(*bad) == arg, i
    assert l.sta_received_attention(*received) == _native.STA_ERR_SCRATCH
    state = [some] * 6
    heavy = [some, some, some, 1, 2, 8, 2, 64, 64, strides, 0.125, 16, 1 << 20, None, None, 0, 0, None, None, *state, some, None, 0,
             None]
    for i in (0, 2, 9, *range(19, 25), 25):
        bad = list(heavy)
        bad[i] = None
        assert l.sta_heavy_attention(*bad) == arg, i
    assert l.sta_heavy_attention(*heavy) == _native.STA_ERR_SCRATCH
    for i in (19, 20, 22, 23):  # the caches, weights and positions lie on 16 bytes
        bad = list(heavy)
        bad[i] = some + 8
        assert l.sta_heavy_attention(*bad) == arg, i
    update = [some, some, 1, 2, 2, 64, 64, strides, 16, 100, *state, None]
    for i in (0, 1, 7, *range(10, 16)):
        bad = list(update)
        bad[i] = None
        assert l.sta_heavy_update(*bad) == arg, i
    start = [some, some, some, 1, 2, 2, 300, 64, 64, strides, 16, 100, None, *state, None, 0, None]
    for i in (0, 1, 2, 9, *range(13, 19)):
        bad = list(start)
        bad[i] = None
        assert l.sta_heavy_start(*bad) == arg, i
    assert l.sta_heavy_start(*start) == _native.STA_ERR_SCRATCH
    assert l.sta_heavy_start(*start[:6], 0, *start[7:]) == _native.STA_ERR_SHAPE
    items = [1, 2, 2, 64, 64, 16, 100, *[some] * 8, None]
    for i in range(7, 15):
        bad = list(items)
        bad[i] = None
        assert l.sta_heavy_items(*bad) == arg, i


def test_declared_and_bound_alike():
    """Every new entry point of the header is bound with as many arguments as it declares."""
    text = (pathlib.Path(_native.__file__).resolve().parents[1] / "include" / "streamattn.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = [n for n in _native.EXPORTED_SYMBOLS if n.startswith(("sta_prefix", "sta_received", "sta_heavy"))]
    assert len(names) == 11
    for name in names:
        args = re.search(name + r"\(([^)]*)\)", text).group(1).split(",")
        assert len(getattr(lib(), name).argtypes) == len(args), name


def test_the_statement_keeps_what_was_attended():
    """The oracle itself, on a few tokens by hand: kept 2, recent 2."""
    c = ref.Cache(1, 1, 2, 2)
    k = torch.arange(8.0).view(1, 1, 8, 1)
    c.start(k, k, torch.tensor([[[5.0, 1.0, 3.0, 3.0, 9.0, 0.0, 0.0, 0.0]]]), counts=[6])  # recent: 4, 5; of the others 0 and 2
    slots = c.heads[0][0]["slots"]
    assert [None if x is None else x[0] for x in slots] == [None, 4, 5, 0, 2]
    c.update(k[:, :, 0], k[:, :, 0])  # token 6: 4 passes out with 9, 2 has the lowest weight
    assert [None if x is None else x[0] for x in slots] == [6, None, 5, 0, 4]
    c.update(k[:, :, 0], k[:, :, 0])  # token 7: 5 passes out with 0, lower than 5 and 9
    assert [None if x is None else x[0] for x in slots] == [6, 7, None, 0, 4]
    p, _, _, _ = ref._weights(torch.ones(1, 2).double(), torch.zeros(3, 2).double(), torch.zeros(1, 3, dtype=torch.bool), 1.0, 2)
    assert torch.allclose(p, torch.full((1, 3), 1 / 3, dtype=torch.float64))
