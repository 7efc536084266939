"""Plain float64 statements of the windowed attention, the head norm with rotation and the token cache, on the CPU, with
bounds on how far a kernel may be from them.

The bounds are first-order rounding analysis, element by element: u = eps / 2 of the element type for every rounding to
it (the output, and the weights of 16-bit rows), 2^-24 for every fp32 operation of a sum."""

import math

import torch

F24 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def weight_step(dtype):
    """Relative error of a weight as the value sums take it: 16-bit rows' weights are rounded to 16 bits."""
    return 0.0 if dtype == torch.float32 else half_step(dtype)


def visible(n, length, window, sinks):
    i = torch.arange(n)[:, None]
    j = torch.arange(n)[None]
    return (j <= i) & ((i - j < window) | (j < sinks)) & (i < length)


def window_attention(q, k, v, *, window, sinks, scale=None, lengths=None, grad=None):
    """[B,H,N,D], [B,Hkv,N,D], [B,Hkv,N,Dv]: {"out": (value, bound)} in float64, with "dq", "dk", "dv" if grad is given."""
    dt = q.dtype
    u, w = half_step(dt), weight_step(dt)
    b, h, n, d = q.shape
    hk = k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    res = {name: [torch.zeros(*shape, dtype=torch.float64) for _ in range(2)]
           for name, shape in (("out", (b, h, n, v.shape[3])), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape))}
    for bi in range(b):
        length = n if lengths is None else max(0, min(n, int(lengths[bi])))
        see = visible(n, length, window, sinks)
        for hi in range(h):
            kk, vv, qq = k[bi, hi * hk // h].clone(), v[bi, hi * hk // h].clone(), q[bi, hi].clone()
            for x in (kk, vv, qq):
                x[length:] = 0
            x = (qq @ kk.T) * scale
            size = (qq.abs() @ kk.abs().T) * abs(scale)
            p = torch.where(see, x, -math.inf)
            p = torch.where(see, torch.exp(p - p.amax(1, keepdim=True)), 0.0)
            p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            # relative error of an fp32 weight: its logit's dot product, the exponent's argument, the row's sum
            ep = F24 * (2 * (d + 4) * torch.where(see, size, 0.0).amax(1, keepdim=True) + n + 32)
            o = p @ vv
            eo = u * o.abs() + (w + ep) * (p @ vv.abs()) + F24 * n * (p @ vv.abs())
            res["out"][0][bi, hi], res["out"][1][bi, hi] = o, eo
            if grad is None:
                continue
            go = grad[bi, hi].double().clone()
            go[length:] = 0
            dp = go @ vv.T
            delta = (go * o).sum(1, keepdim=True)
            # error of dp - delta: fp32 dot products, and the output as it was rounded
            ed = (d + 32) * F24 * (go.abs() @ vv.abs().T) + (go.abs() * (eo + 2 * (d + 32) * F24 * o.abs())).sum(1, keepdim=True)
            ds = p * (dp - delta) * scale
            es = (w + ep) * ds.abs() + p * ed * abs(scale)
            if dt == torch.float16:  # subnormal weights: half a step of 2^-24 over the power of two they carry
                lift = 2.0 ** min(10, int(math.log2(max(1, min(window + sinks, n)))))
                tiny = see * (2.0 ** -25 / lift)
            else:
                tiny = see * 0.0
            dv, ev = p.T @ go, ((w + ep) * p + tiny).T @ go.abs()
            dk, ek = ds.T @ qq, (es + tiny * abs(scale)).T @ qq.abs()
            dq, eq = ds @ kk, (es + tiny * abs(scale)) @ kk.abs()
            n_sum = F24 * n
            res["dq"][0][bi, hi], res["dq"][1][bi, hi] = dq, eq + n_sum * (ds.abs() @ kk.abs())
            for name, val, err, mag in (("dk", dk, ek, ds.abs().T @ qq.abs()), ("dv", dv, ev, p.T @ go.abs())):
                res[name][0][bi, hi * hk // h] += val
                res[name][1][bi, hi * hk // h] += err + n_sum * (h // hk) * mag
    for name in ("dq", "dk", "dv"):
        res[name][1].add_(u * res[name][0].abs())
        if dt == torch.float16:
            res[name][1].add_(2.0 ** -25)  # results below fp16's normal range
    if dt == torch.float16:
        res["out"][1].add_(2.0 ** -25)
    return {name: tuple(x) for name, x in res.items() if grad is not None or name == "out"}


def over(got, want):
    """How many times over its bound the worst element is; infinite where finiteness differs."""
    value, bound = want
    got = got.detach().double().cpu()
    if not torch.isfinite(got).all():
        return math.inf
    # 1e-30: elements with nothing to add up are zero on both sides
    return float(((got - value).abs() / (bound * 1.05 + 1e-30)).max()) if got.numel() else 0.0


def norm_rotary(x, w, cos, sin, *, eps, interleaved, grad=None):
    """Rows [B,H,N,D] with cos and sin [B,N,R/2]: {"y": (value, bound)} in float64, with "dx" and "dw" if grad is given."""
    dt = x.dtype
    u = half_step(dt)
    d = x.shape[-1]
    x = x.double()
    w = torch.ones(d, dtype=torch.float64) if w is None else w.double()
    cos, sin = cos.double()[:, None], sin.double()[:, None]
    pairs = cos.shape[-1]

    def turn(h, sin):
        a = h[..., 0:2 * pairs:2] if interleaved else h[..., :pairs]
        b = h[..., 1:2 * pairs:2] if interleaved else h[..., pairs:2 * pairs]
        y = h.clone()
        parts = a * cos - b * sin, b * cos + a * sin
        if interleaved:
            y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = parts
        else:
            y[..., :pairs], y[..., pairs:2 * pairs] = parts
        return y

    def size(h):  # |a cos| + |b sin|
        y = h.abs().clone()
        a = y[..., 0:2 * pairs:2] if interleaved else y[..., :pairs]
        b = y[..., 1:2 * pairs:2] if interleaved else y[..., pairs:2 * pairs]
        parts = a * cos.abs() + b * sin.abs(), b * cos.abs() + a * sin.abs()
        if interleaved:
            y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = parts
        else:
            y[..., :pairs], y[..., pairs:2 * pairs] = parts
        return y

    inv = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    hat = x * inv
    small = 2.0 ** -25 if dt == torch.float16 else 0.0
    ops = F24 * (d + 12)  # the sum of squares' d operations and a dozen others
    y = turn(hat * w, sin)
    out = {"y": (y, u * y.abs() + ops * size(hat * w) + small)}
    if grad is not None:
        g = grad.double()
        t, big = turn(g, -sin), size(g)
        m = (t * w * hat).mean(-1, keepdim=True)
        dx = inv * (t * w - hat * m)
        err = ops * 2 * inv * (big * w.abs() + hat.abs() * (big * w.abs() * hat.abs()).mean(-1, keepdim=True))
        out["dx"] = (dx, u * dx.abs() + err + small)
        rows = x.numel() // d
        dw = (t * hat).sum((0, 1, 2))
        out["dw"] = (dw, F24 * (rows + d + 12) * (big * hat.abs()).sum((0, 1, 2)))
    return out


def as_held(x, storage):
    """The float64 values that rows stand for in a cache: themselves, or 4-bit floats with a power of two for 32 columns."""
    x = x.double()
    if storage is None:
        return x
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    y = torch.zeros_like(x)
    for lo in range(0, x.shape[-1], 32):
        z = x[..., lo:lo + 32]
        top = z.abs().amax(-1, keepdim=True)
        power = torch.floor(torch.log2(top.clamp_min(2.0 ** -140))) - 2
        unit = 2.0 ** power.clamp_min(-126)
        m = z.abs() / unit
        code = torch.zeros_like(m, dtype=torch.long)
        for i in range(7):  # the border between codes i and i + 1 belongs to the even one
            mid = (grid[i] + grid[i + 1]) / 2
            code += (m > mid) if i % 2 == 0 else (m >= mid)
        v = torch.tensor(grid, dtype=torch.float64)[code] * unit * z.sign()
        y[..., lo:lo + 32] = torch.where(torch.isfinite(top), v, math.nan)
    return y


class TokenCache:
    """Per-token statement of the ring: a dict of positions a stream, every token held."""

    def __init__(self, streams, window, sinks, storage):
        self.window, self.sinks, self.storage = window, sinks, storage
        self.held = [dict() for _ in range(streams)]
        self.n = [0] * streams

    def put(self, s, k, v):
        p = self.n[s]
        if p >= self.sinks + self.window:
            self.held[s].pop(p - self.window, None)
        self.held[s][p] = as_held(k, self.storage), as_held(v, self.storage)
        self.n[s] = p + 1

    def slot(self, p):
        return p if p < self.sinks else self.sinks + (p - self.sinks) % self.window

    def query(self, s, q, scale, dtype):
        """(value, bound) [H, dv] of q [H, d]."""
        u = half_step(dtype)
        q = q.double()
        if not self.held[s]:
            return None
        keys, values = (torch.stack([self.held[s][p][i] for p in sorted(self.held[s])], 1) for i in (0, 1))
        g = q.shape[0] // keys.shape[0]
        keys, values = keys.repeat_interleave(g, 0), values.repeat_interleave(g, 0)
        x = (keys @ q[..., None])[..., 0] * scale
        size = (keys.abs() @ q.abs()[..., None])[..., 0].amax(-1, keepdim=True) * abs(scale)
        p = x.softmax(-1)
        out, mag = (p[:, None] @ values)[:, 0], (p[:, None] @ values.abs())[:, 0]
        # fp32 products and sums of d and n terms, three planes of 8 bits or more (2^-23), 16-bit rows' weights as two planes
        # (2^-16 bf16; half a step of fp16's smallest, 2^-25, in units of the largest weight, of which n add up)
        n, d = x.shape[-1], q.shape[-1]
        planes = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -16
        ep = F24 * (2 * (d + 8) * size + 2 * n + 64) + planes
        bound = u * out.abs() + ep * mag
        if dtype == torch.float16:
            bound = bound + 2.0 ** -25 + 2.0 ** -25 * values.abs().sum(1)
        return out, bound
