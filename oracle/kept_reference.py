"""Plain float64 statements of the attention over a shared prefix, the weights that tokens receive and the cache that
keeps the most attended ones, on the CPU, with bounds on how far a kernel may be from them (first-order rounding
analysis, as in window_reference)."""

import math

import torch

from window_reference import F24, half_step, over, weight_step  # noqa: F401


def clamp(x, most, default, count):
    """A list of `count` lengths: x (a list or None) within 0 .. most."""
    return [default] * count if x is None else [max(0, min(int(y), most)) for y in x]


def rows_of(b, n, m, lengths, counts):
    """(own tokens, query rows) of every sequence."""
    lengths = clamp(lengths, m, m, b)
    return lengths, [min(c, x) for c, x in zip(clamp(counts, n, n, b), lengths)]


def small(dtype, values):
    """fp16's subnormal outputs, and weights below 2^-36 of a row's largest."""
    return 2.0 ** -25 + 2.0 ** -36 * values.abs().sum(0) if dtype == torch.float16 else 0.0


def _weights(q, keys, hidden, scale, d):
    """(weights [rows, keys], log2 of their sums, relative bound of a weight, absolute bound of the log2)."""
    x = (q @ keys.T) * scale
    size = torch.where(hidden | ~torch.isfinite(x), 0.0, (q.abs() @ keys.abs().T) * abs(scale)).amax(1, keepdim=True)
    x = torch.where(hidden, -math.inf, x)
    top = x.amax(1, keepdim=True)
    p = torch.exp(x - top)
    den = p.sum(1, keepdim=True)
    # dot products in fp32, the exponents' arguments, the sum of as many weights
    rel = F24 * (2 * (d + 4) * size + keys.shape[0] + 32)
    lse = (top + den.log()) / math.log(2.0)
    return p / den, lse[:, 0], rel, (rel / math.log(2.0) + F24 * 8 * (lse[:, None, 0] .abs() + 1))[:, 0]


def prefix_attention(q, k, v, pk, pv, *, lengths=None, counts=None, prefix_lengths=None, scale=None):
    """q [B,H,N,D], own k, v [B,Hkv,M,D | Dv], prefixes pk, pv [G,Hkv,P,D | Dv]:
    {"out": (value, bound), "lse": (value, bound)}."""
    u, w = half_step(q.dtype), weight_step(q.dtype)
    b, h, n, d = q.shape
    hk, m, sets, p_rows = k.shape[1], k.shape[2], pk.shape[0], pk.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    lengths, counts = rows_of(b, n, m, lengths, counts)
    plens = clamp(prefix_lengths, p_rows, p_rows, sets)
    res = {"out": [torch.zeros(b, h, n, v.shape[3], dtype=torch.float64) for _ in range(2)],
           "lse": [torch.zeros(b, h, n, dtype=torch.float64) for _ in range(2)]}
    for i in range(b):
        s, c, length = i * sets // b, counts[i], lengths[i]
        if c == 0:
            continue
        hidden = torch.zeros(c, plens[s] + length, dtype=torch.bool)
        hidden[:, plens[s]:] = torch.ones(c, length, dtype=torch.bool).triu(length - c + 1)
        for j in range(h):
            g = j * hk // h
            keys = torch.cat([pk[s, g, :plens[s]], k[i, g, :length]]).double()
            values = torch.cat([pv[s, g, :plens[s]], v[i, g, :length]]).double()
            p, lse, rel, el = _weights(q[i, j, :c].double(), keys, hidden, scale, d)
            o, a = p @ values, p @ values.abs()
            res["out"][0][i, j, :c] = o
            res["out"][1][i, j, :c] = u * o.abs() + (w + 2 * rel + F24 * keys.shape[0]) * a + small(q.dtype, values)
            res["lse"][0][i, j, :c], res["lse"][1][i, j, :c] = lse, el
    return {name: tuple(x) for name, x in res.items()}


def received(q, k, *, lengths=None, counts=None, lse=None, scale=None, hide=None):
    """(value, bound) [B,Hkv,M] of the weights that the own tokens receive; hide: bool [M], keys with logits of -inf."""
    b, h, n, d = q.shape
    hk, m = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    lengths, counts = rows_of(b, n, m, lengths, counts)
    out = [torch.zeros(b, hk, m, dtype=torch.float64) for _ in range(2)]
    for i in range(b):
        c, length = counts[i], lengths[i]
        if c == 0:
            continue
        hidden = torch.ones(c, length, dtype=torch.bool).triu(length - c + 1)
        if hide is not None:
            hidden |= hide[:length]
        for j in range(h):
            g = j * hk // h
            p, own, rel, el = _weights(q[i, j, :c].double(), k[i, g, :length].double(), hidden, scale, d)
            if lse is not None:  # the weights' arguments, and the statistics as they were given
                p = p * torch.exp2(own - lse[i, j, :c].double())[:, None]
                rel = rel + F24 * 8 * (lse[i, j, :c].double().abs()[:, None] + 1)
            else:
                rel = 2 * rel + el[:, None]
            out[0][i, g, :length] += p.sum(0)
            # a sum of c weights a head: sixteen at a time, the rest compensated, the heads' and splits' totals
            out[1][i, g, :length] += (p * rel).sum(0) + F24 * 48 * p.sum(0)
    return tuple(out)


LEAST = -torch.finfo(torch.float32).max  # weight of a token whose logits are not finite


class Cache:
    """The cache that keeps the most attended tokens, one key head of one stream after the other, in float64 lists."""

    def __init__(self, streams, kv_heads, kept, recent):
        self.streams, self.kv_heads, self.kept, self.recent = streams, kv_heads, kept, recent
        self.heads = [[self._empty() for _ in range(kv_heads)] for _ in range(streams)]

    def _empty(self):
        """n tokens so far; a slot is None or [position, weight, key, value]."""
        return {"n": 0, "slots": [None] * (self.recent + 1 + self.kept)}

    def reset(self, stream):
        self.heads[stream] = [self._empty() for _ in range(self.kv_heads)]

    def start(self, k, v, weights, counts=None):
        ring = self.recent + 1
        for s in range(self.streams):
            n = k.shape[2] if counts is None else max(0, min(int(counts[s]), k.shape[2]))
            if n == 0:
                continue  # holds what it held
            for h in range(self.kv_heads):
                c = self.heads[s][h] = self._empty()
                c["n"] = n
                w = [float(x) for x in weights[s, h, :n]]
                w = [0.0 if x != x else x for x in w]

                def item(p):
                    return [p, w[p], k[s, h, p], v[s, h, p]]

                older = list(range(max(0, n - self.recent)))
                if len(older) > self.kept:
                    older = sorted(sorted(older, key=lambda p: (-w[p], p))[:self.kept])
                for i, p in enumerate(older):
                    c["slots"][ring + i] = item(p)
                for p in range(max(0, n - self.recent), n):
                    c["slots"][p % ring] = item(p)

    def update(self, k, v):
        ring = self.recent + 1
        for s in range(self.streams):
            for h in range(self.kv_heads):
                c = self.heads[s][h]
                n, slots = c["n"], c["slots"]
                if n >= self.recent:
                    at = (n - self.recent) % ring
                    old, gone = slots[at], n - self.recent
                    if gone < self.kept:
                        slots[ring + gone] = old
                    else:
                        low = min(range(self.kept), key=lambda j: (slots[ring + j][1], j))
                        if old[1] >= slots[ring + low][1]:
                            slots[ring + low] = old
                    slots[at] = None
                slots[n % ring] = [n, 0.0, k[s, h], v[s, h]]
                c["n"] = n + 1

    def query(self, q, scale, prefix=None, prefix_length=None):
        """q [S,H,D]: ((out, bound), (weights, bound) [S,Hkv,slots], positions); the weights grow."""
        u, w16 = half_step(q.dtype), weight_step(q.dtype)
        s_, h_, d = q.shape
        group = h_ // self.kv_heads
        out = None
        for s in range(s_):
            for h in range(self.kv_heads):
                held = [x for x in self.heads[s][h]["slots"] if x is not None]
                keys = [x[2] for x in held]
                values = [x[3] for x in held]
                if prefix is not None:
                    keys += list(prefix[0][h, :prefix_length])
                    values += list(prefix[1][h, :prefix_length])
                if out is None:
                    dv = prefix[1].shape[2] if prefix is not None else held[0][3].shape[0] if held else d
                    out = [torch.zeros(s_, h_, dv, dtype=torch.float64) for _ in range(2)]
                if not keys:
                    continue
                keys, values = torch.stack(keys).double(), torch.stack(values).double()
                rows = q[s, h * group:(h + 1) * group].double()
                p, _, rel, _ = _weights(rows, keys, torch.zeros(group, keys.shape[0], dtype=torch.bool), scale, d)
                # logits of +inf (beyond float32) or NaN: the row has no weights, the token the least, if the query is sane
                logits = rows @ keys.T * (-1.0 if scale < 0 else 1.0)
                lost = ~(logits <= -LEAST)
                p = torch.where(lost.any(1, keepdim=True), math.nan, p)
                lost = (lost & (rows.abs() < 2.0 ** 64).all(1, keepdim=True)).any(0)
                o, a = p @ values, p @ values.abs()
                out[0][s, h * group:(h + 1) * group] = o
                out[1][s, h * group:(h + 1) * group] = (u * o.abs() + (w16 + 2 * rel + F24 * keys.shape[0]) * a
                                                        + small(q.dtype, values))
                for i, x in enumerate(held):
                    if lost[i]:
                        x[1:] = [min(x[1], LEAST), x[2], x[3], 0.0]
                        continue
                    fine = torch.isfinite(p[:, i])
                    x[1] += float(p[fine, i].sum())
                    # the weights' own errors, their sum over the heads, its addition
                    grown = float((p[:, i] * (2 * rel[:, 0] + F24 * (group + 8)))[fine].sum()) + F24 * abs(x[1])
                    if len(x) == 4:
                        x.append(0.0)
                    x[4] += grown
        return tuple(out)

    def state(self):
        """(weights, their bounds, positions) [S,Hkv,slots]."""
        def table(f, empty, dtype):
            return torch.tensor([[[empty if x is None else f(x) for x in c["slots"]] for c in row] for row in self.heads],
                                dtype=dtype)

        return (table(lambda x: x[1], 0.0, torch.float64), table(lambda x: x[4] if len(x) == 5 else 0.0, 0.0, torch.float64),
                table(lambda x: x[0], -1, torch.int64))

    def adopt(self, weights):
        """The slots' weights as another cache holds them (exactly, so that what leaves next is decided by equal numbers)."""
        weights = weights.tolist()
        for s in range(self.streams):
            for h in range(self.kv_heads):
                for i, x in enumerate(self.heads[s][h]["slots"]):
                    if x is not None:
                        x[1:] = [weights[s][h][i], x[2], x[3]]
