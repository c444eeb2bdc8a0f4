"""The 8-bit key/value cache in plain 64-bit torch on the CPU: what the kernels are compared with."""

import math

import torch

LIMIT = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def scale_of(amax, dtype):
    """amax / limit, up to the next bfloat16: 8 significant bits, multiples of 2^-133 below 2^-126."""
    s = amax / torch.full_like(amax, LIMIT[dtype])
    step = torch.ldexp(torch.ones_like(s), (torch.frexp(s).exponent - 8).clamp(min=-133))
    return torch.ceil(s / step) * step


def round_code(y, dtype):
    """To the nearest code, ties to even; float64 in and out."""
    if dtype == torch.int8:
        return torch.round(y)
    ex = torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 1
    step = torch.ldexp(torch.ones_like(y), ex - 3)
    return torch.round(y / step) * step


def encode(x, s, dtype):
    return torch.where(s > 0, round_code(x / torch.where(s > 0, s, torch.ones_like(s)), dtype), torch.zeros_like(x))


class Cache:
    """codes (as float64 values of the codes) and scales of keys, or of values."""

    def __init__(self, n, h, cap, e, dtype, block):
        self.codes = torch.zeros((n, h, cap, e), dtype=torch.float64)
        self.scale = torch.zeros((n, h, cap // block), dtype=torch.float64)
        self.dtype, self.block, self.cap = dtype, block, cap

    def values(self):
        return self.codes * self.scale.repeat_interleave(self.block, dim=2)[..., None]

    def append(self, new, lengths, counts=None):
        n, h, t, _ = new.shape
        for i in range(n):
            c = t if counts is None else min(max(int(counts[i]), 0), t)
            at = min(max(int(lengths[i]), 0), self.cap)
            end = min(at + c, self.cap)
            for b in range(at // self.block, -(-end // self.block) if end > at else 0):
                lo, hi = max(at, b * self.block), min(end, (b + 1) * self.block)
                x = new[i, :, lo - at:hi - at].double()
                held = lo - b * self.block
                for j in range(h):
                    old = self.scale[i, j, b].clone() if held else torch.zeros((), dtype=torch.float64)
                    if not torch.isfinite(x[j]).all():
                        s = torch.tensor(math.nan, dtype=torch.float64)
                    else:
                        s = scale_of(x[j].abs().max(), self.dtype)
                        if not s > old:  # an old NaN stays
                            s = old
                    if held and s > old:
                        c0 = self.codes[i, j, b * self.block:lo]
                        self.codes[i, j, b * self.block:lo] = encode(c0 * old, s, self.dtype)
                    self.codes[i, j, lo:hi] = encode(x[j], s, self.dtype)
                    self.scale[i, j, b] = s


def attention(q, k, v, lengths, counts=None, causal=True, scale=None):
    """q (N, Hq, T, E), k and v (N, H, cap, E), all float64. Returns out, lse, weights, and for the tolerances
    sum |p v| (N, Hq, T, E) and, of each query, the largest scale * sum |q k| (N, Hq, T)."""
    n, hq, t, e = q.shape
    h, cap = k.shape[1], k.shape[2]
    g = hq // h
    scale = 1.0 / math.sqrt(e) if scale is None else scale
    out = torch.zeros_like(q)
    mag = torch.zeros_like(q)
    size = torch.zeros((n, hq, t), dtype=torch.float64)
    lse = torch.full((n, hq, t), -math.inf, dtype=torch.float64)
    weights = torch.zeros((n, h, cap), dtype=torch.float64)
    for i in range(n):
        l = min(max(int(lengths[i]), 0), cap)
        c = t if counts is None else min(max(int(counts[i]), 0), t)
        for j in range(hq):
            for r in range(c):
                lim = l - c + r + 1 if causal else l
                if lim <= 0:
                    continue
                kk, vv = k[i, j // g, :lim], v[i, j // g, :lim]
                s = scale * (kk @ q[i, j, r])
                p = torch.softmax(s, 0)
                out[i, j, r] = p @ vv
                mag[i, j, r] = p @ vv.abs()
                size[i, j, r] = abs(scale) * (kk.abs() @ q[i, j, r].abs()).max()
                lse[i, j, r] = torch.logsumexp(s, 0)
                weights[i, j // g, :lim] += p
    return out, lse, weights, mag, size


def keep(weights, lengths, budget, recent):
    """Kept positions (N, H, budget), -1 behind the last. A stable sort of Python tuples: NaN first, then by weight."""
    n, h, cap = weights.shape
    kept = torch.full((n, h, budget), -1, dtype=torch.int32)
    for i in range(n):
        l = min(max(int(lengths[i]), 0), cap)
        late = min(l, recent)
        for j in range(h):
            w = weights[i, j].tolist()
            order = sorted(range(l - late), key=lambda a: (0 if math.isnan(w[a]) else 1, 0.0 if math.isnan(w[a]) else -w[a], a))
            pos = sorted(order[:min(l, budget) - late]) + list(range(l - late, l))
            kept[i, j, :len(pos)] = torch.tensor(pos, dtype=torch.int32)
    return kept


def evict(cache, kept, new_cap):
    """The kept tokens in a new Cache."""
    n, h, budget = kept.shape
    e = cache.codes.shape[3]
    out = Cache(n, h, new_cap, e, cache.dtype, cache.block)
    vals = cache.values()
    for i in range(n):
        for j in range(h):
            at = kept[i, j][kept[i, j] >= 0].long()
            for b in range(-(-len(at) // cache.block)):
                x = vals[i, j, at[b * cache.block:(b + 1) * cache.block]]
                s = scale_of(x.abs().max(), cache.dtype) if torch.isfinite(x).all() else torch.tensor(math.nan).double()
                out.codes[i, j, b * cache.block:b * cache.block + len(x)] = encode(x, s, cache.dtype)
                out.scale[i, j, b] = s
    return out


def attention_bounds(exact_out, mag, size, dtype):
    """How far a kernel may be from `exact_out`: half a step of the output's type; the weights' rounding to fp16
    (2^-11); the scores' error d, which changes a weight and the sum by a factor e^(+-2d); 2^-19 for fp32 sums and
    exponentials. d: 8 to 16 additions of 16-product steps, each off by 2^-23 of the running magnitude, and four roundings
    of factors: 2^-19 of scale * sum |q k|. fp16 outputs below 2^-14 step by 2^-24."""
    d = 2.0 ** -19 * size[..., None]
    eps = torch.finfo(dtype).eps / 2
    return eps * exact_out.abs() + (2.0 ** -11 + 2 * d + 2.0 ** -19) * mag * (1 + eps) + 2.0 ** -24
