"""Plain forms in float64 of the 8-bit caches and of attention through a window, that the tests compare with."""
import math

import torch

D = 128
SCALE = D ** -0.5
E = 2.0 ** -24
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def grid(dtype):
    """Every value that a code stands for, ascending; its middle is 0."""
    if dtype == torch.int8:
        return torch.arange(-127, 128, dtype=torch.float64)
    up = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()  # pattern 127 is NaN
    return torch.cat([-up[1:].flip(0), up])


def nearest(x, dtype):
    """x to the nearest code's value, of two as near ones to the even one (every second from 0 on)."""
    g = grid(dtype)
    j = torch.searchsorted(g, x.contiguous()).clamp(1, g.numel() - 1)
    lo, hi = g[j - 1], g[j]
    even = (j - g.numel() // 2) % 2 == 0
    return torch.where((hi - x < x - lo) | ((hi - x == x - lo) & even), hi, lo)


def exponent_of(top, dtype):
    """The least exponent >= -126 at which values up to `top` have codes; -128 for one that is not finite."""
    if not math.isfinite(top):
        return -128
    e = -126
    while TOP[dtype] * 2.0 ** e < top:
        e += 1
    return e


class Plain8:
    """A cache's codes as values, float64, and exponents, written one block at a time."""

    def __init__(self, cache):
        self.dtype, self.bs = cache.k.dtype, cache.k.shape[1]
        self.held = [t.cpu().double() for t in (cache.k, cache.v)]
        self.exponents = cache.exponents.cpu().clone()

    def write(self, key, value, slots):
        blocks = {}
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < self.held[0].shape[0] * self.bs:
                blocks.setdefault(s // self.bs, {})[s % self.bs] = t
        for z, x in enumerate((key.cpu().double(), value.cpu().double())):
            for b, places in blocks.items():
                for h in range(x.shape[1]):
                    rows = x[list(places.values()), h]
                    old, e = int(self.exponents[b, h, z]), exponent_of(rows.abs().max().item() if rows.isfinite().all() else math.nan, self.dtype)
                    if 0 not in places:
                        e = -128 if -128 in (old, e) else max(old, e)
                        if e > old:
                            rest = [i for i in range(self.bs) if i not in places]
                            self.held[z][b, rest, h] = nearest(self.held[z][b, rest, h] * 2.0 ** (old - e), self.dtype)
                    self.held[z][b, list(places), h] = nearest(rows * 2.0 ** -e, self.dtype) if e != -128 else torch.zeros(len(places), D).double()
                    self.exponents[b, h, z] = e

    def same(self, cache):
        """Whether the cache holds this, value for value (a code that is NaN, as in rows never written, as itself)."""
        return (all(torch.equal(a.nan_to_num(999.0), t.cpu().double().nan_to_num(999.0)) for a, t in zip(self.held, (cache.k, cache.v)))
                and torch.equal(self.exponents, cache.exponents.cpu()))

    def rows(self, z, slots):
        """[n, heads, 128] float64 at slots; zeros outside the cache."""
        s = torch.as_tensor(slots)
        there = (s >= 0) & (s < self.held[0].shape[0] * self.bs)
        s = torch.where(there, s, 0)
        e = self.exponents[s // self.bs, :, z].double()
        scale = torch.where(e == -128, math.nan, torch.exp2(e))
        return torch.where(there[:, None, None], self.held[z][s // self.bs, s % self.bs] * scale[..., None], 0.0)


def visible(L, window):
    """Places that the token at place L - 1 sees."""
    if window is None:
        return list(range(L))
    return [s for s in range(L) if L - 1 - s < window.size or s < window.sinks]


def attention(q, k, v, scale=SCALE):
    """(out, sum p |v|, the scores' largest error by fp32 sums, the largest score) of q [G, 128] over k, v [t, 128]."""
    s = q @ k.t() * scale
    ds = (132 * E * abs(scale) * (q.abs() @ k.abs().t())).max().item()
    p = torch.softmax(s, dim=-1)
    return p @ v, p @ v.abs(), ds, s.abs().max().item()
