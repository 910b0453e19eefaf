"""The 16-bit paged cache behind a shared prefix in plain numpy, and rotary positions: rows held in fp32 as
the cache's type holds them, attention and angles in 64 bits and more.  Shared by the tests of ``n730_kv16_*``."""
import numpy as np
import torch

HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TINY = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}  # half of the smallest step
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def rounded(x, dtype):
    """x as the type holds it, in fp32."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TYPES[dtype]).float().numpy()


def turned(x, pos, freq, factor, layout):
    """Rows x [..., heads, dim] rotated at positions pos [...], and the bound that their computation in fp32 keeps:
    an angle's rest of a turn is rounded to 2^-24 (half a turn: pi 2^-24 rad) behind an error of 2^-52 of the angle,
    sincospif is off by 2 ulp, the factor rounds once; two products and a sum round each."""
    x = np.asarray(x, np.float64)
    n = 2 * len(freq)
    a = pos.astype(np.longdouble)[..., None, None] * freq.astype(np.longdouble)
    pi2 = 2 * np.arccos(np.longdouble(-1))
    r = (a - pi2 * np.rint(a / pi2)).astype(np.float64)
    c, s = factor * np.cos(r), factor * np.sin(r)
    i, j = (np.arange(n // 2), np.arange(n // 2, n)) if layout == "half" else (np.arange(0, n, 2), np.arange(1, n, 2))
    y, e = x.copy(), np.zeros_like(x)
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    off = abs(factor) * (10 * 2.0 ** -24 + np.abs(a).astype(np.float64) * 2.0 ** -52) * (np.abs(x[..., i]) + np.abs(x[..., j]))
    e[..., i], e[..., j] = off, off
    return y, e


class Cache:
    """Host mirror of one layer's cache behind a prefix."""

    def __init__(self, batch, max_pages, prefix_pages, prefix_len, kv, dim, page, dtype, rng, spare=2, fill=None):
        self.kv, self.dim, self.page, self.dtype, self.max_pages, self.prefix_pages = kv, dim, page, dtype, max_pages, prefix_pages
        self.n_pages = batch * max_pages + prefix_pages + spare
        shape = (self.n_pages, kv, page, dim)
        self.k, self.v = (rounded(rng.standard_normal(shape) if fill is None else np.full(shape, fill), dtype) for _ in range(2))
        ids = rng.permutation(self.n_pages).astype(np.int32)
        self.prefix_table, self.table = ids[:prefix_pages], ids[prefix_pages:prefix_pages + batch * max_pages].reshape(batch, max_pages)
        self.prefix_len = prefix_len
        self.cap = max_pages * page

    @property
    def prefix(self):
        return min(max(self.prefix_len, 0), self.prefix_pages * self.page)

    def slot(self, ids, p):
        """(page, offset) of a position, None where it has no page."""
        pg = int(ids[p // self.page])
        return (pg, p % self.page) if 0 <= pg < self.n_pages else None

    def len(self, lens, b):
        return min(max(int(lens[b]), 0), self.cap)

    def append(self, k, v, lens, new):
        """Rows k, v [B, T, kv, dim] (fp32)."""
        for b in range(k.shape[0]):
            for t in range(min(max(int(new[b]), 0), k.shape[1])):
                p = self.len(lens, b) + t
                at = self.slot(self.table[b], p) if p < self.cap else None
                if at:
                    self.k[at[0], :, at[1]], self.v[at[0], :, at[1]] = rounded(k[b, t], self.dtype), rounded(v[b, t], self.dtype)

    def attention(self, q, lens, new, scale):
        """(out, bound) [B, T, heads, dim]: see the tests for the bound."""
        B, T, H, D = q.shape
        g = H // self.kv
        out, bound = np.zeros(q.shape), np.zeros(q.shape)
        first = [self.slot(self.prefix_table, p) for p in range(self.prefix)]
        for b in range(B):
            for t in range(min(max(int(new[b]), 0), T)):
                own = [self.slot(self.table[b], p) for p in range(min(self.len(lens, b) + t + 1, self.cap))]
                at = [x for x in first + own if x]
                if not at:
                    continue
                pg, off = np.array(at).T
                for h in range(H):
                    k, v = self.k[pg, h // g, off].astype(np.float64), self.v[pg, h // g, off].astype(np.float64)
                    x = k @ q[b, t, h].astype(np.float64) * scale
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    y = p @ v
                    big = np.abs(v).max(0)
                    dx = (D + 8) * 2.0 ** -23 * abs(scale) * (np.abs(k) @ np.abs(q[b, t, h].astype(np.float64))).max() + 2.0 ** -20
                    s = p @ np.abs(v)
                    out[b, t, h] = y
                    bound[b, t, h] = HALF[self.dtype] * (np.abs(y) + s) + 2 * dx * s + TINY[self.dtype] * (len(at) * big + 1)
        return out, bound
