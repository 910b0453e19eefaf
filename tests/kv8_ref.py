"""The 8-bit key/value cache in plain numpy: codes and scales by the definition (fp32 quotients and
products, rounded to nearest, ties to even), attention and eviction in 64 bits.

Shared by the tests of ``n730_kv8_*``; works on host arrays only.
"""
import numpy as np

TOP = {"int8": np.float32(127), "e4m3": np.float32(448)}


def e4m3_values():
    """The value of each of the 256 e4m3 codes (NaN for 0x7f and 0xff)."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))
    v = np.where((e == 15) & (m == 7), np.nan, v)
    return np.where(c >> 7, -v, v)


E4M3 = e4m3_values()


def decode(codes, code):
    return codes.view(np.int8).astype(np.float64) if code == "int8" else E4M3[codes]


def encode(y, code):
    """uint8 codes of fp32 values in units of the scale (NaN: 0)."""
    y = np.asarray(y, np.float32)
    if code == "int8":
        return np.where(np.isnan(y), 0, np.clip(np.rint(y), -127, 127)).astype(np.int8).view(np.uint8)
    a = np.minimum(np.abs(np.where(np.isnan(y), 0, y)).astype(np.float64), 448.0)
    e = np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6.0)
    q = np.minimum(np.rint(a / 2.0 ** (e - 3)) * 2.0 ** (e - 3), 448.0)
    c = np.searchsorted(E4M3[:127], q).astype(np.uint8)
    return np.where(np.signbit(y), c | 0x80, c).astype(np.uint8)


class Cache:
    """Host mirror of one layer's cache."""

    def __init__(self, n_pages, max_pages, batch, kv, dim, page, block, code, rng, fill=None):
        self.n_pages, self.max_pages, self.kv, self.dim = n_pages, max_pages, kv, dim
        self.page, self.block, self.code = page, block, code
        shape = (n_pages, kv, page, dim)
        self.k, self.v = (np.full(shape, fill, np.uint8) if fill is not None else
                          rng.integers(0, 256, shape, np.uint8) for _ in range(2))
        if code == "int8":
            self.k[self.k == 128] = 129  # -128 is no code
            self.v[self.v == 128] = 129
        elif fill is None:  # finite codes
            self.k[(self.k & 127) == 127] = 1
            self.v[(self.v & 127) == 127] = 1
        s = 0.03 if code == "int8" else 0.01
        self.ks, self.vs = ((s * np.exp(0.5 * rng.standard_normal(shape[:2] + (page // block,)))).astype(np.float32)
                            for _ in range(2))
        self.table = rng.permutation(n_pages)[:batch * max_pages].astype(np.int32).reshape(batch, max_pages)
        self.cap = max_pages * page

    def where(self, b, p):
        """(page, offset) of position p, None without a page."""
        pg = int(self.table[b, p // self.page])
        return (pg, p % self.page) if 0 <= pg < self.n_pages else None

    def append(self, k, v, lens, new):
        """k, v [batch][tokens][kv][dim] in any float type."""
        for b in range(len(lens)):
            L = min(max(int(lens[b]), 0), self.cap)
            end = min(L + int(new[b]), self.cap)
            for p0 in range(L // self.block * self.block, end, self.block):
                at = self.where(b, p0)
                if at is None or L >= end:
                    continue
                pg, off = at
                r0, r1 = max(L - p0, 0), min(end - p0, self.block)
                for x, codes, scales in ((k, self.k, self.ks), (v, self.v, self.vs)):
                    for h in range(self.kv):
                        rows = np.asarray(x[b, p0 + r0 - L:p0 + r1 - L, h], np.float32)
                        fin = np.abs(rows[np.isfinite(rows)])
                        s1 = np.float32((fin.max() if fin.size else np.float32(0)) / TOP[self.code])
                        blk = codes[pg, h, off:off + self.block]
                        if r0 > 0:
                            s0 = scales[pg, h, off // self.block]
                            s1 = max(s0, s1)
                            if s0 != s1:
                                r = np.float32(s0 / (s1 if s1 > 0 else np.float32(1)))
                                blk[:r0] = encode(decode(blk[:r0], self.code).astype(np.float32) * r, self.code)
                        with np.errstate(over="ignore", invalid="ignore"):
                            blk[r0:r1] = encode(rows / s1 if s1 > 0 else np.zeros_like(rows), self.code)
                        scales[pg, h, off // self.block] = s1

    def dense(self, b, n):
        """K and V values [kv][n][dim] in 64 bits and which positions have a page."""
        K, V = np.zeros((self.kv, n, self.dim)), np.zeros((self.kv, n, self.dim))
        ok = np.zeros(n, bool)
        for p in range(n):
            at = self.where(b, p)
            if at is None:
                continue
            pg, off = at
            ok[p] = True
            K[:, p] = decode(self.k[pg, :, off], self.code) * self.ks[pg, :, off // self.block, None].astype(np.float64)
            V[:, p] = decode(self.v[pg, :, off], self.code) * self.vs[pg, :, off // self.block, None].astype(np.float64)
        return K, V, ok

    def attention(self, q, lens, new, scale):
        """(out [batch][tokens][heads][dim], weights [batch][kv][cap], sums of p |v| like out, the largest
        scale * sum |q k|) in 64 bits; out is NaN where a row is not written."""
        B, T, H, D = q.shape
        G = H // self.kv
        out = np.full(q.shape, np.nan)
        mag = np.zeros(q.shape)
        w = np.zeros((B, self.kv, self.cap))
        big = 0.0
        for b in range(B):
            L = min(max(int(lens[b]), 0), self.cap)
            n = int(new[b])
            total = min(L + n, self.cap)
            K, V, ok = self.dense(b, total)
            for t in range(n):
                sees = ok & (np.arange(total) <= L + t)
                for h in range(H):
                    x = scale * (K[h // G] @ q[b, t, h].astype(np.float64))
                    if not sees.any():
                        out[b, t, h] = 0
                        continue
                    big = max(big, abs(scale) * float((np.abs(K[h // G][sees]) @ np.abs(q[b, t, h].astype(np.float64))).max()))
                    e = np.where(sees, np.exp(x - x[sees].max()), 0)
                    p = e / e.sum()
                    out[b, t, h] = p @ V[h // G]
                    mag[b, t, h] = p @ np.abs(V[h // G])
                    w[b, h // G, :total] += p
        return out, w, mag, big

    def evict(self, keep, first, recent, seen, lens, w, pos):
        """(lens, w, pos) after eviction; codes and scales change in place."""
        lens, w, pos = lens.copy(), w.copy(), pos.copy()
        for b in range(len(lens)):
            n = min(max(int(lens[b]), 0), self.cap)
            for h in range(self.kv):
                if n <= keep:
                    w[b, h, n:] = 0
                    continue
                safe = (pos[b, h, :n] < first) | (pos[b, h, :n] >= seen[b] - recent)
                val = np.where(np.isnan(w[b, h, :n]), -np.inf, w[b, h, :n]).astype(np.float64)
                isnan = np.isnan(w[b, h, :n])
                order = np.lexsort((np.arange(n), isnan, -val, ~safe))
                stays = np.zeros(n, bool)
                stays[order[:keep]] = True
                src = np.arange(keep)
                src[~stays[:keep]] = keep + np.nonzero(stays[keep:])[0]
                places = [self.where(b, int(s)) for s in src]
                for codes, scales in ((self.k, self.ks), (self.v, self.vs)):
                    rows = np.array([codes[a[0], h, a[1]] if a else np.zeros(self.dim, np.uint8) for a in places])
                    old = np.array([scales[a[0], h, a[1] // self.block] if a else 0 for a in places], np.float32)
                    for p0 in range(0, keep, self.block):
                        r = slice(p0, p0 + self.block)
                        at = self.where(b, p0)
                        if at is None or (src[r] == np.arange(p0, p0 + self.block)).all():
                            continue
                        s1 = old[r].max()
                        for i in range(p0, p0 + self.block):
                            y = rows[i]
                            if places[i] and old[i] != s1:
                                f = np.float32(old[i] / (s1 if s1 > 0 else np.float32(1)))
                                y = encode(decode(y, self.code).astype(np.float32) * f, self.code)
                            codes[at[0], h, at[1] + i - p0] = y
                        scales[at[0], h, at[1] // self.block] = s1
                w[b, h, :keep], pos[b, h, :keep] = w[b, h, src], pos[b, h, src]
                w[b, h, keep:] = 0
                pos[b, h, keep:] = seen[b] + np.arange(pos.shape[2] - keep)
            lens[b] = min(n, keep)
        return lens, w, pos
