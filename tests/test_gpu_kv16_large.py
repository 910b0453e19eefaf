"""Attention over the 16-bit cache where scores are very large: finite queries and keys, as far as the types go.

Key p is a_p times a pattern of signs and query rows are powers of two times it, so that products and their sums are exact in
fp32 whatever their order, and rounding by the scale keeps their order.  Values of a_p differ by 2^-8 (bf16) or
2^-11 of themselves or not at all; with scores from 2^20 upwards (in powers of two of a weight) all keys but the
largest have no weight, and the answer is the mean of the largest ones' values.

Bound.  All weights of a row are equal, up to the reference of the part that they are summed in, which its join takes back
exactly; a part's weights are 2 to less than 1 of a power of two, and their rounding to the cache's type, half a step, is in
the numerator alone and may differ from part to part: half a step of the mean of |v|.  The output rounds once more; sums of n terms
in fp32 add n 2^-23 of the mean of |v|, exp2 2^-20 of it.
"""
import numpy as np
import pytest

from kv16_ref import HALF, TINY, Cache, rounded
from test_gpu_kv16 import OnDevice, attend, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,largest,query", [("f16", 60000.0, 2.0 ** e) for e in (-2, 3, 5, 8, 12, 14)] + [("f16", 3000.0, 2048.0)] +
                         [("bf16", 1e5, 2.0 ** e) for e in (0, 10, 20)] + [("bf16", 1e18, 2.0 ** e) for e in (-30, 0, 50)])
@pytest.mark.parametrize("batch,T,heads,kv,dim,prefix", [(2, 1, 14, 2, 64, 700), (3, 1, 28, 4, 128, 100), (40, 1, 14, 2, 64, 200), (2, 60, 4, 2, 128, 300),
                                                         (1, 150, 6, 1, 64, 40)])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_scores(dtype, largest, query, batch, T, heads, kv, dim, prefix, sign):
    rng = np.random.default_rng(batch + T + heads)
    page = 64
    ref = Cache(batch, -(-(50 + T) // page), -(-prefix // page), prefix, kv, dim, page, dtype, rng)
    pattern = rng.choice([-1.0, 1.0], dim)
    a = rounded(largest * rng.choice(np.linspace(0.2, 1.0, 40), ref.k.shape[:3]), dtype)
    ref.k = (a[..., None] * pattern).astype(np.float32)
    lens = rng.integers(0, 51, batch)
    q = np.broadcast_to(sign * query * pattern * rng.choice([1.0, 0.5, 2.0], (batch, T, heads, 1)), (batch, T, heads, dim))
    got = attend(OnDevice(ref), q, lens, None)
    want, bound = np.zeros(q.shape), np.zeros(q.shape)
    first = [ref.slot(ref.prefix_table, p) for p in range(prefix)]
    for b in range(batch):
        at = np.array(first + [ref.slot(ref.table[b], p) for p in range(lens[b] + T)]).T
        for t in range(T):
            pg, off = at[:, :prefix + lens[b] + t + 1]
            for h in range(kv):
                x = sign * a[pg, h, off]
                v = ref.v[pg, h, off][x == x.max()].astype(np.float64)
                rows = slice(h * heads // kv, (h + 1) * heads // kv)
                y, s = v.mean(0), np.abs(v).mean(0)
                want[b, t, rows] = y
                bound[b, t, rows] = 1.01 * HALF[dtype] * (np.abs(y) + s) + TINY[dtype] + (len(v) * 2.0 ** -23 + 2.0 ** -20) * s
    near(got, want, bound)
