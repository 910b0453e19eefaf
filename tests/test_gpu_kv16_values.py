"""Attention over a bf16 cache whose values come near the type's end: weights do not carry them past fp32's.

Values of 4e37, the others 1, lie at positions whose scores are up to 2^7.5 times as heavy as what came before them: a weight
against an older reference must not be that much above 1.  No channel has more than three of them in a part.

Bound.  That of the tests of ordinary values: a score's error dx goes into weights twice, weights are rounded by half a
step, the output by another; sums and exp2 add 2^-20.
"""
import numpy as np
import pytest

from kv16_ref import HALF, Cache, rounded
from test_gpu_kv16 import OnDevice, attend, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,T,heads,kv,dim,prefix", [(1, 1, 2, 2, 64, 600), (2, 1, 28, 4, 128, 300), (40, 1, 14, 2, 64, 20), (2, 60, 4, 2, 128, 300),
                                                         (130, 1, 64, 64, 64, 600)])
@pytest.mark.parametrize("block,step", [(16, 0.5), (16, 3.0), (16, 5.2), (128, 5.2), (64, 2.6)])
def test_large_values(batch, T, heads, kv, dim, prefix, block, step):
    rng = np.random.default_rng(batch * T + heads)
    page, own = 64, 300
    ref = Cache(batch, -(-(own + T) // page), -(-prefix // page), prefix, kv, dim, page, "bf16", rng)
    lens = rng.integers(200, own + 1, batch)
    ref.k[:], ref.v[:] = 0, 1
    for ids, n in [(ref.prefix_table, prefix)] + [(ref.table[b], lens[b] + T) for b in range(batch)]:
        for p in range(n):  # channel 0 holds the score, in natural units; it rises by `step` a block, up to 5.2
            pg, off = ref.slot(ids, p)
            ref.k[pg, :, off, 0] = min(step * (p // block), 5.2)
        for p in range(17, n, 16):
            pg, off = ref.slot(ids, p)
            ref.v[pg, :, off, p % dim] = 4e37 if p < 17 + 16 * 12 else 1
    ref.k, ref.v = rounded(ref.k, "bf16"), rounded(ref.v, "bf16")
    q = np.zeros((batch, T, heads, dim))
    q[..., 0] = 1.0
    got = attend(OnDevice(ref), q, lens, None, scale=1.0)
    assert np.isfinite(got).all()
    want, _ = ref.attention(rounded(q, "bf16"), lens, [T] * batch, 1.0)
    dx = (dim + 8) * 2.0 ** -23 * 5.2 + 2.0 ** -20
    near(got, want, np.abs(want) * (2.02 * HALF["bf16"] + 2 * dx + 2.0 ** -20))
