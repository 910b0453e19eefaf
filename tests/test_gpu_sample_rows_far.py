"""n730_sample_rows on rows whose logits lie far from zero against their spread and temperature.

Bound.  Distances from the largest logit are exact wherever they carry a weight.  A token's mass in its bin is then off by
what fp32 makes of exp(y) - 1, y = (logit - edge) / T in [-2.1, 2^-6] at T of 0.01 and more: 2^-24 of its edge's weight for
the rounding of y and as much for the function's and the sum's, against a weight of e^-2.1 of the edge's or more: less
than 2^-19 of the mass.  A border compares two such sums: 2^-18.
"""
import numpy as np
import pytest

from test_gpu_sample_rows import check

pytestmark = pytest.mark.gpu
FAR = 2.0 ** -18


@pytest.mark.parametrize("hi,lo,n,T", [(21868.0, 21867.0, 1000, 1.0), (5800.25, 5800.0, 1000, 1.0), (6500.25, 6500.0, 3000, 0.5),
                                       (-21867.0, -21868.0, 20000, 1.0), (1e6, 1e6 - 0.0625, 2000, 0.05), (3e7, 3e7 - 2, 1500, 2.0),
                                       (1.0, 1.0 - 2.0 ** -23, 4000, 1e-7), (65504.0, 65472.0, 1100, 40.0)])
def test_rows_of_two_values(hi, lo, n, T):
    """Both values are drawn as often as they should be, and cuts between them are found."""
    rng = np.random.default_rng(n)
    x = np.empty((12, 2 * n))
    for r in range(12):
        at = rng.permutation(2 * n)
        x[r, at[:n]], x[r, at[n:]] = hi, lo
    u = np.r_[0, np.linspace(0.02, 0.98, 10), 1 - 2.0 ** -24]
    check(x, "f32", T, 0, 1.0, 0.0, u, slack=FAR)
    check(x, "f32", T, [0, 0, 0, 0, n - 7, n, n + 1, n + 300, 2 * n - 1, n + 300, 0, n + 300], [0.3, 0.5, 0.73, 0.9, 1, 1, 1, 1, 1, 0.9, 0.99, 0.999],
          [0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0.9, 0.1], u, slack=FAR)


@pytest.mark.parametrize("offset", [-5e3, 2e4, 1e5, -4e5, 1e6, -1.6e7, 3e7, 1e12])
def test_rows_with_an_offset(offset):
    """Gaussian rows of many spreads around a far value, at many temperatures, uncut and with cuts that bins settle."""
    rng = np.random.default_rng(abs(int(offset)) % 1000)
    base = rng.standard_normal((5, 9000))
    step = np.spacing(np.float32(abs(offset))).astype(float)
    for spread in (0.01, 0.25, 2.2, 8.0, 30.0, 3 * step):
        x = offset + spread * base
        for T in (0.01, 0.05, 0.1, 1.0, 2.0, 2 * step + 0.01):
            check(x, "f32", T, [0, 0, 600, 3000, 0], [1.0, 0.9, 0.99, 1.0, 1.0], [0, 0, 0, 0, 0.01], rng.random(5), slack=FAR)


@pytest.mark.parametrize("dtype,offset,spread,T", [("f16", 6e4, 300.0, 1.0), ("f16", -5e3, 20.0, 0.1), ("bf16", 1e6, 2e4, 1.0), ("bf16", 300.0, 3.0, 0.05),
                                                   ("bf16", 1e30, 1e29, 1.0)])
def test_coarse_types(dtype, offset, spread, T):
    rng = np.random.default_rng(int(spread % 1000))
    x = offset + spread * rng.standard_normal((5, 40000))
    check(x, dtype, T, [0, 0, 600, 3000, 0], [1.0, 0.9, 0.99, 1.0, 1.0], [0, 0, 0, 0, 0.01], rng.random(5), slack=FAR)


@pytest.mark.parametrize("V", [152064, 600011])
def test_long_rows(V):
    """Several thousand tokens of a bin in a CTA, and rows that shared memory does not hold."""
    rng = np.random.default_rng(V)
    x = np.round(4e5 + 0.05 * rng.standard_normal((3, V)), 3)
    check(x, "f32", 0.05, [0, 0, 90000], [1.0, 0.95, 0.9], 0.0, rng.random(3), slack=FAR)
