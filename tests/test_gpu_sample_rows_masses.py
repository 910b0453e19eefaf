"""n730_sample_rows where bins of masses settle a row, held to what their arithmetic keeps.

Bound.  A token's mass in its bin is its edge's weight, in 64 bits, times exp(y), y = (logit - edge) / T in [-1/38, 2^-7].
The difference is exact or off by 2^-24 of itself, the quotient by 2^-23 of itself, the polynomial's last sums and
products by 3 2^-24 of exp(y) - 1: less than 2^-27 of the mass together.  In fixed point half a unit is lost, 2^-32 of the edge's
weight, or 2^-27 with the room that a bin of up to 128000 tokens a CTA is given.  A cumulative mass is off by 2^-26 of itself
then, and so is what it is compared with: an answer is accepted where its border lies within 2^-25 of the mass.
Tokens more than 40 temperatures below the largest have no mass: V e^-40, below 2^-38.
"""
import numpy as np
import pytest

from test_gpu_sample_rows import check, rows

pytestmark = pytest.mark.gpu
MASSES = 2.0 ** -25


@pytest.mark.parametrize("V,n,d,T", [(152064, 100000, 0.0155, 0.001), (152064, 30000, 0.018, 0.001), (152064, 100000, 0.0205, 0.002),
                                     (40000, 3000, 0.019, 0.0015), (5000, 4000, 0.0005, 2e-5), (32000, 20000, 0.3, 0.03),
                                     (152064, 90000, 0.6, 0.05)])
def test_crowd_below_one_at_small_temperatures(V, n, d, T):
    """A token, a crowd of equal ones some temperatures below it, and masked places far behind, so that the row's bins
    would be wide if they went by its spread."""
    rng = np.random.default_rng(n)
    x = np.full((16, V), -300.0)
    for r in range(16):
        at = rng.permutation(V)[:n + 1]
        x[r, at[1:]], x[r, at[0]] = -d, 0.0
    w = float(np.exp(np.float64(np.float32(-d)) / np.float64(np.float32(T))))
    u = 1 / (1 + n * w) + np.linspace(-1e-3, 1e-3, 16)  # around where the crowd begins
    check(x, "f32", T, 0, 1.0, 0.0, np.clip(u, 0, 0.99999), slack=MASSES)
    check(x[:6], "f32", T, [700, n, n + 1, n + 7, 0, 0], [1.0, 1.0, 0.99, 0.95, 0.9, 0.999], 0.0, rng.random(6), slack=MASSES)


@pytest.mark.parametrize("hi,lo,n,T", [(21868.0, 21867.0, 1000, 1.0), (-6500.0, -6500.25, 3000, 0.1), (3e7, 3e7 - 2, 1500, 0.5),
                                       (1.0, 1.0 - 2.0 ** -23, 4000, 1e-7), (0.0, -6e-31, 2000, 1e-30), (5e-31, -5e-31, 2000, 9e-31)])
def test_two_values(hi, lo, n, T):
    """Rows of two values, far from zero, near each other, or both."""
    rng = np.random.default_rng(n)
    x = np.full((12, 2 * n), lo)
    for r in range(12):
        x[r, rng.permutation(2 * n)[:n]] = hi
    u = np.r_[0, np.linspace(0.02, 0.98, 10), 1 - 2.0 ** -24]
    check(x, "f32", T, 0, 1.0, 0.0, u, slack=MASSES)
    check(x, "f32", T, [0, 0, 0, 0, n - 7, n, n + 1, n + 300, 2 * n - 1, n + 300, 0, n + 300], [0.3, 0.5, 0.73, 0.9, 1, 1, 1, 1, 1, 0.9, 0.99, 0.999],
          0.0, u, slack=MASSES)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [0.002, 0.02, 0.1, 0.3, 0.7, 1.0, 3.0])
def test_masses_at_all_temperatures(dtype, T):
    """Ordinary rows, uncut and with cuts that bins settle; top-k beyond the last bin of masses."""
    rng = np.random.default_rng(int(T * 1000))
    k = np.array([0, 0, 0, 600, 2000, 5000, 30000, 2000, 0, 0])
    p = np.array([1.0, 0.95, 0.5, 1.0, 0.9, 1.0, 0.999, 0.95, 1.0, 0.99])
    q = np.array([0, 0, 0, 0, 0, 1e-4, 0, 1e-3, 0, 1e-20])
    check(rows(rng, 10, 50257), dtype, T, k, p, q, rng.random(10), slack=MASSES)
    check(rows(rng, 10, 33000, peaks=24), dtype, T, k, p, q, rng.random(10), slack=MASSES)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_the_longest_row(dtype):
    """2^23 logits: half a unit is 2^-23 of an edge's weight there, and a sum is off by 2^-22 of itself."""
    rng = np.random.default_rng(23)
    check(2.2 * rng.standard_normal((2, 1 << 23)) + 5, dtype, [1.0, 0.3], [0, 300000], [0.99, 1.0], 0.0, rng.random(2), slack=2.0 ** -21)
