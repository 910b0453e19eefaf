"""n730_sample_rows at numbers of 1 and more, which count as the largest below 1: 1 - 2^-24, as fp32 holds it.

No bound: the last token with a mass has 2^-20 of it or more, and what follows has none at all.
"""
import numpy as np
import pytest

from test_gpu_sample_rows import draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("u", [1 - 2.0 ** -24, 1.0, 1.5, np.inf])
@pytest.mark.parametrize("V,allowed,lowest", [(100, 7, -3.4e38), (5000, 20, -1e9), (152064, 30, -3.4e38), (152064, 3000, -1e4)])
def test_nothing_without_a_mass(V, allowed, lowest, u):
    """Rows masked by low finite values: the answer is an allowed token however many are kept."""
    rng = np.random.default_rng(V + allowed)
    x = np.full((5, V), lowest)
    for r in range(5):
        x[r, rng.permutation(V)[:allowed]] = rng.standard_normal(allowed)
    (tok, prob, kept), held = draw(x, "f32", 1.0, [0, allowed + 5, min(V, 600), allowed + 1, 0], [1, 1, 1, 0.999999, 1], 0.0, u)
    # the last kept token that has a mass
    last = [np.lexsort((np.arange(V), -row))[min(allowed, n) - 1] for row, n in zip(held, (V, allowed + 5, 600, V, V))]
    assert list(tok[[0, 1, 2, 4]]) == [last[r] for r in (0, 1, 2, 4)]
    assert held[3, tok[3]] > lowest and np.all(prob > 0)
    assert list(kept[[0, 1, 4]]) == [V, min(V, allowed + 5), V]
