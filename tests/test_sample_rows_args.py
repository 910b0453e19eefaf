"""Refusals of n730_sample_rows, and the tests' own statement of its rule (addresses are never read here)."""
import numpy as np
import pytest

from n730_b200 import _lib, sampling
from sample_ref import sample

A = 1 << 20


def refused(code, **kw):
    a = dict(logits=A, dtype="f32", batch=2, vocab=100, u=A, tokens=A)
    a.update(kw)
    plain = [a.pop(n) for n in ("logits", "dtype", "batch", "vocab", "u", "tokens")]
    with pytest.raises(_lib.N730Error) as e:
        sampling.sample_rows(*plain, **a)
    assert e.value.code == code, e.value


@pytest.mark.parametrize("kw,code", [({"logits": 0}, -12), ({"u": 0}, -12), ({"tokens": 0}, -12), ({"batch": 0}, -13),
                                     ({"batch": (1 << 24) + 1}, -13), ({"vocab": 0}, -13), ({"vocab": (1 << 24) + 1}, -13),
                                     ({"ld": 99}, -13), ({"logits": A + 2}, -13), ({"logits": A + 1, "dtype": "f16"}, -13),
                                     ({"u": A + 2}, -13), ({"tokens": A + 1}, -13), ({"temperature": A + 1}, -13),
                                     ({"top_k": A + 2}, -13), ({"top_p": A + 3}, -13), ({"min_p": A + 1}, -13),
                                     ({"prob": A + 2}, -13), ({"kept": A + 2}, -13)])
def test_refusals(kw, code):
    refused(code, **kw)


def test_unknown_type():
    assert _lib.cuda().n730_sample_rows(A, 3, 1, 10, 10, None, None, None, None, A, A, None, None, None) == -13


def test_rule():
    x = np.log([0.1, 0.4, 0.1, 0.25, 0.15])
    assert sample(x, 0, 0, 1, 0, 0.9)[0] == {1}
    assert sample(x, 1, 2, 1, 0, 0.99) == ({3}, {(3, 2): pytest.approx(0.25 / 0.65)}, {2})
    assert sample(x, 1, 0, 0.5, 0, 0.99)[2] == {2}          # 0.4 + 0.25 reaches 0.5
    assert sample(x, 1, 2, 0.5, 0, 0.99)[2] == {1}          # 0.4 reaches half of 0.65
    assert sample(x, 1, 0, 1, 0.3, 0.99)[2] == {3}          # 0.15 >= 0.3 * 0.4 > 0.1
    assert sample(x, 1, 0, 1, 0, 0.999)[0] == {2}           # ties by index: the later of the equal ones
    assert sample(x, 1, 0, 1, 2.0, 0.999)[2] == {1}         # one token is always kept
    assert sample([np.nan, -np.inf], 1, 0, 1, 0, 0.5)[0] == {-1}
    assert sample([0, np.inf, np.inf], 1, 0, 1, 0, 0.6) == ({2}, {(2, 3): 0.5}, {3})
