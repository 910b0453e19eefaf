"""The largest row of n730_sample_rows is 2^23 logits, one more is refused (addresses are never read here)."""
import pytest

from n730_b200 import _lib, sampling

A = 1 << 20


@pytest.mark.parametrize("vocab,ld", [((1 << 23) + 1, 0), (1 << 24, 0), ((1 << 23) + 1, 1 << 24)])
def test_rows_that_are_too_long(vocab, ld):
    with pytest.raises(_lib.N730Error) as e:
        sampling.sample_rows(A, "f32", 2, vocab, A, A, ld=ld)
    assert e.value.code == -13
