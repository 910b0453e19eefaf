"""Scales of the 16-bit cache's attention that cannot be held with their log2 e (addresses are never read here)."""
import pytest

from n730_b200 import _lib, kv16

A = 1 << 20


@pytest.mark.parametrize("scale", [3e38, -2.5e38])
def test_scale_times_log2e(scale):
    c = kv16.KV16Cache(A, A, A, n_pages=8, max_pages=4, n_kv=2, head_dim=64)
    with pytest.raises(_lib.N730Error) as e:
        c.attention(A, A, 1, 1, 2, A, scale=scale, ws=A, ws_bytes=1)
    assert e.value.code == -13 and "scale" in str(e.value)
