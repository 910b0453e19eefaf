"""Refusals of the 16-bit cache's and the rotary's calls: every bad argument is turned into a return code on the
host, before any device work (addresses here are never read); and the rotary's frequencies, which are host work."""
import ctypes as C

import numpy as np
import pytest

from n730_b200 import _lib, kv16

A = 1 << 20  # an address that no refused call touches
GOOD = dict(n_pages=8, max_pages=4, n_kv=2, head_dim=64, page_size=64, dtype="f16", prefix_table=A, prefix_pages=3, prefix_len=A)


def cache(**kw):
    ptrs = [kw.pop(n, A) for n in ("k", "v", "block_table")]
    dtype = kw.pop("code", None)
    c = kv16.KV16Cache(*ptrs, **{**GOOD, **kw})
    if dtype is not None:
        c.c.dtype = dtype
    return c


def turn(**kw):
    r = kv16.Rotary(kw.pop("freq", A), kw.pop("dim", 64), **{k: v for k, v in kw.items() if k != "code"})
    if "code" in kw:
        r.c.layout = kw["code"]
    return r


def refused(call, code):
    with pytest.raises(_lib.N730Error) as e:
        call()
    assert e.value.code == code, e.value


BAD_CACHES = [({"k": 0}, -12), ({"v": 0}, -12), ({"block_table": 0}, -12), ({"prefix_table": 0}, -12), ({"prefix_len": 0}, -12),
              ({"k": A + 8}, -13), ({"v": A + 2}, -13), ({"code": 0}, -13), ({"code": 3}, -13), ({"head_dim": 96}, -14),
              ({"head_dim": 256}, -14), ({"page_size": 24}, -13), ({"page_size": 0}, -13), ({"page_size": 8}, -13), ({"n_kv": 0}, -13),
              ({"n_pages": 0}, -13), ({"max_pages": 0}, -13), ({"prefix_pages": -1}, -13), ({"block_table": A + 1}, -13),
              ({"prefix_table": A + 2}, -13), ({"prefix_len": A + 1}, -13), ({"n_pages": 1 << 24, "n_kv": 8}, -13),
              ({"max_pages": 1 << 24}, -13), ({"prefix_pages": 1 << 24}, -13)]


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_bad_cache(kw, code):
    c = cache(**kw)
    heads = 8 * max(c.c.n_kv, 1)
    refused(lambda: c.append(A, A, "f16", 1, 1, A), code)
    refused(lambda: c.attention_workspace(1, 1, heads), code)
    refused(lambda: c.attention(A, A, 1, 1, heads, A, ws=A, ws_bytes=1 << 40), code)


def test_pool_of_more_rows_than_64_bits_count():
    """2^30 pages of 2^14 heads and 2^20 positions: their product is 2^64."""
    c = cache(n_pages=1 << 30, n_kv=1 << 14, page_size=1 << 20, max_pages=1, prefix_pages=1)
    refused(lambda: c.attention_workspace(1, 1, 1 << 14), -13)


def test_null_cache():
    lib = _lib.cuda()
    assert lib.n730_kv16_append(None, None, None, 0, None, 0, 0, A, A, 128, 1, 1, 1, A, None, None, None) == -12
    assert lib.n730_kv16_attention_ws(None, 1, 1, 2) == -12
    assert lib.n730_kv16_attention(None, A, 128, 1, 1, 2, 1.0, A, None, A, 128, A, 1 << 40, None) == -12


def test_no_prefix_needs_no_table():
    assert cache(prefix_pages=0, prefix_table=0, prefix_len=0).attention_workspace(1, 1, 2) > 0


def test_append_arguments():
    c = cache()

    def call(**kw):
        a = dict(k=A, v=A, dtype="f16", batch=1, tokens=1, lens=A)
        a.update(kw)
        return lambda: c.append(a.pop("k"), a.pop("v"), a.pop("dtype"), a.pop("batch"), a.pop("tokens"), a.pop("lens"), **a)

    for name in ("k", "v", "lens"):
        refused(call(**{name: 0}), -12)
    for kw in (dict(batch=0), dict(batch=65536), dict(tokens=0), dict(tokens=(1 << 24) + 1), dict(ld=127), dict(k=A + 1),
               dict(dtype="f32", v=A + 2), dict(lens=A + 2), dict(new=A + 1), dict(pos=A + 3)):
        refused(call(**kw), -13)
    q = dict(q=A, q_out=A, heads=4, rotary=turn())
    refused(call(**{**q, "q_out": 0}), -12)
    refused(call(**{**q, "q": 0}), -12)
    refused(call(**{**q, "rotary": None}), -13)
    refused(call(**{**q, "heads": 0, "ldq": 256, "ldqo": 256}), -13)
    refused(call(**{**q, "ldq": 255}), -13)
    refused(call(**{**q, "ldqo": 255}), -13)
    refused(call(**{**q, "ldq": 300, "ldqo": 256}), -13)  # in place with two strides
    refused(call(**{**q, "q": A + 1}), -13)
    assert c.lib.n730_kv16_append(c._ref, None, None, 0, None, 0, 0, A, A, 128, 5, 1, 1, A, None, None, None) == -13


BAD_TURNS = [({"freq": 0}, -12), ({"freq": A + 4}, -13), ({"dim": 0}, -13), ({"dim": 63}, -13), ({"dim": 66}, -13), ({"dim": -2}, -13),
             ({"code": 2}, -13), ({"factor": float("nan")}, -13), ({"factor": float("inf")}, -13)]


@pytest.mark.parametrize("kw,code", BAD_TURNS)
def test_bad_rotary(kw, code):
    refused(lambda: turn(**kw).apply(A, A, "f16", 1, 1, 64, A), code)
    refused(lambda: cache().append(A, A, "f16", 1, 1, A, rotary=turn(**kw)), code)


def test_rotary_arguments():
    r = turn()
    refused(lambda: r.apply(0, A, "f32", 1, 1, 64, A), -12)
    refused(lambda: r.apply(A, 0, "f32", 1, 1, 64, A), -12)
    refused(lambda: r.apply(A, A, "f32", 1, 1, 64, 0), -12)
    for args, kw in (((A, A, "f32", 0, 1, 64, A), {}), ((A, A, "f32", 1 << 31, 1, 64, A), {}), ((A, A, "f32", 1, 0, 64, A), dict(ldx=64, ldy=64)),
                     ((A, A, "f32", 1, 1, 62, A), {}), ((A, A, "f32", 1, 1, 514, A), {}), ((A, A, "f32", 1, 2, 64, A), dict(ldx=127)),
                     ((A, A, "f32", 1, 2, 64, A), dict(ldy=127)), ((A, A, "f32", 1, 2, 64, A), dict(ldx=130)), ((A + 2, A, "f32", 1, 1, 64, A), {}),
                     ((A, A + 1, "f16", 1, 1, 64, A), {}), ((A, A, "f32", 1, 1, 64, A + 2), {})):
        refused(lambda: r.apply(*args, **kw), -13)
    assert r.lib.n730_rotary(None, A, 64, A, 64, 0, 1, 1, 64, A, None) == -12
    assert r.lib.n730_rotary(r._ref, A, 64, A, 64, 3, 1, 1, 64, A, None) == -13


def test_attention_arguments():
    c = cache()
    need = c.attention_workspace(2, 3, 14)

    def call(**kw):
        a = dict(q=A, out=A, batch=2, tokens=3, heads=14, lens=A, ws=A, ws_bytes=need)
        a.update(kw)
        return lambda: c.attention(a.pop("q"), a.pop("out"), a.pop("batch"), a.pop("tokens"), a.pop("heads"), a.pop("lens"), **a)

    for name in ("q", "out", "lens", "ws"):
        refused(call(**{name: 0}), -12)
    for kw in (dict(heads=13), dict(heads=0, ldq=64, ldo=64), dict(tokens=0), dict(tokens=(1 << 20) + 1), dict(batch=0), dict(batch=4097),
               dict(ldq=14 * 64 - 1), dict(ldo=14 * 64 - 1), dict(ws_bytes=need - 1), dict(ws=A + 4), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(q=A + 1), dict(out=A + 1), dict(lens=A + 2), dict(new=A + 2)):
        refused(call(**kw), -13)


def test_frequencies():
    i = np.arange(0, 64, 2) / 64
    f, m = kv16.frequencies(64, 1e6)
    assert np.allclose(f, 1e6 ** -i, rtol=1e-14) and m == 1
    assert np.allclose(kv16.frequencies(64, 1e6, "linear", factor=8)[0], 1e6 ** -i / 8, rtol=1e-14)
    f, m = kv16.frequencies(64, 1e4, "base", factor=4)
    assert f[0] == 1 and np.isclose(f[-1], 1e4 ** -i[-1] / 4, rtol=1e-12) and m == 1  # the slowest pair is slowed by the factor
    f, m = kv16.frequencies(64, 1e4, "ramp", factor=4, trained=4096, low=1, high=32)
    g = 1e4 ** -i
    turns = 4096 * g / (2 * np.pi)
    assert np.allclose(f[turns > 40], g[turns > 40], rtol=1e-14) and np.allclose(f[turns < 0.8], g[turns < 0.8] / 4, rtol=1e-14)
    between = (turns > 1.5) & (turns < 25)
    assert between.any() and np.all(f[between] < g[between]) and np.all(f[between] > g[between] / 4)
    assert m == pytest.approx(0.1 * np.log(4) + 1, rel=1e-6)
    f, m = kv16.frequencies(64, 1e4, "bands", factor=4, trained=4096, low=1, high=4)
    keep = np.clip((turns - 1) / 3, 0, 1)
    assert np.allclose(f, g / 4 * (1 - keep) + g * keep, rtol=1e-12) and m == 1


@pytest.mark.parametrize("args,kw", [((63,), {}), ((0,), {}), ((64, 1.0), {}), ((64, float("nan")), {}), ((64, 1e4, "linear"), dict(factor=0.5)),
                                     ((64, 1e4, "ramp"), dict(factor=2, trained=0)), ((64, 1e4, "bands"), dict(factor=2, trained=9, low=4, high=4)),
                                     ((2, 1e4, "base"), dict(factor=2)), ((64, 1e4, "ramp"), dict(factor=2, trained=9, low=0))])
def test_bad_frequencies(args, kw):
    refused(lambda: kv16.frequencies(*args, **kw), -13)


def test_bad_frequency_pointers():
    lib, m = _lib.cuda(), C.c_float()
    assert lib.n730_rotary_frequencies(64, 1e4, 0, 1.0, 1.0, 2.0, 0, None, C.byref(m)) == -12
    f = np.empty(32)
    assert lib.n730_rotary_frequencies(64, 1e4, 5, 1.0, 1.0, 2.0, 0, f.ctypes.data, C.byref(m)) == -13
