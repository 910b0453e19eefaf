"""Refusals of the 8-bit key/value cache calls: every bad argument is turned into a return code on
the host, before any device work (addresses here are never read)."""
import numpy as np
import pytest

from kv8_ref import E4M3, encode
from n730_b200 import _lib, kv8

A = 1 << 20  # an address that no refused call touches
GOOD = dict(n_pages=8, max_pages=4, n_kv=2, head_dim=64, page_size=64, block=16, code="int8")


def cache(**kw):
    ptrs = [kw.pop(n, A) for n in ("k_codes", "v_codes", "k_scales", "v_scales", "block_table")]
    c = kv8.KV8Cache(*ptrs, **{**GOOD, **{k: v for k, v in kw.items() if k in GOOD and k != "code"}})
    if "code" in kw:
        c.c.code = kw["code"]
    return c


def refused(call, code):
    with pytest.raises(_lib.N730Error) as e:
        call()
    assert e.value.code == code, e.value


BAD_CACHES = [({"k_codes": 0}, -12), ({"v_codes": 0}, -12), ({"k_scales": 0}, -12), ({"v_scales": 0}, -12),
              ({"block_table": 0}, -12), ({"k_codes": A + 8}, -13), ({"code": 2}, -13), ({"head_dim": 96}, -14),
              ({"head_dim": 256}, -14), ({"block": 8}, -13), ({"block": 48}, -13), ({"page_size": 24}, -13),
              ({"page_size": 0}, -13), ({"block": 64, "page_size": 96}, -13), ({"n_kv": 0}, -13), ({"n_pages": 0}, -13),
              ({"max_pages": 0}, -13), ({"k_scales": A + 2}, -13), ({"block_table": A + 1}, -13), ({"n_pages": 1 << 24, "n_kv": 8}, -13), ({"max_pages": 1 << 25}, -13)]


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_bad_cache(kw, code):
    c = cache(**kw)
    refused(lambda: c.append(A, A, "f16", 1, 1, A), code)
    refused(lambda: c.read(A, A, "f16", 1, 1, A), code)
    refused(lambda: c.attention(A, A, "f16", 1, 1, 8 * max(c.c.n_kv, 1), A, ws=A, ws_bytes=1 << 40), code)
    refused(lambda: c.attention_workspace(1, 1, 8 * max(c.c.n_kv, 1)), code)
    refused(lambda: c.evict_workspace(1, 64), code)
    refused(lambda: c.evict(1, 64, A, A, A, A, A, A, 1 << 31, seen=A, ws=A, ws_bytes=1 << 40), code)


def test_null_cache():
    lib = _lib.cuda()
    assert lib.n730_kv8_append(None, A, A, 1, 128, 1, 1, A, None, None) == -12
    assert lib.n730_kv8_read(None, A, A, 1, 128, 1, 1, None, A, None) == -12
    assert lib.n730_kv8_attention_ws(None, 1, 1, 2, 0) == -12
    assert lib.n730_kv8_evict_ws(None, 1, 16) == -12


def test_append_and_read_arguments():
    c = cache()
    for call in (c.append, c.read):
        refused(lambda: call(0, A, "f16", 1, 1, A), -12)
        refused(lambda: call(A, 0, "f16", 1, 1, A), -12)
        refused(lambda: call(A, A, "f16", 1, 1, 0), -12)
        refused(lambda: call(A, A, "f16", 0, 1, A), -13)
        refused(lambda: call(A, A, "f16", 65536, 1, A), -13)
        refused(lambda: call(A, A, "f16", 1, 0, A), -13)
        refused(lambda: call(A, A, "f16", 1, -3, A), -13)
        refused(lambda: call(A, A, "f16", 1, 1, A, ld=127), -13)
        refused(lambda: call(A + 1, A, "f16", 1, 1, A), -13)
        refused(lambda: call(A, A + 2, "f32", 1, 1, A), -13)
        refused(lambda: call(A, A, "f16", 1, 1, A + 2), -13)
    assert c.lib.n730_kv8_append(c._ref, A, A, 3, 128, 1, 1, A, None, None) == -13
    assert c.lib.n730_kv8_read(c._ref, A, A, -1, 128, 1, 1, None, A, None) == -13


def test_attention_arguments():
    c = cache()
    need = c.attention_workspace(2, 3, 14, weights=True)
    assert need > c.attention_workspace(2, 3, 14) > 0

    def call(**kw):
        a = dict(q=A, out=A, dtype="f16", batch=2, tokens=3, heads=14, lens=A, ws=A, ws_bytes=need, w_out=A, ld_w=256)
        a.update(kw)
        return lambda: c.attention(a.pop("q"), a.pop("out"), a.pop("dtype"), a.pop("batch"), a.pop("tokens"),
                                   a.pop("heads"), a.pop("lens"), **a)

    for name in ("q", "out", "lens", "ws"):
        refused(call(**{name: 0}), -12)
    refused(call(heads=13), -13)
    refused(call(heads=0), -13)
    refused(call(tokens=0), -13)
    refused(call(batch=0), -13)
    refused(call(batch=5000), -13)
    refused(call(ldq=14 * 64 - 1), -13)
    refused(call(ldo=14 * 64 - 1), -13)
    refused(call(ld_w=255), -13)
    refused(call(w_in=A, w_out=0), -13)
    refused(call(ws_bytes=need - 1), -13)
    refused(call(ws=A + 4), -13)
    refused(call(scale=float("nan")), -13)
    refused(call(q=A + 1), -13)
    refused(call(out=A + 1), -13)
    refused(call(dtype="f32", q=A + 2), -13)
    refused(call(lens=A + 2), -13)
    refused(call(w_out=A + 1), -13)
    refused(lambda: cache(max_pages=1 << 20).attention_workspace(4096, 1, 2), -13)  # 2^31 tiles
    refused(lambda: cache(n_kv=1).attention_workspace(1, 1, 8193), -13)
    refused(lambda: cache().attention_workspace(4096, 1 << 20, 18), -13)  # more rows than a grid has CTAs for
    refused(call(scale=float("inf")), -13)
    assert c.lib.n730_kv8_attention(c._ref, A, 7, 896, 2, 3, 14, 1.0, A, None, A, 896, None, None, 0, A, need, None) == -13


def test_evict_arguments():
    c = cache()
    need = c.evict_workspace(3, 64)

    def call(**kw):
        a = dict(batch=3, keep=64, lens=A, lens_out=A, w=A, w_out=A, pos=A, pos_out=A, ld_w=256, seen=A, first=4,
                 recent=8, ws=A, ws_bytes=need)
        a.update(kw)
        plain = [a.pop(n) for n in ("batch", "keep", "lens", "lens_out", "w", "w_out", "pos", "pos_out", "ld_w")]
        return lambda: c.evict(*plain, **a)

    for name in ("lens", "lens_out", "w", "w_out", "pos", "pos_out", "seen", "ws"):
        refused(call(**{name: 0}), -12)
    refused(call(keep=0), -13)
    refused(call(keep=24), -13)
    refused(call(keep=272), -13)
    refused(call(first=-1), -13)
    refused(call(recent=-1), -13)
    refused(call(first=60, recent=5), -13)
    refused(call(ld_w=255), -13)
    refused(call(ws_bytes=need - 1), -13)
    refused(call(ws=A + 2), -13)
    refused(call(pos=A + 2), -13)
    refused(call(w=A + 1), -13)


def test_reference_codes_round_to_nearest_even():
    """The tests' own e4m3 encoder against every code, every midpoint and torch's conversion."""
    import torch
    fin = E4M3[:127]
    assert np.array_equal(encode(fin, "e4m3"), np.arange(127))
    mid = ((fin[1:] + fin[:-1]) / 2).astype(np.float32)
    x = np.concatenate([mid, -mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(1e9))]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(encode(x, "e4m3"), want)
    assert encode(np.float32(1e6), "e4m3") == 126 and encode(np.float32(np.inf), "int8").view(np.int8) == 127


def test_model_batch():
    """A model with an 8-bit cache takes the batches that its attention does."""
    from n730_b200 import synthetic
    from n730_b200.engine import Engine
    with pytest.raises(RuntimeError, match="batch of 4097"):
        Engine(synthetic.SHAPES["tiny"], max_ctx=64, max_batch=4097, kv_bits=8)


def test_wait_check_arguments():
    lib = _lib.cuda()
    for ns, arrives in ((0, 0), (-1, 1), (1_000_000_001, 0), (1000, 3), (1000, -1)):
        assert lib.n730_kv8_wait_check(ns, arrives, None) == -13


def test_workspace_of_a_type():
    """A type's own workspace is enough for its calls and no more is asked for; the query without one covers all."""
    c = cache(max_pages=128, n_kv=8, head_dim=128, n_pages=4096)
    for batch, tokens, heads, weights in ((32, 300, 64, True), (1, 1, 64, False), (4, 3, 8, True), (2, 70, 16, False)):
        every = {t: c.attention_workspace(batch, tokens, heads, weights, dtype=t) for t in ("f32", "f16", "bf16")}
        assert c.attention_workspace(batch, tokens, heads, weights) == max(every.values())
        assert every["f16"] == every["bf16"]
        for t, need in every.items():
            with pytest.raises(_lib.N730Error, match=f"{need} needed"):
                c.attention(A, A, t, batch, tokens, heads, A, w_out=A if weights else 0, ld_w=8192, ws=A, ws_bytes=need - 1)
    every = [c.attention_workspace(32, 300, 64, True, dtype=t) for t in ("f16", "f32")]
    assert every[0] < 20 << 20 < 500 << 20 < every[1]
    assert c.lib.n730_kv8_attention_ws_of(c._ref, 3, 1, 1, 8, 0) == -13
    assert c.lib.n730_kv8_attention_ws_of(None, 1, 1, 1, 8, 0) == -12
