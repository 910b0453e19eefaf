"""The 8-bit key/value cache on the GPU against the plain numpy statement of it (``kv8_ref.py``).

Codes and scales are exact (the same fp32 quotients, products and roundings).  Attention is held to
    h |y| + u S + e S + n 2^-25 V,      S = sum p |v|, V = max |v|
with h the half step of the output type, u the half step of P's fp16 (0 for fp32 rows, whose P has two
terms), n 2^-25 V P's smallest fp16 step, and e = 2 dx with dx the error of a score: products are exact
in fp32 and the running sum of head_dim of them truncates, (head_dim + 8) 2^-23 of scale * sum |q k|,
times two because numerator and denominator both carry it; exp2 and the 2^-22 of a split query add 2^-20.
"""
import numpy as np
import pytest

from gpu_util import dev, torch
from kv8_ref import Cache, decode
from n730_b200 import kv8

pytestmark = pytest.mark.gpu
NP = {"f16": np.float16, "f32": np.float32}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def tt(dtype):
    t = torch()
    return {"f16": t.float16, "bf16": t.bfloat16, "f32": t.float32}[dtype]


def rounded(x, dtype):
    """x as the type holds it, in fp32."""
    return torch().from_numpy(np.ascontiguousarray(x, np.float32)).to(tt(dtype)).float().numpy()


class OnDevice:
    def __init__(self, ref: Cache):
        self.ref = ref
        self.t = {n: dev(getattr(ref, n)) for n in ("k", "v", "ks", "vs", "table")}
        self.h = kv8.KV8Cache(*(self.t[n].data_ptr() for n in ("k", "v", "ks", "vs", "table")), n_pages=ref.n_pages,
                              max_pages=ref.max_pages, n_kv=ref.kv, head_dim=ref.dim, page_size=ref.page,
                              block=ref.block, code=ref.code)

    def same_as_reference(self):
        for n in ("k", "v", "ks", "vs"):
            got, want = self.t[n].cpu().numpy(), getattr(self.ref, n)
            assert np.array_equal(got, want), f"{n}: {np.mean(got != want):.2g} of the entries differ"


def ints(x):
    return dev(np.asarray(x, np.int32))


def make(rng, batch=2, max_pages=3, kv=2, dim=64, page=64, block=16, code="int8", fill=None, spare=2):
    return Cache(batch * max_pages + spare, max_pages, batch, kv, dim, page, block, code, rng, fill)


def rows(rng, *shape):
    return rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[-2:]))


def append(d, k, v, dtype, lens, new=None, ld=0, stream=0, shift=0):
    """Both sides append; rows ld elements apart, `shift` elements into their buffer."""
    B, T, kv, D = k.shape
    ld = ld or kv * D
    t = torch()
    bufs = []
    for x in (k, v):
        buf = t.full((shift + B * T * ld,), 7.0, dtype=tt(dtype), device="cuda")
        buf[shift:].view(B * T, ld)[:, :kv * D] = dev(x.reshape(B * T, kv * D).astype(np.float32)).to(tt(dtype))
        bufs.append(buf[shift:])
    dl, dn = ints(lens), ints(new) if new is not None else None
    t.cuda.synchronize()
    d.h.append(bufs[0].data_ptr(), bufs[1].data_ptr(), dtype, B, T, dl.data_ptr(), new=dn.data_ptr() if new is not None else 0,
               ld=ld, stream=stream)
    t.cuda.synchronize()
    d.ref.append(rounded(k, dtype), rounded(v, dtype), lens, np.clip(new, 0, T) if new is not None else [T] * B)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim,page,block", [(64, 16, 16), (64, 32, 32), (64, 128, 64), (128, 64, 16), (128, 96, 32),
                                            (128, 64, 64)])
def test_append_exact(code, dtype, dim, page, block):
    """A prompt, single tokens that grow a block's scale and ones that do not, ragged counts."""
    rng = np.random.default_rng(dim + page + block)
    d = OnDevice(make(rng, 3, 4, 2, dim, page, block, code))
    lens = np.array([0, 5, page - 1])
    for new, T, amp in ((np.array([37, 0, 2]), 37, 1.0), (np.array([1, 1, 1]), 1, 5.0), (None, 1, 0.1),
                        (np.array([2, 9, -4]), 3, 20.0)):
        append(d, amp * rows(rng, 3, T, 2, dim), amp * rows(rng, 3, T, 2, dim), dtype, lens, new)
        d.same_as_reference()
        lens = lens + (np.clip(new, 0, T) if new is not None else T)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_edges(code):
    """Zeros, NaN and infinities, values that leave the codes' range, a full table, bad lengths and pages."""
    rng = np.random.default_rng(3)
    d = OnDevice(make(rng, 4, 2, 2, 64, 32, 16, code))
    d.ref.table[1, 0], d.ref.table[2, 1] = -1, d.ref.n_pages
    d.t["table"].copy_(dev(d.ref.table))
    k, v = rows(rng, 4, 40, 2, 64), rows(rng, 4, 40, 2, 64)
    k[0, :16] = 0
    k[0, 17, 0, :5] = [np.nan, np.inf, -np.inf, 3e38, -3e38]
    v[3, 2, 1, 7] = np.nan
    v[3, 20] = 1e-42
    append(d, k, v, "f32", np.array([0, 0, 20, 50]))  # 20 + 40 and 50 + 40 pass 64 positions
    d.same_as_reference()
    append(d, k, v, "f32", np.array([-7, 64, 63, 1 << 30]), np.array([1, 40, 99, 3]))
    d.same_as_reference()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("amp", [1.0, 2.0 ** -70])
def test_append_zeros_keep_their_sign(code, amp):
    """Zeros of both signs and values that round to them, by either way of dividing (scales below 2^-60 take the other)."""
    rng = np.random.default_rng(23)
    d = OnDevice(make(rng, 2, 2, 2, 64, 32, 16, code))
    k, v = amp * rows(rng, 2, 20, 2, 64), amp * rows(rng, 2, 20, 2, 64)
    for x in (k, v):
        x[..., ::4] = -0.0
        x[..., 1::8] *= 1e-5
        x[..., 2::8] = 0.0
    append(d, k, v, "f32", np.array([0, 7]))
    d.same_as_reference()


@pytest.mark.parametrize("dtype,extra,shift", [("f16", 8, 0), ("f16", 3, 0), ("bf16", 0, 1), ("f32", 5, 3), ("f16", 0, 8)])
def test_append_and_read_strides(dtype, extra, shift):
    """Rows inside wider rows, at addresses that are not 16-byte aligned."""
    rng = np.random.default_rng(5)
    t = torch()
    d = OnDevice(make(rng, 2, 2, 3, 64, 32, 16, "int8"))
    ld = 3 * 64 + extra
    lens = np.array([3, 17])
    append(d, rows(rng, 2, 9, 3, 64), rows(rng, 2, 9, 3, 64), dtype, lens, ld=ld, shift=shift)
    d.same_as_reference()
    y = [t.full((shift + 2 * 30 * ld,), 5.0, dtype=tt(dtype), device="cuda") for _ in range(2)]
    first, total = ints([-2, 10]), ints(lens + 9)
    d.h.read(y[0][shift:].data_ptr(), y[1][shift:].data_ptr(), dtype, 2, 30, total.data_ptr(), first=first.data_ptr(), ld=ld)
    t.cuda.synchronize()
    for b in range(2):
        n = int(lens[b]) + 9
        K, V, _ = d.ref.dense(b, n)
        for x, want in zip(y, (K, V)):
            assert (x[:shift] == 5).all()
            got = x[shift:].view(2, 30, ld)[b].float().cpu().numpy()
            assert (got[:, 3 * 64:] == 5).all()  # between the rows
            for i in range(30):
                p = (-2, 10)[b] + i
                w = want[:, p].astype(np.float32) if 0 <= p < n else np.zeros((3, 64), np.float32)
                assert np.array_equal(got[i, :3 * 64].reshape(3, 64), rounded(w, dtype))


def run_attention(d, q, dtype, lens, new=None, weights=None, scale=None, ws=None, ldq=0, ldo=0, stream=0, in_place=False,
                  fill=9.0):
    """(out, weights out) of the device call; out rows start from `fill`, weights out from -1."""
    t = torch()
    B, T, H, D = q.shape
    ldq, ldo = ldq or H * D, ldo or H * D
    dq = t.full((B * T, ldq), float("nan"), dtype=tt(dtype), device="cuda")
    dq[:, :H * D] = dev(q.reshape(B * T, H * D).astype(np.float32)).to(tt(dtype))
    out = t.full((B * T, ldo), fill, dtype=tt(dtype), device="cuda")
    dl, dn = ints(lens), ints(new) if new is not None else None
    w_in = dev(weights.astype(np.float32)) if weights is not None else None
    w_out = w_in if in_place else t.full_like(w_in, -1.0) if weights is not None else None
    need = d.h.attention_workspace(B, T, H, weights=weights is not None)
    ws = t.zeros(need, dtype=t.uint8, device="cuda") if ws is None else ws
    t.cuda.synchronize()
    d.h.attention(dq.data_ptr(), out.data_ptr(), dtype, B, T, H, dl.data_ptr(), new=dn.data_ptr() if new is not None else 0,
                  scale=scale, ldq=ldq, ldo=ldo, w_in=w_in.data_ptr() if weights is not None else 0,
                  w_out=w_out.data_ptr() if weights is not None else 0, ld_w=w_in.shape[2] if weights is not None else 0,
                  ws=ws.data_ptr(), ws_bytes=ws.numel(), stream=stream)
    t.cuda.synchronize()
    assert (out[:, H * D:] == fill).all()
    return (out[:, :H * D].float().cpu().numpy().reshape(q.shape).astype(np.float64),
            w_out.cpu().numpy() if weights is not None else None)


def tolerance(ref, dtype, want, mag, big):
    """(relative error of a weight, absolute tolerances of the outputs), as derived above."""
    dx = 2 * ((ref.dim + 8) * 2.0 ** -23 * big + 2.0 ** -20)
    vmax = max(float(np.nanmax(np.abs(decode(ref.v, ref.code)))) * float(ref.vs.max()), 1e-30)
    u = 0.0 if dtype == "f32" else 2.0 ** -11
    return dx, HALF[dtype] * np.abs(want) + (u + dx) * mag + ref.cap * 2.0 ** -25 * vmax + 2.0 ** -24


def near(got, want, tol):
    over = np.abs(got - want) / tol
    assert not (over > 1).any() and not np.isnan(over).any(), f"off by {np.max(over):.3g} of the tolerance"


def check_attention(d, q, dtype, lens, new=None, weights=None, scale=None, **kw):
    B, T, H, D = q.shape
    count = np.clip(new, 0, T) if new is not None else np.full(B, T)
    scale = D ** -0.5 if scale is None else scale
    out, w = run_attention(d, q, dtype, lens, new, weights, scale, **kw)
    want, p, mag, big = d.ref.attention(rounded(q, dtype), lens, count, scale)
    written = ~np.isnan(want)
    assert (out[~written] == 9.0).all(), "rows behind the new ones were written"
    dx, tol = tolerance(d.ref, dtype, want, mag, big)
    near(out[written], want[written], tol[written])
    if weights is not None:
        for b in range(B):
            L = min(max(int(lens[b]), 0), d.ref.cap)
            n = min(L + int(count[b]), d.ref.cap)
            exp = p[b, :, :n].copy()
            exp[:, :L] += weights[b, :, :L].astype(np.float32)
            assert (np.abs(w[b, :, :n] - exp) <= dx * p[b, :, :n] + 2.0 ** -22 * exp + 1e-9).all()
            if not kw.get("in_place"):
                assert (w[b, :, n:] == -1).all()
    return out, w


SHAPES = [  # kv, heads, dim, page, block
    (4, 28, 128, 64, 16), (2, 14, 64, 64, 64), (8, 64, 128, 64, 32), (1, 1, 64, 16, 16), (2, 2, 128, 32, 16),
    (1, 17, 64, 32, 32), (2, 64, 128, 96, 32)]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("kv,heads,dim,page,block", SHAPES)
def test_single_token(code, dtype, kv, heads, dim, page, block):
    """Ragged lengths from an empty cache on: tiles cut at each place, pages that end inside a tile's run."""
    rng = np.random.default_rng(heads * dim)
    lens = np.array([0, 1, 15, 16, 17, 2 * page - 1, 2 * page, 3 * page - 1])
    d = OnDevice(make(rng, len(lens), 3, kv, dim, page, block, code))
    q = 2 * rng.standard_normal((len(lens), 1, heads, dim))
    check_attention(d, q, dtype, lens, weights=rng.random((len(lens), kv, d.ref.cap)))


@pytest.mark.parametrize("code,dtype,kv,heads,dim,lens", [
    ("int8", "f16", 4, 28, 128, [2047]), ("int8", "f32", 4, 28, 128, [2047]), ("e4m3", "bf16", 2, 14, 64, [5000]),
    ("int8", "f16", 1, 8, 128, [9000, 3, 0, 700]), ("int8", "f32", 2, 16, 64, [1, 6000, 0, 17])])
def test_single_token_split(code, dtype, kv, heads, dim, lens):
    """Long contexts and few sequences: runs that many CTAs share, joined from parts."""
    rng = np.random.default_rng(11)
    d = OnDevice(make(rng, len(lens), max(lens) // 64 + 1, kv, dim, 64, 16, code))
    q = 2 * rng.standard_normal((len(lens), 1, heads, dim))
    out, w = check_attention(d, q, dtype, np.array(lens), weights=rng.random((len(lens), kv, d.ref.cap)))
    again, w2 = run_attention(d, q, dtype, np.array(lens), weights=np.zeros((len(lens), kv, d.ref.cap)))
    assert np.array_equal(out, again)  # whichever CTA joins


@pytest.mark.parametrize("code,dtype,kv,heads,dim,T,lens,new", [
    ("int8", "f16", 2, 14, 64, 5, [40, 0, 100], None), ("int8", "bf16", 4, 28, 128, 3, [70, 1, 0], [3, 0, 2]),
    ("e4m3", "f16", 1, 5, 128, 33, [0, 90], [33, 7]), ("int8", "f16", 2, 16, 128, 130, [0, 61], None),
    ("int8", "f16", 2, 4, 64, 190, [1, 0, 2], [190, 1, 64]), ("e4m3", "bf16", 2, 14, 64, 64, [128, 5], None),
    ("int8", "f32", 2, 4, 64, 9, [30, 0], None)])
def test_several_tokens(code, dtype, kv, heads, dim, T, lens, new):
    """Prompts and chunks: causal among the new rows, ragged counts, rows behind them untouched."""
    rng = np.random.default_rng(T)
    d = OnDevice(make(rng, len(lens), 3, kv, dim, 64, 16, code))
    q = 2 * rng.standard_normal((len(lens), T, heads, dim))
    check_attention(d, q, dtype, np.array(lens), None if new is None else np.array(new),
                    weights=rng.random((len(lens), kv, d.ref.cap)))
    check_attention(d, q, dtype, np.array(lens), None if new is None else np.array(new))


@pytest.mark.parametrize("code,dtype,kv,heads,dim,page,T,lens,new", [
    ("int8", "f16", 2, 8, 128, 64, 300, [1700, 0], None),                   # positions in shares
    ("e4m3", "bf16", 1, 14, 64, 48, 40, [2900, 700, 0], [40, 3, 0]),        # pages of three blocks
    ("int8", "bf16", 2, 8, 64, 16, 130, [1111], None),
    ("int8", "f16", 1, 65, 128, 128, 1, [1500, 0, 127], None),              # one token of many heads
    ("int8", "f16", 4, 64, 64, 64, 300, [740, 0], None),                    # shares in a last, partial wave of CTAs
    ("e4m3", "f16", 8, 32, 64, 64, 160, [900, 0, 129, 511], [160, 160, 0, 97])])
def test_prompts_over_many_tiles(code, dtype, kv, heads, dim, page, T, lens, new):
    """Chunks far into a context, with the positions in shares where there are few rows; scores that
    move the references from tile to tile."""
    rng = np.random.default_rng(T + page)
    d = OnDevice(make(rng, len(lens), (max(lens) + T) // page + 1, kv, dim, page, 16, code))
    q = 2 * rng.standard_normal((len(lens), T, heads, dim))
    q[:, ::5] *= 6
    out, _ = check_attention(d, q, dtype, np.array(lens), None if new is None else np.array(new),
                             weights=rng.random((len(lens), kv, d.ref.cap)))
    again, _ = run_attention(d, q, dtype, np.array(lens), None if new is None else np.array(new))
    assert np.array_equal(out, again)


@pytest.mark.parametrize("T", [1, 70])
def test_missing_pages_far_apart(T):
    """A long table most of whose pages are missing, whole tiles and shares of it among them."""
    rng = np.random.default_rng(T)
    d = OnDevice(make(rng, 2, 40, 1, 64, 64, 32, "int8"))
    d.ref.table[rng.random(d.ref.table.shape) < 0.7] = -1
    d.ref.table[0, :20] = d.ref.n_pages
    d.t["table"].copy_(dev(d.ref.table))
    for dtype in ("f16", "f32"):
        check_attention(d, rng.standard_normal((2, T, 4, 64)), dtype, np.array([2560 - T, 2011]),
                        weights=rng.random((2, 1, 2560)))


@pytest.mark.parametrize("T,heads", [(1, 6), (30, 6)])
def test_no_new_rows_and_shared_pages(T, heads):
    """A batch without a new row keeps its output and weights; two sequences that read the same pages agree."""
    rng = np.random.default_rng(T)
    d = OnDevice(make(rng, 3, 3, 2, 64, 64, 16, "int8"))
    d.ref.table[1] = d.ref.table[0]
    d.t["table"].copy_(dev(d.ref.table))
    q = rng.standard_normal((3, T, heads, 64))
    q[1] = q[0]
    lens, w = np.array([130, 130, 0]), rng.random((3, 2, 192))
    w[1] = w[0]
    check_attention(d, q, "f16", lens, np.zeros(3, int), weights=w)
    out, w = check_attention(d, q, "f16", lens, weights=w)
    assert np.array_equal(out[0], out[1]) and np.array_equal(w[0], w[1])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_many_sequences(dtype):
    """More sequences than CTAs, most of them short or empty."""
    rng = np.random.default_rng(6)
    B = 600
    d = OnDevice(make(rng, B, 3, 1, 64, 16, 16, "e4m3"))
    lens = rng.integers(0, 47, B) * (rng.random(B) < 0.6)
    check_attention(d, rng.standard_normal((B, 1, 3, 64)), dtype, lens, (rng.random(B) < 0.8).astype(int),
                    weights=rng.random((B, 1, 48)))


@pytest.mark.parametrize("heads", [80, 200])
def test_many_heads_of_one_kv_head(heads):
    """fp32 rows of more heads than a call's rows at a time, one token after the other."""
    rng = np.random.default_rng(heads)
    d = OnDevice(make(rng, 2, 3, 1, 64, 64, 16, "int8"))
    check_attention(d, rng.standard_normal((2, 3, heads, 64)), "f32", np.array([100, 0]), np.array([3, 2]),
                    weights=rng.random((2, 1, 192)))


def test_missing_pages_and_empty_rows():
    """Ids outside the pool are unseen positions; a row that sees none gives zeros."""
    rng = np.random.default_rng(2)
    d = OnDevice(make(rng, 3, 3, 2, 64, 32, 16, "int8"))
    d.ref.table[0, 1], d.ref.table[1, :], d.ref.table[2, 0] = -1, d.ref.n_pages + 5, -(1 << 31)
    d.t["table"].copy_(dev(d.ref.table))
    for T in (1, 4, 70):
        q = rng.standard_normal((3, T, 14, 64))
        lens = np.array([96 - T, 50 - min(T, 50), 64 - min(T, 64)])
        for dtype in ("f16", "f32"):
            out, w = check_attention(d, q, dtype, lens, np.array([T, min(T, 50), min(T, 64)]),
                                     weights=rng.random((3, 2, 96)))
            assert (out[1, :min(T, 50)] == 0).all()


@pytest.mark.parametrize("T", [1, 6, 80])
def test_codes_behind_the_last_position(T):
    """Rows that were never written may hold e4m3 NaN codes and any scale: nothing of them is seen."""
    rng = np.random.default_rng(4)
    d = OnDevice(make(rng, 2, 2, 2, 128, 64, 16, "e4m3", fill=0x7f))
    d.ref.ks[:] = d.ref.vs[:] = np.nan
    for n in ("ks", "vs"):
        d.t[n].copy_(dev(getattr(d.ref, n)))
    lens = np.array([0, 21])
    append(d, rows(rng, 2, 21, 2, 128), rows(rng, 2, 21, 2, 128), "f16", np.zeros(2, int), np.array([0, 21]))
    append(d, rows(rng, 2, T, 2, 128), rows(rng, 2, T, 2, 128), "f16", lens)
    out, _ = run_attention(d, rng.standard_normal((2, T, 6, 128)), "f16", lens)
    assert np.isfinite(out).all()


def test_scales_of_any_size():
    """V scales that differ by 2^20 between blocks, a zero scale, and scores far apart."""
    rng = np.random.default_rng(8)
    for T in (1, 70):
        d = OnDevice(make(rng, 1, 3, 2, 64, 64, 16, "int8"))
        d.ref.vs[:] = np.float32(0.01) * np.exp2(rng.integers(-12, 9, d.ref.vs.shape)).astype(np.float32)
        d.ref.vs.reshape(-1)[::5] = 0
        d.ref.ks.reshape(-1)[::7] = 0
        for n in ("ks", "vs"):
            d.t[n].copy_(dev(getattr(d.ref, n)))
        for dtype in ("f16", "f32"):
            check_attention(d, 4 * rng.standard_normal((1, T, 4, 64)), dtype, np.array([190 - T]))


@pytest.mark.parametrize("T", [1, 70])
def test_tiny_scales(T):
    """V scales down to fp32's smallest: blocks below 2^-100 add nothing, alone or beside others."""
    rng = np.random.default_rng(14)
    for tiny in (np.float32(1e-44), np.float32(1e-38), np.float32(2.0 ** -99)):
        for share in (1.0, 0.5):
            d = OnDevice(make(rng, 1, 3, 2, 64, 64, 16, "int8"))
            d.ref.vs[rng.random(d.ref.vs.shape) < share] = tiny
            d.t["vs"].copy_(dev(d.ref.vs))
            for dtype in ("bf16", "f32"):
                check_attention(d, rng.standard_normal((1, T, 4, 64)), dtype, np.array([180 - T]),
                                weights=rng.random((1, 2, 192)))


@pytest.mark.parametrize("T", [1, 70])
def test_scales_far_apart(T):
    """V scales from 2^-99 to 2^100 in one row's blocks: the softmax weights do not feel them."""
    rng = np.random.default_rng(15)
    for lo, hi in ((-99, 100), (-24, 60), (60, 100), (0, 100)):
        d = OnDevice(make(rng, 1, 6, 2, 64, 64, 16, "int8"))
        d.ref.vs[:] = np.exp2(rng.choice([lo, hi, 0], d.ref.vs.shape, p=[0.3, 0.2, 0.5])).astype(np.float32)
        d.t["vs"].copy_(dev(d.ref.vs))
        for dtype in ("bf16", "f32"):
            check_attention(d, rng.standard_normal((1, T, 4, 64)), dtype, np.array([380 - T]),
                            weights=np.zeros((1, 2, 384)))


@pytest.mark.parametrize("dtype,T", [("f16", 70), ("f32", 70), ("bf16", 3), ("f32", 1), ("f16", 300)])
def test_workspace_of_a_type(dtype, T):
    """A call stays within the workspace of its own type."""
    rng = np.random.default_rng(T)
    t = torch()
    d = OnDevice(make(rng, 2, 8, 2, 64, 64, 16, "int8"))
    for weights in (False, True):
        need = d.h.attention_workspace(2, T, 14, weights=weights, dtype=dtype)
        ws = t.full((need + 4096,), 0x5a, dtype=t.uint8, device="cuda")
        ws[:4] = 0
        check_attention(d, rng.standard_normal((2, T, 14, 64)), dtype, np.array([100, 0]), ws=ws[:need],
                        weights=rng.random((2, 2, 512)) if weights else None)
        assert (ws[need:] == 0x5a).all() and (ws[:4] == 0).all()


@pytest.mark.parametrize("dim,heads,T,lens", [(64, 4, 70, [0, 300]), (128, 14, 300, [40, 0])])
def test_short_prompts_in_a_wide_table(dim, heads, T, lens):
    """A table of 8192 positions: rows that see fewer than eight tiles of 128 are answered without parts."""
    rng = np.random.default_rng(T)
    t = torch()
    d = OnDevice(make(rng, 2, 128, 2, dim, 64, 16, "int8"))
    need = d.h.attention_workspace(2, T, heads, dtype="f16")
    ws = t.full((need,), 0x5a, dtype=t.uint8, device="cuda")
    ws[:4] = 0
    check_attention(d, rng.standard_normal((2, T, heads, dim)), "f16", np.array(lens), ws=ws)
    assert (ws[4:] == 0x5a).all()
    # one sequence sees enough for two shares, the other does not
    lens = np.array([1300, lens[1]])
    check_attention(d, rng.standard_normal((2, T, heads, dim)), "f16", lens, weights=rng.random((2, 2, 8192)))


def one_hot_cache(rng, pages, dim=64):
    """One sequence, one KV head; every 16th key scores 0 and has no V, the others are -100 in channel 0; scales 1."""
    d = OnDevice(make(rng, 1, pages, 1, dim, 64, 16, "int8", spare=0))
    d.ref.ks[:], d.ref.vs[:] = 1, 1
    d.ref.k[..., 0] = np.int8(-100).view(np.uint8)
    d.ref.v[:] = rng.integers(1, 128, d.ref.v.shape)
    d.ref.k[:, :, 5::16, 0], d.ref.v[:, :, 5::16] = 0, 0
    for n in ("k", "v", "ks", "vs"):
        d.t[n].copy_(dev(getattr(d.ref, n)))
    return d


@pytest.mark.parametrize("dtype,T,depth", [("f32", T, x) for T in (1, 5, 70) for x in (12.5, 13.9, 17.9)] +
                         [("f16", T, x) for T in (1, 12, 70) for x in (17.9, 18.7)] +
                         [("bf16", T, x) for T in (1, 12, 70) for x in (18.4, 18.7)])
def test_long_tail_under_peaks(dtype, T, depth):
    """All that is answered comes from weights 2^-depth of the largest, all alike, so that their roundings do not cancel:
    they are held to 2^-11 of each (fp32 rows 2^-22) down to 2^-21 (2^-16) of the largest.

    Queries are one-hot, so scores are exact up to three fp32 roundings of up to `depth`, 3 depth 2^-24, and exp2's
    2^-22, twice for numerator and denominator; sums of n / 16 products truncate by 2^-23 each at most; below the depths
    named, P's smallest step leaves 2^-32 (2^-38) of the largest weight x V."""
    rng = np.random.default_rng(int(10 * depth))
    n, heads = 2048, 4
    d = one_hot_cache(rng, n // 64)
    q = np.zeros((1, T, heads, 64))
    q[..., 0] = 1
    scale = float(np.float32(depth * np.log(2) / 100))
    out, _ = run_attention(d, q, dtype, np.array([n - T]), scale=scale)
    want, _, mag, _ = d.ref.attention(q, [n - T], [T], scale)
    u, low = (2.0 ** -22, 2.0 ** -38) if dtype == "f32" else (2.0 ** -11, 2.0 ** -32)
    dx = 2 * (3 * depth * 2.0 ** -24 + 2.0 ** -22) + n / 16 * 2.0 ** -23
    peak = 1 / ((n - T) // 16)  # the largest weight, at most
    near(out, want, HALF[dtype] * np.abs(want) + (u + dx) * mag + n * low * peak * 127)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("T", [1, 12, 40])
@pytest.mark.parametrize("far", ["behind", "below"])
def test_one_block_of_large_scale(dtype, T, far):
    """V scales of 2^-99 and one block of 2^100 that a row does not see, or whose scores lie 2^260 below: the row
    answers by the others alone.

    The one-hot queries' scores are 0 or about -260 and exact; weights count as in test_long_tail_under_peaks."""
    rng = np.random.default_rng(T)
    d = OnDevice(make(rng, 1, 2, 1, 64, 64, 16, "int8", spare=0))
    d.ref.ks[:], d.ref.vs[:] = 1, 2.0 ** -99
    pg, off = d.ref.where(0, 48)
    d.ref.vs[pg, 0, off // 16] = 2.0 ** 100
    d.ref.k[..., 0] = 0
    if far == "below":
        d.ref.k[pg, 0, off:off + 16, 0] = np.int8(-100).view(np.uint8)
    for n in ("k", "ks", "vs"):
        d.t[n].copy_(dev(getattr(d.ref, n)))
    q = np.zeros((1, T, 3, 64))
    q[..., 0] = 1
    scale = float(np.float32(2.6 * np.log(2)))
    L = 48 - T if far == "behind" else 90  # behind: the block's first rows are new, the last query sees position 47
    lens, new = np.array([L]), np.array([T])
    if far == "behind":  # rows that do see it follow in the same tile
        q = np.concatenate([q, q[:, :1]], 1)
        new = new + 1
    out, _ = run_attention(d, q, dtype, lens, new, scale=scale)
    want, p, mag, _ = d.ref.attention(q, lens, new, scale)
    u, low = (2.0 ** -22, 2.0 ** -38) if dtype == "f32" else (2.0 ** -11, 2.0 ** -32)
    top = 127 * 2.0 ** -99
    tol = HALF[dtype] * np.abs(want) + (u + 2.0 ** -19) * mag + 128 * low * top
    if dtype == "f16":  # smaller than fp16's numbers
        tol += 2.0 ** -25
    near(out[:, :T], want[:, :T], tol[:, :T])
    assert not np.isnan(out).any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 12, 70])
@pytest.mark.parametrize("depth", [110, 122, 200])
def test_all_v_far_below_a_block_of_zeros(dtype, T, depth):
    """The largest scores meet a V scale of 0, the rest weigh 2^-depth: the answer is that small, down to fp32's
    smallest normal weight, 2^-126, below which it is 0; scores as in test_long_tail_under_peaks."""
    rng = np.random.default_rng(T)
    d = one_hot_cache(rng, 8)
    d.ref.k[..., 0] = np.int8(-100).view(np.uint8)
    for p0 in range(0, 512, 128):
        pg, off = d.ref.where(0, p0)
        d.ref.k[pg, 0, off:off + 16, 0] = 0
        d.ref.vs[pg, 0, off // 16] = 0
    for n in ("k", "vs"):
        d.t[n].copy_(dev(getattr(d.ref, n)))
    q = np.zeros((1, T, 4, 64))
    q[..., 0] = 1
    scale = float(np.float32(depth * np.log(2) / 100))
    out, _ = run_attention(d, q, dtype, np.array([512 - T]), scale=scale)
    want, _, mag, _ = d.ref.attention(q, [512 - T], [T], scale)
    u = 2.0 ** -22 if dtype == "f32" else 2.0 ** -11
    dx = 2 * (3 * depth * 2.0 ** -24 + 2.0 ** -22) + 32 * 2.0 ** -23
    near(out, want, HALF[dtype] * np.abs(want) + (u + dx) * mag + (0 if depth < 126 else 2.0 ** -126 * 127 * 512))


def test_two_graphs_on_two_streams():
    """A single token and a prompt with weights, captured with a workspace each and replayed side by side; an
    eviction captured too.  Every replay gives the eager call's bits."""
    t = torch()
    rng = np.random.default_rng(41)
    sides = []
    for T, H, lens in ((1, 14, [700, 3, 90]), (60, 6, [500, 0, 130])):
        d = OnDevice(make(rng, 3, 12, 2, 64, 64, 16, "int8"))
        q = dev(rng.standard_normal((3, T, H, 64)).astype(np.float16))
        s = {"d": d, "q": q, "T": T, "H": H, "lens": ints(lens), "w": dev(rng.random((3, 2, 768)).astype(np.float32)),
             "ws": t.zeros(d.h.attention_workspace(3, T, H, weights=True), dtype=t.uint8, device="cuda"),
             "st": t.cuda.Stream()}
        s["out"], s["wo"] = t.zeros_like(q), t.zeros_like(s["w"])
        n = d.h.evict_workspace(3, 64)
        s.update(ews=t.zeros(n, dtype=t.uint8, device="cuda"), eb=n, pos=t.arange(768, dtype=t.int32, device="cuda").expand(3, 2, -1).contiguous(),
                 ew=t.zeros_like(s["w"]), ep=t.zeros(3, 2, 768, dtype=t.int32, device="cuda"), el=ints([0, 0, 0]))
        sides.append(s)

    def call(s, stream):
        s["d"].h.attention(s["q"].data_ptr(), s["out"].data_ptr(), "f16", 3, s["T"], s["H"], s["lens"].data_ptr(),
                           w_in=s["w"].data_ptr(), w_out=s["wo"].data_ptr(), ld_w=768, ws=s["ws"].data_ptr(),
                           ws_bytes=s["ws"].numel(), stream=stream)
        s["d"].h.evict(3, 64, s["lens"].data_ptr(), s["el"].data_ptr(), s["wo"].data_ptr(), s["ew"].data_ptr(),
                       s["pos"].data_ptr(), s["ep"].data_ptr(), 768, seen=s["lens"].data_ptr(), recent=8,
                       ws=s["ews"].data_ptr(), ws_bytes=s["eb"], stream=stream)

    t.cuda.synchronize()
    names = ("out", "wo", "ew", "ep", "el")
    for s in sides:
        pools = {n: s["d"].t[n].clone() for n in ("k", "v", "ks", "vs")}
        call(s, 0)
        t.cuda.synchronize()
        s["want"] = [s[n].clone() for n in names] + [s["d"].t[n].clone() for n in pools]
        for n, x in pools.items():
            s["d"].t[n].copy_(x)
        for n in names:
            s[n].zero_()
        s["pools"] = pools
    t.cuda.synchronize()
    for s in sides:
        s["graph"] = t.cuda.CUDAGraph()
        with t.cuda.graph(s["graph"], stream=s["st"]):
            call(s, t.cuda.current_stream().cuda_stream)
    for _ in range(5):
        for s in sides:
            for n, x in s["pools"].items():
                s["d"].t[n].copy_(x)
        t.cuda.synchronize()
        for s in sides:
            with t.cuda.stream(s["st"]):
                s["graph"].replay()
        t.cuda.synchronize()
        for s in sides:
            got = [s[n] for n in names] + [s["d"].t[n] for n in s["pools"]]
            assert all(t.equal(g, w) for g, w in zip(got, s["want"]))
            assert int(s["ws"][:4].view(t.int32)[0]) == 0  # no wait ran out


def test_query_ranges():
    """Queries of zeros, huge and tiny ones, other scales; an infinity or NaN stays in its own row."""
    rng = np.random.default_rng(9)
    for T in (1, 70):
        d = OnDevice(make(rng, 1, 3, 1, 64, 64, 16, "int8"))
        q = rng.standard_normal((1, T, 6, 64))
        q[0, 0, 1], q[0, 0, 2], q[0, 0, 3] = 0, q[0, 0, 2] * 1e-6, q[0, 0, 3] * 40
        for dtype in ("f16", "bf16", "f32"):
            check_attention(d, q, dtype, np.array([150 - T]), scale=0.2)
            check_attention(d, q, dtype, np.array([150 - T]), scale=-0.05)
            bad = q.copy()
            bad[0, 0, 4, 3], bad[0, 0, 5, 9] = np.nan, np.inf
            out, _ = run_attention(d, bad, dtype, np.array([150 - T]), scale=0.2)
            good, _ = run_attention(d, q, dtype, np.array([150 - T]), scale=0.2)
            assert np.isnan(out[0, 0, 4]).all()
            assert np.array_equal(out[0, :, :4], good[0, :, :4])


def test_strides_workspace_and_in_place_weights():
    """Rows inside wider rows; one workspace for calls of other shapes, one after the other."""
    rng = np.random.default_rng(12)
    t = torch()
    d = OnDevice(make(rng, 3, 3, 2, 64, 64, 16, "int8"))
    need = max(d.h.attention_workspace(3, T, H, weights=True) for T, H in ((1, 14), (7, 14), (90, 6), (1, 2)))
    ws = t.zeros(need, dtype=t.uint8, device="cuda")
    for T, H, dtype, ldq, ldo in ((1, 14, "f16", 14 * 64 + 13, 14 * 64 + 1), (7, 14, "bf16", 0, 14 * 64 + 8),
                                  (90, 6, "f16", 6 * 64 + 5, 0), (1, 2, "f32", 131, 129), (1, 14, "f16", 0, 0)):
        for in_place in (False, True):
            check_attention(d, rng.standard_normal((3, T, H, 64)), dtype, np.array([99, 0, 60]),
                            weights=rng.random((3, 2, 192 + 5 * in_place)), ws=ws, ldq=ldq, ldo=ldo, in_place=in_place)


def test_positions_past_32_bits():
    """A pool of more than 2^32 bytes: pages at its far end."""
    t = torch()
    rng = np.random.default_rng(13)
    n_pages, kv, dim, page = 70000, 8, 128, 64  # 4.6 GB a pool
    k, v = (t.zeros(n_pages, kv, page, dim, dtype=t.uint8, device="cuda") for _ in range(2))
    ks, vs = (t.zeros(n_pages, kv, page // 16, device="cuda") for _ in range(2))
    small = make(rng, 1, 2, kv, dim, page, 16, "int8", spare=0)
    far = np.array([[n_pages - 1, n_pages - 3]], np.int32)
    table = dev(far)
    h = kv8.KV8Cache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), table.data_ptr(), n_pages=n_pages,
                     max_pages=2, n_kv=kv, head_dim=dim, page_size=page, block=16, code="int8")
    small.table[:] = [[0, 1]]
    x = [rows(rng, 1, 100, kv, dim).astype(np.float16) for _ in range(2)]
    dx, zero = [dev(a) for a in x], ints([0])
    h.append(dx[0].data_ptr(), dx[1].data_ptr(), "f16", 1, 100, zero.data_ptr())
    small.append(x[0], x[1], [0], [100])
    t.cuda.synchronize()
    for i in range(2):
        for got, want in ((k, small.k), (v, small.v)):
            n = 64 if i == 0 else 36
            assert np.array_equal(got[int(far[0, i])].cpu().numpy()[:, :n], want[i][:, :n])
    d = OnDevice(small)
    d.h = h
    check_attention(d, rng.standard_normal((1, 1, 16, dim)), "f16", np.array([99]))
    check_attention(d, rng.standard_normal((1, 20, 16, dim)), "f16", np.array([80]))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,page,block,keep,first,recent", [(64, 16, 16, 16, 0, 0), (64, 64, 16, 64, 4, 20),
                                                              (128, 32, 32, 96, 0, 96), (128, 128, 64, 64, 1, 0),
                                                              (64, 64, 64, 128, 128, 0)])
def test_evict_exact(code, dim, page, block, keep, first, recent):
    """Lengths around the budget, ties, NaN and infinite weights; a second eviction of the result."""
    rng = np.random.default_rng(keep + dim)
    t = torch()
    lens = np.array([0, keep - 1, keep, keep + 1, 2 * keep - 5, 256])
    cap = -(-256 // page) * page
    d = OnDevice(make(rng, len(lens), cap // page, 3, dim, page, block, code))
    w = rng.choice([0.0, 0.5, 1.25, 3.0], (len(lens), 3, cap + 3)).astype(np.float32) + \
        (rng.random((len(lens), 3, cap + 3)) < 0.5) * rng.random((len(lens), 3, cap + 3)).astype(np.float32)
    w[4, 0, 3], w[4, 1, 7], w[5, 2, ::9], w[5, 1, 4] = np.inf, -np.inf, np.nan, -0.0
    w = w.astype(np.float32)
    pos = np.broadcast_to(np.arange(cap + 3, dtype=np.int32), w.shape).copy()
    seen = lens.copy()
    need = d.h.evict_workspace(len(lens), keep)
    ws = t.full((need,), 0x5a, dtype=t.uint8, device="cuda")
    for turn in range(2):
        in_place = turn == 1
        dw, dp, dl, ds = dev(w), dev(pos), ints(lens), ints(seen)
        wo, po, lo = (dw, dp, dl) if in_place else (t.full_like(dw, 8), t.full_like(dp, 8), t.full_like(dl, 8))
        d.h.evict(len(lens), keep, dl.data_ptr(), lo.data_ptr(), dw.data_ptr(), wo.data_ptr(), dp.data_ptr(),
                  po.data_ptr(), cap + 3, seen=ds.data_ptr(), first=first, recent=recent, ws=ws.data_ptr(), ws_bytes=need)
        t.cuda.synchronize()
        lens, w, pos = d.ref.evict(keep, first, recent, seen, lens, w, pos)
        d.same_as_reference()
        assert np.array_equal(lo.cpu().numpy(), lens)
        assert np.array_equal(wo.cpu().numpy(), w, equal_nan=True)
        assert np.array_equal(po.cpu().numpy(), pos)
        # grow again: 30 tokens behind what is left
        T = 30
        n = np.minimum(T, np.maximum(d.ref.cap - lens, 0))
        append(d, rows(rng, len(lens), T, 3, dim), rows(rng, len(lens), T, 3, dim), "f16", lens, n)
        lens, seen = lens + n, seen + n
        w = w + rng.random(w.shape).astype(np.float32)


@pytest.mark.parametrize("max_pages,keep", [(700, 20032), (900, 4096), (900, 56000)])
def test_evict_long(max_pages, keep):
    """Contexts and budgets beyond what the selection holds on chip."""
    rng = np.random.default_rng(keep)
    t = torch()
    d = OnDevice(make(rng, 1, max_pages, 1, 64, 64, 64, "int8", spare=0))
    cap = d.ref.cap
    w = np.round(rng.random((1, 1, cap)) * 5000).astype(np.float32)
    pos = np.broadcast_to(np.arange(cap, dtype=np.int32), w.shape).copy()
    lens = np.array([cap - 7])
    dw, dp, dl = dev(w), dev(pos), ints(lens)
    ws = t.empty(d.h.evict_workspace(1, keep), dtype=t.uint8, device="cuda")
    d.h.evict(1, keep, dl.data_ptr(), dl.data_ptr(), dw.data_ptr(), dw.data_ptr(), dp.data_ptr(), dp.data_ptr(), cap,
              seen=ints(lens).data_ptr(), first=4, recent=100, ws=ws.data_ptr(), ws_bytes=ws.numel())
    t.cuda.synchronize()
    lens, w, pos = d.ref.evict(keep, 4, 100, lens, lens, w, pos)
    d.same_as_reference()
    assert np.array_equal(dl.cpu().numpy(), lens)
    assert np.array_equal(dw.cpu().numpy(), w) and np.array_equal(dp.cpu().numpy(), pos)


def test_evict_missing_pages():
    rng = np.random.default_rng(21)
    t = torch()
    d = OnDevice(make(rng, 2, 4, 2, 64, 32, 16, "int8"))
    d.ref.table[0, 3], d.ref.table[1, 0] = -5, d.ref.n_pages
    d.t["table"].copy_(dev(d.ref.table))
    w = rng.random((2, 2, 128)).astype(np.float32)
    pos = np.broadcast_to(np.arange(128, dtype=np.int32), w.shape).copy()
    lens = np.array([128, 120])
    dw, dp, dl = dev(w), dev(pos), ints(lens)
    ws = t.empty(d.h.evict_workspace(2, 64), dtype=t.uint8, device="cuda")
    d.h.evict(2, 64, dl.data_ptr(), dl.data_ptr(), dw.data_ptr(), dw.data_ptr(), dp.data_ptr(), dp.data_ptr(), 128,
              seen=ints(lens).data_ptr(), ws=ws.data_ptr(), ws_bytes=ws.numel())
    t.cuda.synchronize()
    lens, w, pos = d.ref.evict(64, 0, 0, lens, lens, w, pos)
    d.same_as_reference()
    assert np.array_equal(dw.cpu().numpy(), w) and np.array_equal(dp.cpu().numpy(), pos)


def test_serving_run():
    """The operators as a decoder uses them: a prompt, single tokens with accumulated weights, an
    eviction when a sequence outgrows its budget, more tokens; on a side stream, and the step once
    captured and replayed."""
    t = torch()
    rng = np.random.default_rng(31)
    B, kv, H, D, keep = 3, 2, 14, 64, 64
    d = OnDevice(make(rng, B, 3, kv, D, 64, 16, "int8"))
    cap = d.ref.cap
    lens, seen = np.zeros(B, int), np.zeros(B, int)
    w, pos = np.zeros((B, kv, cap)), np.broadcast_to(np.arange(cap, dtype=np.int32), (B, kv, cap)).copy()
    new = np.array([60, 33, 1])
    append(d, rows(rng, B, 60, kv, D), rows(rng, B, 60, kv, D), "f16", lens, new)
    _, w1 = check_attention(d, rng.standard_normal((B, 60, H, D)), "f16", lens, new, weights=w)
    w = np.where(w1 < 0, 0, w1)
    lens, seen = lens + new, seen + new

    st = t.cuda.Stream()
    dl, dw = ints(lens), dev(w.astype(np.float32))
    k, v = (t.zeros(B, 1, kv, D, dtype=t.float16, device="cuda") for _ in range(2))
    q, out = (t.zeros(B, 1, H, D, dtype=t.float16, device="cuda") for _ in range(2))
    ws = t.zeros(d.h.attention_workspace(B, 1, H, weights=True), dtype=t.uint8, device="cuda")

    def step(stream):
        d.h.append(k.data_ptr(), v.data_ptr(), "f16", B, 1, dl.data_ptr(), stream=stream)
        d.h.attention(q.data_ptr(), out.data_ptr(), "f16", B, 1, H, dl.data_ptr(), w_in=dw.data_ptr(), w_out=dw.data_ptr(),
                      ld_w=cap, ws=ws.data_ptr(), ws_bytes=ws.numel(), stream=stream)

    graph = None
    for i in range(12):
        xs = [rows(rng, B, 1, kv, D).astype(np.float16) for _ in range(2)]
        xq = rng.standard_normal((B, 1, H, D)).astype(np.float16)
        t.cuda.synchronize()
        for a, x in ((k, xs[0]), (v, xs[1]), (q, xq), (dl, lens.astype(np.int32))):
            a.copy_(dev(x))
        t.cuda.synchronize()
        if i == 6:
            graph = t.cuda.CUDAGraph()
            with t.cuda.graph(graph, stream=st):
                step(t.cuda.current_stream().cuda_stream)
        if graph is None:
            step(st.cuda_stream)
        else:
            graph.replay()
        t.cuda.synchronize()
        d.ref.append(xs[0], xs[1], lens, [1] * B)
        d.same_as_reference()
        want, p, mag, big = d.ref.attention(xq, lens, [1] * B, D ** -0.5)
        near(out.float().cpu().numpy(), want, tolerance(d.ref, "f16", want, mag, big)[1])
        for b in range(B):
            w[b, :, lens[b]:] = 0
        w = w + p
        assert np.allclose(dw.cpu().numpy(), w, rtol=1e-4, atol=1e-6)
        w = dw.cpu().numpy().astype(np.float64)
        lens, seen = lens + 1, seen + 1
        if lens.max() > keep + 4:
            dp, ds = dev(pos), ints(seen)
            es = t.empty(d.h.evict_workspace(B, keep), dtype=t.uint8, device="cuda")
            dl.copy_(ints(lens))
            t.cuda.synchronize()
            d.h.evict(B, keep, dl.data_ptr(), dl.data_ptr(), dw.data_ptr(), dw.data_ptr(), dp.data_ptr(), dp.data_ptr(),
                      cap, seen=ds.data_ptr(), first=2, recent=16, ws=es.data_ptr(), ws_bytes=es.numel(),
                      stream=st.cuda_stream)
            t.cuda.synchronize()
            lens, w32, pos = d.ref.evict(keep, 2, 16, seen, lens, w.astype(np.float32), pos)
            w = w32.astype(np.float64)
            d.same_as_reference()
            assert np.array_equal(dl.cpu().numpy(), lens) and np.array_equal(dp.cpu().numpy(), pos)
            assert np.array_equal(dw.cpu().numpy(), w32)
    assert seen.max() > lens.max(), "no eviction happened"
