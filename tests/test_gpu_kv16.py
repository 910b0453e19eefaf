"""Rotary positions, the 16-bit cache behind a shared prefix and its attention on the GPU against the plain numpy
statement of them (``kv16_ref.py``).

Rotated values are held to half a step of their type and the fp32 bound that ``turned`` gives; values that are
only moved are exact.  Attention is held to  h |y| + u S + e S + n t V:  S = sum p |v|, V = max |v|, h the half
step of the output's type, u that of the softmax weights (the cache's type), t half of fp16's smallest step against
a largest weight of at least 1, and e = 2 dx with dx the error of a score: products are exact in fp32 and the running
sum of head_dim of them truncates, (head_dim + 8) 2^-23 of scale * sum |q k|, twice because numerator and denominator
both carry it; exp2 adds 2^-20.
"""
import numpy as np
import pytest

from gpu_util import dev, torch
from kv16_ref import HALF, TINY, TYPES, Cache, rounded, turned
from n730_b200 import kv16

pytestmark = pytest.mark.gpu


def ints(x):
    return dev(np.asarray(x, np.int32))


def put(x, dtype, ld=0, shift=0, fill=7.0):
    """Rows x [rows, n] in a buffer with ld elements a row, `shift` elements in: (buffer, view of the rows)."""
    n, t = x.shape[1], torch()
    ld = ld or n
    buf = t.full((shift + len(x) * ld,), fill, dtype=TYPES[dtype], device="cuda")
    rows = buf[shift:].view(len(x), ld)[:, :n]
    rows.copy_(dev(np.ascontiguousarray(x, np.float32)).to(TYPES[dtype]))
    return buf[shift:], rows


class Turn:
    """A rotary with its frequencies on the device."""

    def __init__(self, dim, layout="half", scaling="none", theta=1e4, **kw):
        self.freq, self.factor = kv16.frequencies(dim, theta, scaling, **kw)
        self.t, self.layout = dev(self.freq), layout
        self.h = kv16.Rotary(self.t.data_ptr(), dim, layout=layout, factor=self.factor)

    def bound(self, x, pos, dtype):
        y, e = turned(x, np.asarray(pos), self.freq, self.factor, self.layout)
        moved = np.zeros(x.shape, bool)
        moved[..., 2 * len(self.freq):] = True
        return y, np.where(moved, 0, HALF[dtype] * (np.abs(y) + e) + TINY[dtype] + e)


def near(got, want, bound, what=""):
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got - want) <= bound) & ~(np.isnan(got) & np.isnan(want)) & ~(got == want)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.max(np.where(bad, np.abs(got - want) / np.maximum(bound, 1e-30), 0)):.3g} bounds, at {np.argwhere(bad)[0]}"


# ----------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows,heads,dim,part", [(1, 1, 64, 64), (3, 28, 128, 128), (300, 5, 64, 32), (17, 14, 64, 48), (9, 3, 128, 20),
                                                 (2, 1, 6, 2), (5, 200, 64, 64), (33, 2, 512, 512), (700, 1, 16, 16), (4, 70, 96, 96)])
def test_rotary(dtype, layout, rows, heads, dim, part):
    """Whole heads and parts of them, units that are vectors and ones that are not, rows in one CTA and over many."""
    rng = np.random.default_rng(rows * heads + part)
    turn = Turn(part, layout, "ramp" if dim == 128 else "none", factor=4, trained=2048)
    x, pos = rng.standard_normal((rows, heads * dim)), rng.integers(0, 1 << 20, rows)
    bx, vx = put(x, dtype)
    by, vy = put(np.zeros_like(x), dtype)
    dp = ints(pos)
    torch().cuda.synchronize()
    turn.h.apply(bx.data_ptr(), by.data_ptr(), dtype, rows, heads, dim, dp.data_ptr())
    held = rounded(x, dtype).reshape(rows, heads, dim)
    near(vy.float().cpu().numpy().reshape(held.shape), *turn.bound(held, pos, dtype))
    turn.h.apply(bx.data_ptr(), bx.data_ptr(), dtype, rows, heads, dim, dp.data_ptr())
    assert torch().equal(vx, vy)


def test_rotary_far():
    """The largest and negative positions; angles stay right where fp32 has lost them."""
    rng = np.random.default_rng(1)
    turn = Turn(64)
    pos = np.array([0, 1, 2 ** 31 - 1, 2 ** 31 - 2, -1, -2 ** 31, 10 ** 9, 123456789])
    x = rng.standard_normal((len(pos), 2 * 64))
    bx, vx = put(x, "f32")
    dp = ints(pos)
    turn.h.apply(bx.data_ptr(), bx.data_ptr(), "f32", len(pos), 2, 64, dp.data_ptr())
    got = vx.float().cpu().numpy().reshape(-1, 2, 64)
    held = rounded(x, "f32").reshape(got.shape)
    near(got, *turn.bound(held, pos, "f32"))
    assert np.array_equal(got[0], held[0])


@pytest.mark.parametrize("ldx,ldy,shift,dtype", [(300, 260, 0, "f32"), (257, 300, 1, "f16"), (264, 272, 8, "bf16"), (256, 260, 3, "f32")])
def test_rotary_strides(ldx, ldy, shift, dtype):
    """Rows on any element and apart; what lies between output rows stays."""
    rng = np.random.default_rng(ldx)
    turn = Turn(128)
    x, pos = rng.standard_normal((7, 256)), rng.integers(0, 5000, 7)
    bx, _ = put(x, dtype, ldx, shift)
    by, vy = put(np.zeros_like(x), dtype, ldy, shift, fill=3.0)
    turn.h.apply(bx.data_ptr(), by.data_ptr(), dtype, 7, 2, 128, ints(pos).data_ptr(), ldx=ldx, ldy=ldy)
    held = rounded(x, dtype).reshape(7, 2, 128)
    near(vy.float().cpu().numpy().reshape(held.shape), *turn.bound(held, pos, dtype))
    assert bool((by.view(7, ldy)[:, 256:] == 3).all())


def test_rotary_values():
    """NaN and infinities stay in their pair."""
    turn = Turn(64)
    x = np.ones((2, 64))
    x[0, 3], x[1, 40] = np.nan, np.inf
    bx, vx = put(x, "bf16")
    turn.h.apply(bx.data_ptr(), bx.data_ptr(), "bf16", 2, 1, 64, ints([5, 6]).data_ptr())
    y = vx.float().cpu().numpy()
    assert np.array_equal(np.argwhere(~np.isfinite(y)), [[0, 3], [0, 35], [1, 8], [1, 40]])


# ----------------------------------------------------------------------------- cache
class OnDevice:
    def __init__(self, ref):
        self.ref = ref
        self.t = {n: dev(getattr(ref, n)) for n in ("prefix_table", "table")}
        self.t |= {n: dev(getattr(ref, n)).to(TYPES[ref.dtype]) for n in ("k", "v")}
        self.t["prefix_len"] = ints([ref.prefix_len])
        p = {n: x.data_ptr() for n, x in self.t.items()}
        self.h = kv16.KV16Cache(p["k"], p["v"], p["table"], n_pages=ref.n_pages, max_pages=ref.max_pages, n_kv=ref.kv,
                                head_dim=ref.dim, page_size=ref.page, dtype=ref.dtype, prefix_table=p["prefix_table"],
                                prefix_pages=ref.prefix_pages, prefix_len=p["prefix_len"])
        self.ws = {}

    def tables(self):
        for n in ("prefix_table", "table"):
            self.t[n].copy_(dev(getattr(self.ref, n)))

    def near_reference(self, k_bound=0.0):
        near(self.t["k"].float().cpu().numpy(), self.ref.k, k_bound, "k")
        assert np.array_equal(self.t["v"].float().cpu().numpy(), self.ref.v, equal_nan=True)


def append(d, k, v, dtype, lens, new, turn=None, q=None, pos=None, ld=0, shift=0):
    """Both sides append; the bound of the cached keys is returned with the queries and theirs."""
    B, T = k.shape[:2]
    ref = d.ref
    bk, bv = (put(x.reshape(B * T, -1), dtype, ld, shift)[0] for x in (k, v))
    dl, dn = ints(lens), ints(new) if new is not None else None
    kw = {}
    at = np.array([[ref.prefix + ref.len(lens, b) + t for t in range(T)] for b in range(B)]) if pos is None else np.asarray(pos)
    if turn:
        kw["rotary"] = turn.h
    if pos is not None:
        dp = ints(pos)
        kw["pos"] = dp.data_ptr()
    if q is not None:
        H = q.shape[2]
        bq, vq = put(q.reshape(B * T, -1), dtype, ld and ld + (H - ref.kv) * ref.dim, shift)
        bo, vo = put(np.full((B * T, H * ref.dim), 9.0), dtype, ld and ld + 8 + (H - ref.kv) * ref.dim, shift)
        kw |= dict(q=bq.data_ptr(), q_out=bo.data_ptr(), heads=H, ldq=bq.numel() // (B * T), ldqo=bo.numel() // (B * T))
    torch().cuda.synchronize()
    d.h.append(bk.data_ptr(), bv.data_ptr(), dtype, B, T, dl.data_ptr(), new=dn.data_ptr() if dn is not None else 0, ld=ld, **kw)
    torch().cuda.synchronize()
    n = np.clip(new, 0, T) if new is not None else np.full(B, T)
    hk, hv = rounded(k, dtype), rounded(v, dtype)
    if turn:
        y, e = turned(hk, at, turn.freq, turn.factor, turn.layout)
        e[..., 2 * len(turn.freq):] = 0
        off = Cache.__new__(Cache)
        off.__dict__ = dict(ref.__dict__, k=np.zeros_like(ref.k), v=np.zeros_like(ref.v), dtype="f32")
        off.append(np.where(e > 0, HALF[ref.dtype] * (np.abs(y) + e) + TINY[ref.dtype] + e, 0), hv, lens, n)
        k_bound, hk = off.k, y
        wide = ref.dtype
        # keys are compared with unrounded ones, within the bound
        keep = ref.k
        ref.k = keep.astype(np.float64)
        for b in range(B):
            for t in range(n[b]):
                p = ref.len(lens, b) + t
                slot = ref.slot(ref.table[b], p) if p < ref.cap else None
                if slot:
                    moved = rounded(hk[b, t], wide)
                    ref.k[slot[0], :, slot[1]] = np.where(e[b, t] > 0, hk[b, t], moved)
                    ref.v[slot[0], :, slot[1]] = rounded(hv[b, t], wide)
        d.near_reference(k_bound)
        ref.k = d.t["k"].float().cpu().numpy()  # the roundings that were made
    else:
        ref.append(hk, hv, lens, n)
        d.near_reference()
    if q is not None:
        hq = rounded(q, dtype)
        y, e = turn.bound(hq, at, dtype)
        got = vo.float().cpu().numpy().reshape(q.shape)
        for b in range(B):
            near(got[b, :n[b]], y[b, :n[b]], e[b, :n[b]], "q")
            assert np.all(got[b, n[b]:] == 9.0)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("kept,dim,page,part,layout", [("f16", 64, 16, 64, "half"), ("bf16", 128, 64, 96, "half"), ("f16", 128, 96, 64, "interleaved"),
                                                       ("bf16", 64, 32, 20, "half"), ("f16", 64, 128, 50, "interleaved")])
def test_append(dtype, kept, dim, page, part, layout):
    """A prompt, single tokens and ragged counts behind a prefix that ends inside a page, with and without rotation."""
    rng = np.random.default_rng(dim + page)
    d = OnDevice(Cache(3, 4, 3, 2 * page + 5, 2, dim, page, kept, rng))
    turn = Turn(part, layout, "bands", factor=8, trained=64, low=1, high=4)
    lens = np.array([0, 5, page - 1])
    for new, T, r in ((np.array([37, 0, 2]), 37, True), (np.array([1, 1, 1]), 1, True), (None, 1, False), (np.array([2, 9, -4]), 3, True)):
        k, v = rng.standard_normal((2, 3, T, 2, dim))
        q = rng.standard_normal((3, T, 6, dim)) if r else None
        append(d, k, v, dtype, lens, new, turn if r else None, q)
        lens = lens + (np.clip(new, 0, T) if new is not None else T)


def test_append_edges():
    """A full table, bad lengths and pages, given positions, rows apart and on any element, a prefix out of range."""
    rng = np.random.default_rng(3)
    ref = Cache(4, 2, 2, 1 << 30, 2, 64, 32, "f16", rng)
    ref.table[1, 0], ref.table[2, 1] = -1, ref.n_pages
    d = OnDevice(ref)
    turn = Turn(64)
    k, v = rng.standard_normal((2, 4, 40, 2, 64))
    k[0, 3, 1, 5], v[3, 20, 0, 9] = np.nan, np.inf
    append(d, k, v, "f32", np.array([0, 0, 20, 50]), None)
    k = rng.standard_normal(k.shape)
    append(d, k, v, "f32", np.array([-7, 64, 63, 1 << 30]), np.array([1, 40, 99, 3]), turn, ld=200, shift=1)
    q = rng.standard_normal((4, 40, 4, 64))
    append(d, k, v, "bf16", np.array([3, 0, 9, 11]), np.array([4, 5, 6, 40]), turn, q, pos=rng.integers(0, 1 << 20, (4, 40)), ld=144, shift=8)
    d.t["prefix_len"].fill_(-5)
    ref.prefix_len = -5
    append(d, k, v, "f16", np.array([3, 0, 9, 11]), np.array([4, 5, 6, 40]), turn, q)


# ----------------------------------------------------------------------------- attention
def attend(d, q, lens, new, scale=None, ldq=0, ldo=0, shift=0, stream=0, ws=None):
    """(out, rows between and behind left alone) of the call."""
    B, T, H, D = q.shape
    bq, _ = put(q.reshape(B * T, -1), d.ref.dtype, ldq, shift)
    bo, vo = put(np.full((B * T, H * D), 9.0), d.ref.dtype, ldo, shift, fill=9.0)
    dl, dn = ints(lens), ints(new) if new is not None else None
    need = d.h.attention_workspace(B, T, H)
    ws = torch().zeros(need, dtype=torch().uint8, device="cuda") if ws is None else ws
    torch().cuda.synchronize()
    d.h.attention(bq.data_ptr(), bo.data_ptr(), B, T, H, dl.data_ptr(), new=dn.data_ptr() if dn is not None else 0,
                  scale=scale, ldq=ldq, ldo=ldo, ws=ws.data_ptr(), ws_bytes=need, stream=stream)
    torch().cuda.synchronize()
    assert int(ws[:4].view(torch().int32)[0]) == 0
    if ldo:
        assert bool((bo.view(B * T, ldo)[:, H * D:] == 9).all())
    return vo.float().cpu().numpy().reshape(q.shape)


def check(d, q, lens, new=None, scale=None, **kw):
    B, T = q.shape[:2]
    held = rounded(q, d.ref.dtype)
    n = np.clip(new, 0, T) if new is not None else np.full(B, T)
    got = attend(d, q, lens, new, scale, **kw)
    want, bound = d.ref.attention(held, lens, n, d.ref.dim ** -0.5 if scale is None else scale)
    for b in range(B):
        near(got[b, :n[b]], want[b, :n[b]], bound[b, :n[b]], f"sequence {b}")
        assert np.all(got[b, n[b]:] == 9.0)
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("batch,T,heads,kv,dim,page,prefix,own", [
    (1, 1, 2, 2, 64, 64, 1, 1), (1, 1, 28, 4, 128, 64, 700, 40), (5, 1, 14, 2, 64, 16, 129, 200), (4, 1, 8, 8, 64, 64, 128, 64),
    (3, 5, 28, 4, 128, 32, 333, 150), (2, 3, 16, 1, 128, 128, 1000, 300), (40, 1, 14, 2, 64, 64, 257, 33), (20, 1, 32, 2, 128, 64, 500, 20),
    (2, 70, 4, 2, 64, 48, 100, 90), (1, 150, 6, 1, 128, 96, 130, 200), (33, 2, 16, 2, 64, 64, 300, 10)])
def test_attention(dtype, batch, T, heads, kv, dim, page, prefix, own):
    """Single tokens, drafts and prompts; a row tile that is not full, several of them, groups that cross tiles."""
    rng = np.random.default_rng(batch * heads + prefix)
    d = OnDevice(Cache(batch, -(-(own + T) // page), -(-prefix // page), prefix, kv, dim, page, dtype, rng))
    lens = rng.integers(0, own + 1, batch)
    check(d, 2 * rng.standard_normal((batch, T, heads, dim)), lens, rng.integers(0, T + 1, batch) if T > 1 else None)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_stale_memory(dtype):
    """NaN and infinities behind the prefix's and the sequences' last positions, and in pages of nobody."""
    rng = np.random.default_rng(21)
    for prefix in (0, 1, 63, 64, 65, 127, 128, 129, 200):
        ref = Cache(3, 3, 4, prefix, 2, 64, 64, dtype, rng, fill=np.nan)
        lens = np.array([0, 63, 140])
        for ids, n in [(ref.prefix_table, prefix)] + [(ref.table[b], lens[b] + 1) for b in range(3)]:
            for p in range(n):
                pg, off = ref.slot(ids, p)
                ref.k[pg, :, off], ref.v[pg, :, off] = rounded(rng.standard_normal((2, 2, 64)), dtype)
        ref.k[np.isnan(ref.k)] = np.where(rng.random(np.isnan(ref.k).sum()) < 0.5, np.nan, np.inf)
        check(OnDevice(ref), rng.standard_normal((3, 1, 8, 64)), lens)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_future_values(dtype):
    """A row that only later tokens of the call see may hold anything: earlier ones do not meet it."""
    rng = np.random.default_rng(22)
    for lens0 in (0, 60, 125):
        ref = Cache(2, 4, 1, 50, 1, 128, 64, dtype, rng)
        lens = np.array([lens0, 3])
        for b, t, what in ((0, 2, np.nan), (0, 4, np.inf), (1, 3, -np.inf)):
            pg, off = ref.slot(ref.table[b], lens[b] + t)
            ref.v[pg, :, off, ::3] = what
            ref.k[pg, :, off, 5] = what if t != 4 else ref.k[pg, :, off, 5]
        d = OnDevice(ref)
        q = rng.standard_normal((2, 6, 4, 128))
        got = attend(d, q, lens, None)
        clean = Cache.__new__(Cache)
        clean.__dict__ = dict(ref.__dict__, k=np.nan_to_num(ref.k, posinf=0, neginf=0), v=np.nan_to_num(ref.v, posinf=0, neginf=0))
        want, bound = clean.attention(rounded(q, dtype), lens, [6, 6], 128 ** -0.5)
        for b, t in ((0, 2), (1, 3)):
            near(got[b, :t], want[b, :t], bound[b, :t], f"before {lens0}")
            assert not np.isfinite(got[b, t:, :, ::3]).any()


def test_attention_nothing_to_see():
    """No prefix, no pages: rows without a position give zeros, the others go by what there is."""
    rng = np.random.default_rng(23)
    ref = Cache(4, 2, 3, 100, 2, 64, 64, "f16", rng)
    ref.prefix_table[:] = [-1, ref.n_pages, 1 << 30]
    ref.table[0] = -1
    ref.table[1, 0] = -5
    d = OnDevice(ref)
    q = rng.standard_normal((4, 1, 6, 64))
    got = check(d, q, np.array([5, 70, 0, 100]))
    assert np.all(got[0] == 0)
    ref.prefix_table[1] = 3
    d.tables()
    check(d, q, np.array([5, 70, 0, 100]))
    for n in (0, -3):
        d.t["prefix_len"].fill_(n)
        ref.prefix_len = n
        check(d, q, np.array([0, 1 << 30, -4, 127]))
    h = kv16.KV16Cache(*(d.t[n].data_ptr() for n in ("k", "v", "table")), n_pages=ref.n_pages, max_pages=2, n_kv=2, head_dim=64)
    d.h, ref.prefix_pages = h, 0
    check(d, q, np.array([0, 64, 9, 126]))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 5.0, 1e-4])
def test_attention_scales(dtype, scale):
    """Flat, steep and negative scales; running maxima that move far from tile to tile."""
    rng = np.random.default_rng(24)
    d = OnDevice(Cache(2, 6, 8, 500, 2, 64, 64, dtype, rng))
    ramp = np.linspace(0.01, 3, 64 * d.ref.n_pages).reshape(d.ref.n_pages, 1, 64, 1)
    d.ref.k = rounded(d.ref.k * ramp, dtype)
    d.t["k"].copy_(dev(d.ref.k))
    check(d, rng.standard_normal((2, 2, 10, 64)), np.array([300, 5]), scale=scale)


@pytest.mark.parametrize("ldq,ldo,shift", [(520, 0, 0), (0, 528, 8), (513, 515, 1)])
def test_attention_strides(ldq, ldo, shift):
    rng = np.random.default_rng(25)
    d = OnDevice(Cache(3, 2, 2, 99, 2, 64, 64, "f16", rng))
    check(d, rng.standard_normal((3, 2, 8, 64)), np.array([0, 20, 100]), np.array([2, 1, 2]), ldq=ldq, ldo=ldo, shift=shift)


@pytest.mark.parametrize("dtype,batch,heads,kv", [("f16", 6, 28, 4), ("bf16", 40, 64, 8)])
def test_attention_long_prefix(dtype, batch, heads, kv):
    """A prefix of many tiles, split over CTAs, joined with the sequences' own parts."""
    rng = np.random.default_rng(26)
    d = OnDevice(Cache(batch, 5, 64, 4085, kv, 128, 64, dtype, rng))
    lens = rng.integers(0, 310, batch)
    q = 2 * rng.standard_normal((batch, 1, heads, 128))
    got = attend(d, q, lens, None)
    some = rng.choice(batch, 3, replace=False)
    part = Cache.__new__(Cache)
    part.__dict__ = dict(d.ref.__dict__, table=d.ref.table[some])
    want, bound = part.attention(rounded(q[some], dtype), lens[some], [1] * 3, 128 ** -0.5)
    near(got[some], want, bound)


def test_attention_order():
    """The prefix's pages in another order of the pool give the same bits, as does a second call."""
    rng = np.random.default_rng(27)
    d = OnDevice(Cache(9, 3, 12, 700, 2, 64, 64, "f16", rng))
    q, lens = rng.standard_normal((9, 1, 14, 64)), rng.integers(0, 190, 9)
    a, b = attend(d, q, lens, None), attend(d, q, lens, None)
    assert np.array_equal(a, b)
    order = rng.permutation(d.ref.n_pages)
    where = np.argsort(order).astype(np.int32)
    d.ref.k, d.ref.v = d.ref.k[order], d.ref.v[order]
    d.ref.prefix_table, d.ref.table = where[d.ref.prefix_table], where[d.ref.table]
    assert np.array_equal(attend(OnDevice(d.ref), q, lens, None), a)


def test_step_in_a_graph():
    """Append with rotation and attention, captured on a stream of its own and replayed as lengths grow; two graphs
    with a workspace each, replayed at once."""
    t = torch()
    rng = np.random.default_rng(28)
    B, H, kv, D, prefix = 5, 14, 2, 64, 150
    turn = Turn(D, theta=1e6)
    made = []
    for _ in range(2):
        d = OnDevice(Cache(B, 2, 3, prefix, kv, D, 64, "bf16", rng))
        io = {n: t.zeros(B, h * D, dtype=t.bfloat16, device="cuda") for n, h in (("q", H), ("k", kv), ("v", kv), ("out", H))}
        lens = ints(rng.integers(0, 100, B))
        ws = t.zeros(d.h.attention_workspace(B, 1, H), dtype=t.uint8, device="cuda")
        st, g = t.cuda.Stream(), t.cuda.CUDAGraph()
        t.cuda.synchronize()
        with t.cuda.graph(g, stream=st):
            s = t.cuda.current_stream().cuda_stream
            d.h.append(io["k"].data_ptr(), io["v"].data_ptr(), "bf16", B, 1, lens.data_ptr(), rotary=turn.h, q=io["q"].data_ptr(),
                       q_out=io["q"].data_ptr(), heads=H, stream=s)
            d.h.attention(io["q"].data_ptr(), io["out"].data_ptr(), B, 1, H, lens.data_ptr(), ws=ws.data_ptr(), ws_bytes=ws.numel(),
                          stream=s)
        made.append((d, io, lens, g, st, ws))
    for step in range(3):
        for d, io, lens, g, st, ws in made:
            for n in ("q", "k", "v"):
                io[n].copy_(dev(rng.standard_normal(io[n].shape).astype(np.float32)))
        held = [{n: io[n].float().cpu().numpy() for n in ("q", "k", "v")} for d, io, *_ in made]
        t.cuda.synchronize()
        for d, io, lens, g, st, ws in made:
            with t.cuda.stream(st):
                g.replay()
        t.cuda.synchronize()
        for (d, io, lens, g, st, ws), x in zip(made, held):
            n = lens.cpu().numpy()
            at = (prefix + n)[:, None]
            d.ref.k, d.ref.v = d.t["k"].float().cpu().numpy(), d.t["v"].float().cpu().numpy()
            y, e = turn.bound(x["k"].reshape(B, 1, kv, D), at, "bf16")
            for b in range(B):
                pg, off = d.ref.slot(d.ref.table[b], n[b])
                near(d.ref.k[pg, :, off], y[b, 0], e[b, 0])
                assert np.array_equal(d.ref.v[pg, :, off], x["v"][b].reshape(kv, D))
            q = io["q"].float().cpu().numpy().reshape(B, 1, H, D)
            near(q, *turn.bound(x["q"].reshape(B, 1, H, D), at, "bf16"))
            near(io["out"].float().cpu().numpy().reshape(q.shape), *d.ref.attention(q, n, [1] * B, D ** -0.5))
            assert int(ws[:4].view(t.int32)[0]) == 0
            lens += 1


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,heads,dim,page", [(1, 8, 64, 64), (3, 14, 64, 16), (1, 32, 128, 48), (5, 14, 128, 64), (4, 32, 64, 32)])
def test_attention_many_sequences(dtype, T, heads, dim, page):
    """Enough sequences that each one's own part is a warp's: stale memory, pages that are none, ragged counts."""
    rng = np.random.default_rng(T * heads + page)
    B, kv, prefix = 24, 2, 70
    ref = Cache(B, -(-150 // page), -(-prefix // page), prefix, kv, dim, page, dtype, rng, fill=np.nan)
    lens, new = rng.integers(0, 140, B), rng.integers(0, T + 1, B)
    lens[:4] = 0, 15, 16, 127
    for ids, n in [(ref.prefix_table, prefix)] + [(ref.table[b], lens[b] + new[b]) for b in range(B)]:
        for p in range(n):
            pg, off = ref.slot(ids, p)
            ref.k[pg, :, off], ref.v[pg, :, off] = rounded(rng.standard_normal((2, kv, dim)), dtype)
    ref.table[5:9, 0], ref.table[9, -1] = -1, ref.n_pages
    check(OnDevice(ref), rng.standard_normal((B, T, heads, dim)), lens, new)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,heads", [(6, 4), (5, 14)])
def test_attention_many_sequences_future_values(dtype, T, heads):
    """The same where rows that later tokens of the call see are not finite."""
    rng = np.random.default_rng(T + heads)
    B, kv, dim = 20, 2, 64
    ref = Cache(B, 3, 1, 40, kv, dim, 64, dtype, rng)
    lens = rng.integers(0, 180 - T, B)
    lens[:3] = 0, 62, 126
    for b in range(0, B, 2):
        for t, what in ((2, np.nan), (4, np.inf)):
            pg, off = ref.slot(ref.table[b], lens[b] + t)
            ref.v[pg, :, off, ::3] = what
    d = OnDevice(ref)
    q = rng.standard_normal((B, T, heads, dim))
    got = attend(d, q, lens, None)
    clean = Cache.__new__(Cache)
    clean.__dict__ = dict(ref.__dict__, v=np.nan_to_num(ref.v, posinf=0, neginf=0))
    want, bound = clean.attention(rounded(q, dtype), lens, [T] * B, dim ** -0.5)
    for b in range(B):
        n = 2 if b % 2 == 0 else T
        near(got[b, :n], want[b, :n], bound[b, :n], f"sequence {b}")
        if b % 2 == 0:
            assert not np.isfinite(got[b, 2:, :, ::3]).any() and np.isfinite(got[b, 2:, :, 1::3]).all()
            near(got[b, 2:, :, 1::3], want[b, 2:, :, 1::3], bound[b, 2:, :, 1::3], f"sequence {b}, other channels")
