"""n730_sample_rows on the GPU against the rule in 64 bits (``sample_ref.py``).

Bounds.  A bin's mass is held to half a unit of its fixed point per token and fp32's rounding of a deviation that
is at most 1 - exp(-bin width / T).  With room for 2048 tokens a bin and deviations below 1 the unit is 2^-17 or less
of an edge's weight, in the narrow bins that matter 2^-24; a token is accepted where its border lies within
2^-18 of the whole mass.  Borders that are settled in the sorted list alone (top-k, and what min-p or top-p leave of a
peaked row) are held to 2^-40.  prob: fp32's rounding and the border's slack.
"""
import numpy as np
import pytest

from gpu_util import dev, torch
from n730_b200 import sampling
from sample_ref import sample

pytestmark = pytest.mark.gpu
WIDE, NEAR = 2.0 ** -18, 2.0 ** -40


def tt(dtype):
    t = torch()
    return {"f16": t.float16, "bf16": t.bfloat16, "f32": t.float32}[dtype]


def draw(x, dtype="f32", t=None, k=None, p=None, q=None, u=None, ld=0, shift=0, stream=0):
    """The call's answers for rows x (numpy), and the rows as the type holds them."""
    B, V = x.shape
    tc = torch()
    ld = ld or V
    buf = tc.full((shift + B * ld,), 50.0, dtype=tt(dtype), device="cuda")
    rows = buf[shift:].view(B, ld)[:, :V]
    rows.copy_(dev(np.ascontiguousarray(x, np.float32)).to(tt(dtype)))
    arr = {}
    for name, v, kind in (("temperature", t, np.float32), ("top_k", k, np.int32), ("top_p", p, np.float32), ("min_p", q, np.float32)):
        if v is not None:
            arr[name] = dev(np.broadcast_to(np.asarray(v, kind), (B,)).copy())
    du = dev(np.broadcast_to(np.asarray(u, np.float32), (B,)).copy())
    out = [tc.full((B,), -7, dtype=tc.int32, device="cuda"), tc.full((B,), -7.0, device="cuda"), tc.full((B,), -7, dtype=tc.int32, device="cuda")]
    tc.cuda.synchronize()
    sampling.sample_rows(buf[shift:].data_ptr(), dtype, B, V, du.data_ptr(), out[0].data_ptr(), ld=ld, prob=out[1].data_ptr(),
                         kept=out[2].data_ptr(), stream=stream, **{n: v.data_ptr() for n, v in arr.items()})
    tc.cuda.synchronize()
    return [o.cpu().numpy() for o in out], rows.float().cpu().numpy()


def check(x, dtype="f32", t=1.0, k=0, p=1.0, q=0.0, u=0.5, slack=WIDE, **kw):
    (tok, prob, kept), rows = draw(x, dtype, t, k, p, q, u, **kw)
    B = len(x)
    t, k, p, q, u = (np.broadcast_to(np.asarray(v, d), (B,)) for v, d in ((t, np.float32), (k, np.int64), (p, np.float32),
                                                                          (q, np.float32), (u, np.float32)))
    for r in range(B):
        tokens, probs, counts = sample(rows[r], float(t[r]), int(k[r]), float(p[r]), float(q[r]), float(u[r]), slack)
        assert tok[r] in tokens, (r, tok[r], sorted(tokens)[:8], t[r], k[r], p[r], q[r], u[r])
        assert kept[r] in counts, (r, kept[r], sorted(counts)[:8], t[r], k[r], p[r], q[r])
        want = probs[int(tok[r]), int(kept[r])]
        assert abs(prob[r] - want) <= (2.0 ** -22 + 4 * slack) * want, (r, prob[r], want)


def rows(rng, B, V, spread=2.2, peaks=0):
    x = spread * rng.standard_normal((B, V))
    for r in range(B):
        x[r, rng.integers(0, V, min(peaks, V))] += 4 + 8 * rng.random(min(peaks, V))
    return x


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 7, 100, 1000, 4099, 50257, 152064])
def test_settings(dtype, V):
    """Every kind of cut alone and together, over rows of all lengths."""
    rng = np.random.default_rng(V)
    sets = [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.8, 0, 1.0, 0.05), (1.2, 400, 0.99, 0.01),
            (0.0, 5, 0.5, 0.5), (1.0, 1, 1.0, 0.0), (0.05, 64, 1.0, 0.0), (2.5, 2000, 0.999, 0.0), (1.3, 1500, 1.0, 1e-4),
            (30.0, 0, 0.5, 0.0), (1.0, V, 0.9, 0.0), (1.0, V + 5, 1.0, 0.0), (0.6, 0, 0.3, 0.5)]
    t, k, p, q = (np.array(c) for c in zip(*sets))
    check(rows(rng, len(sets), V, peaks=24), dtype, t, k, p, q, rng.random(len(sets)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_top_k_is_exact(dtype):
    """Rows whose cut a sorted list settles: no border but the 64-bit sums' own."""
    rng = np.random.default_rng(5)
    B = 64
    check(rows(rng, B, 32001, peaks=30), dtype, 0.7, 50, rng.choice([1.0, 0.9, 0.5], B), rng.choice([0.0, 0.05], B), rng.random(B), slack=NEAR)


def test_numbers_at_the_ends():
    """u = 0 takes the first kept token, the largest number below 1 the last, numbers outside [0, 1) the nearest."""
    rng = np.random.default_rng(6)
    x = rows(rng, 6, 3000)
    u = np.array([0.0, 1 - 2.0 ** -24, -3.0, 7.0, np.nan, 0.999])
    for kw in (dict(k=20), dict(q=0.02), dict(p=0.4)):
        (tok, prob, kept), held = draw(x, "f32", 1.0, kw.get("k"), kw.get("p"), kw.get("q"), u)
        for r, at in ((0, "first"), (2, "first"), (4, "first"), (3, "last")):
            order = np.lexsort((np.arange(3000), -held[r]))
            assert tok[r] == order[0 if at == "first" else kept[r] - 1]
    check(x[:2], u=u[:2], k=20, slack=NEAR)


@pytest.mark.parametrize("V", [3, 1000, 40000, 152064])
def test_equal_logits(V):
    """Rows of one value, of two, and of a coarse grid: ties go by index however many they are."""
    rng = np.random.default_rng(V)
    x = np.zeros((10, V))
    x[1] = -3.5
    x[2, V // 2:] = 1.0
    x[3:5] = np.round(2 * rng.standard_normal((2, V)))
    x[5:] = np.round(8 * rng.standard_normal((5, V))) / 8
    for k, p, q in ((0, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.3), (min(V, 700), 0.7, 0.0), (min(V, 30000), 0.9, 0.0),
                    (min(V, 30000), 1.0, 0.01), (2, 1.0, 0.0)):
        check(x, "f32", 1.0, k, p, q, rng.random(10), slack=NEAR if k == 2 else WIDE)
    # sums of equal weights are exact: the picks are too
    u = np.arange(8) / 8
    (tok, prob, kept), _ = draw(np.zeros((8, V)), "f32", 1.0, None, None, None, u)
    assert np.array_equal(tok, np.floor(u * V).astype(int)) and np.all(kept == V)
    (tok, _, kept), _ = draw(np.zeros((8, V)), "f32", 1.0, None, 0.5, None, u)
    assert np.all(kept == -(-V // 2)) and np.array_equal(tok, np.floor(u * -(-V // 2)).astype(int))


def test_masked_rows():
    """-inf, NaN, the types' lowest values, +inf, rows without any token."""
    rng = np.random.default_rng(8)
    x = rows(rng, 12, 5000)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, ::2], x[2, 1::4] = -np.inf, np.nan
    x[3, 7:] = -np.inf
    x[4, 100:] = -3.4e38
    x[5, 100:] = -65504.0
    x[6, [5, 900]] = np.inf
    x[7, :] = -3.4e38
    x[8, 0], x[8, 1:] = 3.4e38, -3.4e38
    x[9, 17] = np.inf
    x[9, 18:] = -np.inf
    x[10, 1:] = -np.inf
    x[11, ::3] = -0.0
    x[11, 1::3] = 0.0
    for t in (1.0, 0.01, 0.0):
        for k, p, q in ((0, 1.0, 0.0), (30, 0.9, 0.0), (0, 0.8, 0.0), (0, 1.0, 0.1), (200, 1.0, 0.0)):
            check(x, "f32", t, k, p, q, rng.random(12))
    check(np.clip(x, -65504, 65504), "f16", 0.7, 120, 0.99, 0.0, rng.random(12))


def test_odd_settings():
    """Tiny and huge temperatures, cuts that are off or out of range."""
    rng = np.random.default_rng(9)
    x = rows(rng, 7, 2500)
    check(x, "f32", [1e-30, 1e-5, 1e5, np.inf, -1.0, np.nan, 1.0], 0, 1.0, 0.0, rng.random(7))
    (a, _, ka), _ = draw(x, "f32", 0.8, -4, 1.5, -0.1, 0.3)
    (b, _, kb), _ = draw(x, "f32", 0.8, None, np.nan, np.nan, 0.3)
    assert np.array_equal(a, b) and np.array_equal(ka, kb) and np.all(ka == 2500)
    (a, _, ka), _ = draw(x, "f32", 0.8, None, 0.0, None, 0.9)
    assert np.array_equal(a, x.astype(np.float32).argmax(1)) and np.all(ka == 1)
    (a, _, _), _ = draw(x, "f32", u=np.full(7, 0.4))
    (b, _, _), _ = draw(x, "f32", 1.0, 0, 1.0, 0.0, 0.4)
    assert np.array_equal(a, b)


@pytest.mark.parametrize("dtype,ld,shift", [("f32", 5003, 0), ("f16", 5001, 0), ("bf16", 5000, 3), ("f32", 5000, 1), ("f16", 5008, 8)])
def test_strides(dtype, ld, shift):
    """Rows on any element; what lies between rows is not looked at."""
    rng = np.random.default_rng(ld)
    check(rows(rng, 5, 4999), dtype, 0.9, [0, 40, 0, 3000, 0], [0.9, 1, 1, 0.9, 0.5], 0.0, rng.random(5), ld=ld, shift=shift)


def test_long_rows():
    """More logits than a cluster's shared memory holds."""
    rng = np.random.default_rng(11)
    check(rows(rng, 3, 600011, peaks=40), "bf16", [1.0, 0.7, 1.2], [0, 50, 0], [0.95, 0.9, 1.0], 0.0, rng.random(3))


def test_many_rows_and_again():
    """More rows than clusters fit at once; the same inputs give the same answers."""
    rng = np.random.default_rng(12)
    x, u = rows(rng, 300, 2049), rng.random(300)
    a, _ = draw(x, "f32", 0.9, None, 0.95, None, u)
    b, _ = draw(x, "f32", 0.9, None, 0.95, None, u)
    assert all(np.array_equal(p, q) for p, q in zip(a, b))
    check(x[:40], "f32", 0.9, 0, 0.95, 0.0, u[:40])


def test_distribution():
    """Numbers on a grid reproduce the probabilities: counts within one of n * p a token."""
    rng = np.random.default_rng(13)
    x = np.tile(rows(rng, 1, 37, 1.0), (2000, 1))
    u = (np.arange(2000) + 0.5) / 2000
    (tok, _, _), held = draw(x, "f32", 1.0, None, None, None, u)
    w = np.exp(held[0].astype(np.float64))
    assert np.all(np.abs(np.bincount(tok, minlength=37) - 2000 * w / w.sum()) <= 1.001)


def test_graph_and_stream():
    """Captured into a graph and replayed with new logits, on a stream of its own."""
    t = torch()
    rng = np.random.default_rng(14)
    x = [rows(rng, 4, 3001) for _ in range(2)]
    d = t.zeros(4, 3001, device="cuda")
    u, tok = dev(rng.random(4).astype(np.float32)), t.zeros(4, dtype=t.int32, device="cuda")
    p = dev(np.full(4, 0.9, np.float32))
    st = t.cuda.Stream()
    g = t.cuda.CUDAGraph()
    t.cuda.synchronize()
    with t.cuda.graph(g, stream=st):
        sampling.sample_rows(d.data_ptr(), "f32", 4, 3001, u.data_ptr(), tok.data_ptr(), top_p=p.data_ptr(),
                             stream=t.cuda.current_stream().cuda_stream)
    for y in x:
        d.copy_(dev(y.astype(np.float32)))
        g.replay()
        t.cuda.synchronize()
        want = draw(y, "f32", None, None, 0.9, None, u.cpu().numpy())[0][0]
        assert np.array_equal(tok.cpu().numpy(), want)


@pytest.mark.parametrize("dtype,B,V", [("f32", 74, 50000), ("f32", 74, 80000), ("f16", 74, 160000), ("bf16", 90, 20000), ("f32", 200, 5000),
                                       ("bf16", 400, 900), ("f16", 60, 156000), ("bf16", 90, 28000), ("f16", 186, 28000), ("bf16", 93, 19000), ("f32", 52, 78001)])
def test_rows_in_smaller_clusters(dtype, B, V):
    """Many rows: 4, 2 and one CTA a row, every kind of cut among them."""
    rng = np.random.default_rng(V)
    t, k = rng.choice([0.0, 0.5, 0.9, 1.3], B), rng.choice([0, 0, 30, 300, 3000], B)
    check(rows(rng, B, V, peaks=24), dtype, t, k, rng.choice([1.0, 0.9, 0.99], B), rng.choice([0.0, 0.0, 0.02], B), rng.random(B))


def test_two_calls_at_once():
    """On two streams, each with its own outputs: nothing is shared between calls."""
    t = torch()
    rng = np.random.default_rng(15)
    x = [dev(rows(rng, 30, 32000, peaks=20).astype(np.float32)) for _ in range(2)]
    u, k = dev(rng.random(30).astype(np.float32)), dev(np.where(np.arange(30) % 2, 40, 0).astype(np.int32))
    p = dev(np.full(30, 0.95, np.float32))
    out = [[t.zeros(30, dtype=t.int32, device="cuda") for _ in range(2)] for _ in range(2)]
    st = [t.cuda.Stream() for _ in range(2)]
    t.cuda.synchronize()
    for i in range(40):
        for a in range(2):
            sampling.sample_rows(x[a].data_ptr(), "f32", 30, 32000, u.data_ptr(), out[a][i % 2].data_ptr(), top_k=k.data_ptr(),
                                 top_p=p.data_ptr(), stream=st[a].cuda_stream)
    t.cuda.synchronize()
    for a in range(2):
        want = draw(x[a].cpu().numpy(), "f32", None, k.cpu().numpy(), 0.95, None, u.cpu().numpy())[0][0]
        assert np.array_equal(out[a][0].cpu().numpy(), want) and np.array_equal(out[a][1].cpu().numpy(), want)
