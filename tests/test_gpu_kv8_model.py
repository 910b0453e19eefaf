"""Models that keep their cache in 8 bits (``Engine(kv_bits=8)``) against the oracle decoder with the same
cache: its K and V go through the numpy statement of the 8-bit cache (``kv8_ref.py``), 64 tokens at a time as
the engine's prefill does.

Tolerance: the logit bar of the fp16 cache (1e-2 of the largest logit: fp16 products of the weights) twice.  The second
time is for codes that round the other way because the engine's K and V are about 2^-11 off the oracle's: two
roundings of values e apart on a grid of step s differ by sqrt(s e) in the mean square, here
sqrt(2^-7 2^-11) = 2^-9 of a block's largest value for values of a quarter of it, below 1e-2 of each, and a head's
sums over positions and channels take the mean of them.
"""
import numpy as np
import pytest

from gpu_util import rel_err
from kv8_ref import Cache, decode
from n730_b200 import synthetic
from n730_b200.engine import Engine, load_tensors
from n730_b200.batching import ContinuousBatcher
from oracle.model import OracleDecoder, apply_rope, attention, rms_norm, swiglu
from test_gpu_model import _blocks, _oracle_weights

pytestmark = pytest.mark.gpu
TOL = 2e-2


class Oracle8(OracleDecoder):
    """The oracle decoder over an 8-bit cache, `chunk` rows appended at a time."""

    def __init__(self, cfg, weights, max_pos, chunk=64):
        super().__init__(cfg, weights, max_pos)
        c, rng = self.cfg, np.random.default_rng(0)
        self.chunk = chunk
        self.caches = []
        for _ in range(c.num_hidden_layers):
            k = Cache(max_pos // 64, max_pos // 64, 1, c.num_kv_heads, c.head_dim, 64, 16, "int8", rng, fill=0)
            k.table[0] = np.arange(max_pos // 64)
            self.caches.append(k)

    def layer(self, i, x, offset):
        c, p, cache = self.cfg, f"model.layers.{i}", self.caches[i]
        h = rms_norm(x, self._norm(f"{p}.input_layernorm.weight"), c.rms_norm_eps)
        q, k, v = (self._lin(h, f"{p}.self_attn.{n}_proj") for n in "qkv")
        q = apply_rope(q, c.num_attention_heads, c.head_dim, offset, self.cos, self.sin)
        k = apply_rope(k, c.num_kv_heads, c.head_dim, offset, self.cos, self.sin)
        n = len(x)
        shape = (1, n, c.num_kv_heads, c.head_dim)
        cache.append(k.reshape(shape), v.reshape(shape), [offset], [n])
        K, V, _ = cache.dense(0, offset + n)
        a = attention(q, K.transpose(1, 0, 2).reshape(offset + n, -1).astype(np.float32),
                      V.transpose(1, 0, 2).reshape(offset + n, -1).astype(np.float32), c.num_attention_heads,
                      c.num_kv_heads, c.head_dim, offset)
        x = (x + self._lin(a, f"{p}.self_attn.o_proj")).astype(np.float32)
        h2 = rms_norm(x, self._norm(f"{p}.post_attention_layernorm.weight"), c.rms_norm_eps)
        return (x + self._lin(swiglu(self._lin(h2, f"{p}.mlp.gate_proj"), self._lin(h2, f"{p}.mlp.up_proj")),
                              f"{p}.mlp.down_proj")).astype(np.float32)

    def forward(self, ids):
        for i in range(0, len(ids), self.chunk):
            y = super().forward(ids[i:i + self.chunk])
        return y


@pytest.fixture(scope="module", params=[("tiny", "int4_g128"), ("tiny-gqa7", "mixed_05b"), ("tiny-128", "int4_g128")])
def model(request, tmp_path_factory):
    shape_name, pmap = request.param
    shape = synthetic.SHAPES[shape_name]
    path = tmp_path_factory.mktemp("m8") / f"{shape_name}.n730"
    synthetic.write_n730(path, shape, pmap, seed=3)
    blocks = _blocks(path)
    return shape, blocks, _oracle_weights(blocks)


def _engine(shape, blocks, **kw):
    e = Engine(shape, max_ctx=512, max_batch=kw.pop("max_batch", 4), max_prefill=64, kv_bits=8, **kw)
    load_tensors(e, blocks)
    e.finalize()
    return e


@pytest.mark.parametrize("graphs,pdl", [(True, True), (False, False)])
def test_prefill_then_decode(model, graphs, pdl):
    shape, blocks, w = model
    e = _engine(shape, blocks, use_graphs=graphs, use_pdl=pdl)
    orc = Oracle8(shape, w, 512)
    rng = np.random.default_rng(11)
    prompt = rng.integers(0, shape.vocab, 100)  # crosses a 64-token prefill chunk and ends inside a block
    assert rel_err(e.forward(prompt), orc.forward(prompt)) <= TOL
    tok = int(rng.integers(0, shape.vocab))
    for step in range(8):
        y, yr = e.decode([tok])[0], orc.forward([tok])
        assert rel_err(y, yr) <= TOL, f"step {step}"
        tok = int(np.argmax(yr))
    y, yr = e.forward([tok, 1, 2]), orc.forward([tok, 1, 2])
    assert rel_err(y, yr) <= TOL
    assert e.seq_len(0) == 111 and not e.info()["persistent_decode"]
    assert e.info()["kv_bytes_per_pos"] == shape.layers * 2 * shape.kv_heads * (16 * shape.head_dim + 4) // 16
    e.close()


def test_batched_ragged_decode(model):
    shape, blocks, w = model
    e = _engine(shape, blocks)
    rng = np.random.default_rng(5)
    oracles = [Oracle8(shape, w, 512) for _ in range(3)]
    for b in range(3):
        p = rng.integers(0, shape.vocab, 7 + 13 * b)
        assert rel_err(e.forward(p, seq=b), oracles[b].forward(p)) <= TOL
    toks = rng.integers(0, shape.vocab, 3)
    for step in range(4):
        y = e.decode(toks)
        for b in range(3):
            assert rel_err(y[b], oracles[b].forward([toks[b]])) <= TOL, (step, b)
        toks = np.argmax(y, axis=1)
    e.close()


def test_batcher_reuses_pages(model):
    """Requests through few slots and pages: a page's old codes and scales are not seen by the next request."""
    shape, blocks, w = model
    e = _engine(shape, blocks, max_batch=2, kv_pool_pages=4)
    b = ContinuousBatcher(e, keep_logits=True)
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, shape.vocab, n) for n in (70, 5, 33, 64)]
    ids = [b.submit(p, 3) for p in prompts]
    done = b.run()
    for rid, p in zip(ids, prompts):
        orc, r = Oracle8(shape, w, 512), done[rid]
        y = orc.forward(p)
        for k, (tok, lg) in enumerate(zip(r.tokens, r.logits)):
            assert rel_err(lg, y) <= TOL, (rid, k)
            y = orc.forward([tok])
    e.close()


@pytest.fixture(scope="module")
def odd_model(tmp_path_factory):
    """One KV head, three layers."""
    shape = synthetic.ModelShape(256, 3, 4, 1, 64, 512, 1000, 1e6, 1e-6, False)
    path = tmp_path_factory.mktemp("m8odd") / "odd.n730"
    synthetic.write_n730(path, shape, "int4_g128", seed=6)
    blocks = _blocks(path)
    return shape, blocks, _oracle_weights(blocks)


@pytest.mark.parametrize("page,pool", [(16, 31), (48, 11), (80, 0)])
def test_odd_pools(odd_model, page, pool):
    """Pages, heads and blocks whose product is odd: every layer's codes still lie where copies can start."""
    shape, blocks, w = odd_model
    e = _engine(shape, blocks, page_size=page, kv_pool_pages=pool, max_batch=1)
    orc = Oracle8(shape, w, 512)
    rng = np.random.default_rng(page)
    prompt = rng.integers(0, shape.vocab, 90)
    assert rel_err(e.forward(prompt), orc.forward(prompt)) <= TOL
    for tok in rng.integers(0, shape.vocab, 3):
        assert rel_err(e.decode([tok])[0], orc.forward([tok])) <= TOL
    e.close()


@pytest.mark.parametrize("prompt", [9, 64])
def test_large_values_with_exact_gemv(model, prompt):
    """V far beyond fp16's range: with the fp32 GEMV prompts answer like single tokens, by either kernel."""
    from n730_b200.engine import BIAS_SLOTS
    shape, blocks, w = model
    e = Engine(shape, max_ctx=512, max_batch=1, max_prefill=64, kv_bits=8, exact_gemv=True)
    load_tensors(e, blocks)
    w = dict(w)
    for i in range(shape.layers):
        name = f"model.layers.{i}.self_attn.v_proj.bias"
        w[name] = w[name].astype(np.float32).copy()
        w[name][::16] += 2e5
        e.set_vector(i, BIAS_SLOTS["self_attn.v_proj"], w[name])
    e.finalize()
    orc = Oracle8(shape, w, 512)
    rng = np.random.default_rng(prompt)
    ids = rng.integers(0, shape.vocab, prompt)
    assert rel_err(e.forward(ids), orc.forward(ids)) <= TOL
    tok = int(rng.integers(0, shape.vocab))
    assert rel_err(e.decode([tok])[0], orc.forward([tok])) <= TOL
    e.close()


def test_sampled_steps_moves_and_rollback(model):
    """Greedy sampled steps, a sequence cut back (its block keeps the scale) and grown again, moved to another slot;
    prefill chunks of one token."""
    shape, blocks, w = model
    e = _engine(shape, blocks, max_batch=3)
    orc = Oracle8(shape, w, 512)
    rng = np.random.default_rng(17)
    ids = rng.integers(0, shape.vocab, 65)  # the second chunk is one token
    assert rel_err(e.forward(ids, seq=1), orc.forward(ids)) <= TOL
    e.set_seq_len(1, 41)
    orc.seq_len = 41
    ids = rng.integers(0, shape.vocab, 12)
    assert rel_err(e.forward(ids, seq=1), orc.forward(ids)) <= TOL
    e.seq_move(0, 1)
    tok = int(rng.integers(0, shape.vocab))
    for _ in range(3):
        y = orc.forward([tok])
        nxt = int(e.decode_sample([tok], temperature=0.0)[0])
        assert y[nxt] >= y.max() - TOL * np.abs(y).max()
        tok = nxt
    assert e.seq_len(0) == 56
    e.reset()
    orc = Oracle8(shape, w, 512)
    assert rel_err(e.forward(ids), orc.forward(ids)) <= TOL
    e.close()


@pytest.mark.parametrize("kw", [dict(stream_depth=2), dict(exact_gemv=True), dict(per_op_decode=1), dict(per_op_decode=-1)])
def test_other_paths_agree(model, kw):
    """Streamed layers give the resident engine's bits, the fp32 GEMV its logits; the decode path is the same whatever
    is asked for."""
    shape, blocks, w = model
    a, b = _engine(shape, blocks, max_batch=2), _engine(shape, blocks, max_batch=2, **kw)
    rng = np.random.default_rng(19)
    ids = rng.integers(0, shape.vocab, 70)
    steps = [(x.forward(ids), x.forward(ids[:9], seq=1), x.decode([3, 5]).copy(), x.decode([7]).copy()) for x in (a, b)]
    for x, y in zip(*steps):
        if "exact_gemv" in kw:
            assert rel_err(y, x) <= TOL
        else:
            assert np.array_equal(x, y)
    a.close()
    b.close()


def test_refused_configurations():
    shape = synthetic.SHAPES["tiny"]
    for kw in (dict(kv_bits=4), dict(kv_bits=8, page_size=24), dict(kv_bits=-8)):
        with pytest.raises(RuntimeError, match="kv_bits"):
            Engine(shape, max_ctx=64, **kw)
