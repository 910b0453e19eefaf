"""What is measured of decoding many continuations of one prompt: rotary positions, rows written into
the 16-bit paged cache, attention over a prefix that the whole batch shares and each sequence's own
positions, and sampling with each row's temperature, top-k, top-p and min-p from given numbers.

The cache is paged, ``[pages][kv heads][page_size][head_dim]`` of 16-bit values.  The prefix's position
p lies in page ``prefix_table[p // page_size]``; position p of sequence b's own part in page
``table[b][p // page_size]``, and stands ``prefix + p`` tokens behind the start.

``run`` computes the operators in their plain form with elementary torch operations, or, where ``own``
is true, through the framework's entry points (``n730_b200.kv16``, ``n730_b200.sampling``).
"""
import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}


# ----------------------------------------------------------------------------- cases
def _rotary(name, rows, heads, dim, part, layout, scaling, dtype, far):
    return {"name": name, "op": "rotary", "rows": rows, "heads": heads, "dim": dim, "part": part, "layout": layout,
            "scaling": scaling, "dtype": dtype, "far": far}


def _append(name, batch, tokens, prefix, ctx, heads, kv, dim, part, layout, scaling, page, dtype, ragged):
    return {"name": name, "op": "append", "batch": batch, "tokens": tokens, "prefix": prefix, "ctx": ctx, "heads": heads,
            "kv": kv, "dim": dim, "part": part, "layout": layout, "scaling": scaling, "page": page, "dtype": dtype,
            "ragged": ragged}


def _attend(name, batch, tokens, prefix, ctx, heads, kv, dim, page, dtype, ragged):
    return {"name": name, "op": "attention", "batch": batch, "tokens": tokens, "prefix": prefix, "ctx": ctx,
            "heads": heads, "kv": kv, "dim": dim, "page": page, "dtype": dtype, "ragged": ragged}


def _sample(name, batch, vocab, mix, dtype):
    return {"name": name, "op": "sample", "batch": batch, "vocab": vocab, "mix": mix, "dtype": dtype}


def listed():
    return [
        # fp32 rows of a checker or a draft model, angles far beyond the trained context
        _rotary("rotary_far_f32", 2048, 28, 128, 128, "half", "ramp", "f32", 1 << 20),
        # half of each head rotated, pairs side by side: another model family's layout
        _rotary("rotary_part", 4099, 16, 64, 32, "interleaved", "none", "bf16", 4099),
        # one new token of one continuation, 7B heads: latency only
        _append("append_step", 1, 1, 2048, 64, 28, 4, 128, 128, "half", "none", 64, "f16", False),
        # one new token of each of a batch behind a long prompt, 72B heads
        _append("append_batch", 64, 1, 8192, 512, 64, 8, 128, 128, "half", "bands", 64, "bf16", True),
        # the prompt itself written once, page by page
        _append("append_prompt", 1, 4133, 0, 4133, 28, 4, 128, 64, "interleaved", "linear", 64, "f16", False),
        # four samples of a short prompt, 0.5B heads
        _attend("attend_few", 4, 1, 501, 40, 14, 2, 64, 64, "f16", True),
        # a batch behind an instruction prompt that ends inside a page, 7B heads
        _attend("attend_batch", 32, 1, 8131, 512, 28, 4, 128, 64, "f16", True),
        # a large batch behind a long document, 72B heads
        _attend("attend_large", 128, 1, 16384, 256, 64, 8, 128, 64, "bf16", True),
        # five drafted tokens of each checked at once
        _attend("attend_drafts", 16, 5, 6001, 700, 28, 4, 128, 32, "bf16", True),
        # one row, the usual settings: latency
        _sample("sample_one", 1, 152064, "usual", "f32"),
        # a serving batch whose requests each bring their own settings, some greedy
        _sample("sample_batch", 64, 151936, "mixed", "f32"),
        # many rows whose whole distribution counts: no cut, a high temperature
        _sample("sample_open", 192, 152064, "open", "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention", "sample", "sample"])
    kv, group, dim = rng.choice([(4, 7, 128), (8, 8, 128), (2, 7, 64), (2, 2, 64), (1, 5, 128), (8, 1, 64), (1, 16, 128)])
    page = rng.choice([16, 32, 64, 64, 128])
    dtype = rng.choice(["f16", "bf16"])
    ragged = rng.random() < 0.6
    part = rng.choice([dim, dim, dim // 2, dim // 4 * 3])
    layout = rng.choice(["half", "interleaved"])
    scaling = rng.choice(["none", "linear", "base", "ramp", "bands"])
    if op == "rotary":
        rows = _log(rng, 1, 4099)
        c = _rotary("", rows, rng.choice([1, 8, 14, 28, 64]), dim, part, layout, scaling, rng.choice(["f32", "f16", "bf16"]),
                    _log(rng, 64, 1 << 21))
    elif op == "append":
        batch = _log(rng, 1, 128)
        tokens = 1 if rng.random() < 0.6 else _log(rng, 2, 4096 // batch + 2)
        c = _append("", batch, tokens, rng.choice([0, _log(rng, 1, 100000)]), tokens + _log(rng, 1, 500), kv * group, kv, dim,
                    part, layout, scaling, page, rng.choice([dtype, dtype, "f32"]), ragged)
    elif op == "attention":
        batch = _log(rng, 1, 128)
        tokens = 1 if rng.random() < 0.65 else _log(rng, 2, 8 if batch > 4 else 256)
        ctx = tokens + _log(rng, 1, 900)
        most = 128 * 64 * 16384 // (batch * kv * group * tokens) - ctx
        c = _attend("", batch, tokens, min(most, _log(rng, 33, 16384)), ctx, kv * group, kv, dim, page, dtype, ragged)
    else:
        vocab = _log(rng, 500, 152064)
        batch = _log(rng, 1, min(256, 192 * 152064 // vocab))
        c = _sample("", batch, vocab, rng.choice(["usual", "mixed", "mixed", "open", "nucleus"]), rng.choice(["f32", "f32", "f16", "bf16"]))
    del c["name"]
    return c


# ----------------------------------------------------------------------------- inputs
def _frequencies(part, scaling):
    """Radians per position of each pair, and the factor of rotated channels."""
    f = 1e6 ** (-np.arange(0, part, 2) / part)
    orig, factor = 32768, 4.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "base":
        return (1e6 * factor ** (part / max(part - 2, 1))) ** (-np.arange(0, part, 2) / part), 1.0
    if scaling == "ramp":  # by the number of a pair's turns over the trained context
        lo, hi = (part * np.log(orig / (2 * np.pi * turns)) / (2 * np.log(1e6)) for turns in (32, 1))
        lo, hi = max(np.floor(lo), 0), min(np.ceil(hi), part - 1)
        keep = 1 - np.clip((np.arange(part // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        return f / factor * (1 - keep) + f * keep, 0.1 * np.log(factor) + 1
    if scaling == "bands":
        turns = orig * f / (2 * np.pi)
        keep = np.clip((turns - 1) / (4 - 1), 0, 1)
        return f / factor * (1 - keep) + f * keep, 1.0
    return f, 1.0


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, dtype, dev = case["op"], TYPES[case["dtype"]], "cuda"
    s = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def ints(x):
        return torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(dev)

    if op == "sample":
        batch, vocab, mix = case["batch"], case["vocab"], case["mix"]
        x = normal(batch, vocab).mul_(1.0 if mix == "open" else 2.2)
        if mix != "open":  # the few tokens that fit
            at = torch.randint(0, vocab, (batch, 1), generator=gen, device=dev)
            at = (at + torch.arange(48, device=dev) * (vocab // 48)) % vocab
            x.scatter_add_(1, at, 4 + 8 * torch.rand(batch, 48, generator=gen, device=dev))
        s["x"] = x.to(dtype)
        pick = (lambda of: rng.choice(of, batch)) if mix == "mixed" else lambda of: np.full(batch, of[0])
        t, k, p, m = {"usual": ([0.7], [50], [0.9], [0.0]), "nucleus": ([0.9], [0], [0.95], [0.0]),
                      "open": ([1.3], [0], [1.0], [0.0]),
                      "mixed": ([0.0, 0.6, 0.8, 1.0, 1.2], [0, 0, 20, 50, 400], [1.0, 0.9, 0.95, 0.99], [0.0, 0.0, 0.02, 0.1])}[mix]
        for name, of, kind in (("temperature", t, np.float32), ("top_k", k, np.int32), ("top_p", p, np.float32), ("min_p", m, np.float32)):
            s[name] = torch.from_numpy(pick(of).astype(kind)).to(dev)
        s["u"] = torch.rand(batch, generator=gen, device=dev)
        s["token"] = torch.zeros(batch, dtype=torch.int32, device=dev)
        s["kept"] = torch.zeros(batch, dtype=torch.int32, device=dev)
        s["prob"] = torch.zeros(batch, device=dev)
        return s
    if op != "attention":
        freq, s["factor"] = _frequencies(case["part"], case["scaling"])
        s["freq"] = torch.from_numpy(freq).to(dev)
    if op == "rotary":
        s["x"] = normal(case["rows"], case["heads"], case["dim"]).to(dtype)
        s["y"] = torch.zeros_like(s["x"])
        first = int(rng.integers(0, max(1, case["far"] - case["rows"])))
        s["pos"] = ints(first + np.arange(case["rows"]))
        return s
    batch, tokens, ctx, kv, dim, page, heads = (case[k] for k in ("batch", "tokens", "ctx", "kv", "dim", "page", "heads"))
    kept = torch.float16 if case["dtype"] == "f16" else torch.bfloat16
    most, shared = -(-ctx // page), -(-case["prefix"] // page) if op == "attention" else 0
    pages = rng.permutation(batch * most + shared)
    s["k"], s["v"] = normal(len(pages), kv, page, dim).to(kept), normal(len(pages), kv, page, dim).to(kept)
    s["prefix_table"], s["table"] = ints(pages[:shared]), ints(pages[shared:].reshape(batch, most))
    if op == "append":  # reads and writes no page of the prefix: any ids stand for them
        s["prefix_table"] = ints(np.arange(-(-case["prefix"] // page)) % len(pages))
    s["prefix"] = ints([case["prefix"]])
    total = np.full(batch, ctx)
    new = np.full(batch, tokens)
    if case["ragged"]:
        total = rng.integers(max(1, ctx // 8), ctx + 1, batch)
        total[rng.integers(0, batch)] = ctx
        if tokens > 1:
            new = rng.integers(1, tokens + 1, batch)
            new[rng.integers(0, batch)] = tokens
    total = np.maximum(total, new)
    s["lens"], s["new"], s["all"] = ints(total - new), ints(new), ints(total)
    s["q"] = (2.0 * normal(batch, tokens, heads, dim)).to(dtype)
    s["out"] = torch.zeros_like(s["q"])
    if op == "append":
        s["x_k"], s["x_v"] = normal(batch, tokens, kv, dim).to(dtype), normal(batch, tokens, kv, dim).to(dtype)
    return s


# ----------------------------------------------------------------------------- plain form
def _turn(x, pos, s):
    """Rows x [..., heads, dim] rotated at positions pos [...], in 32 bits; angles in 64."""
    c = s["case"]
    part = c["part"]
    a = pos.double()[..., None] * s["freq"]
    cos, sin = (torch.cos(a) * s["factor"]).float()[..., None, :], (torch.sin(a) * s["factor"]).float()[..., None, :]
    y = x.float().clone()
    if c["layout"] == "half":
        x0, x1 = x[..., :part // 2].float(), x[..., part // 2:part].float()
        y[..., :part // 2], y[..., part // 2:part] = x0 * cos - x1 * sin, x1 * cos + x0 * sin
    else:
        x0, x1 = x[..., 0:part:2].float(), x[..., 1:part:2].float()
        y[..., 0:part:2], y[..., 1:part:2] = x0 * cos - x1 * sin, x1 * cos + x0 * sin
    return y


def _plain_append(s):
    c = s["case"]
    batch, tokens, page = c["batch"], c["tokens"], c["page"]
    t = torch.arange(tokens, device="cuda")
    at = s["lens"].long()[:, None] + t
    live = t < s["new"].long()[:, None]
    pos = at + s["prefix"].long()
    q, k = _turn(s["q"], pos, s), _turn(s["x_k"], pos, s)
    b = torch.arange(batch, device="cuda")[:, None].expand(-1, tokens)[live]
    at = at[live]
    pg = s["table"].long()[b, at // page]
    s["k"][pg, :, at % page] = k[live].to(s["k"].dtype)
    s["v"][pg, :, at % page] = s["x_v"][live].to(s["v"].dtype)
    return {"q": torch.where(live[..., None, None], q.to(s["q"].dtype), s["out"]), "k": s["k"], "v": s["v"]}


def _plain_attention(s):
    c = s["case"]
    batch, tokens, heads, kv, dim, prefix = (c[k] for k in ("batch", "tokens", "heads", "kv", "dim", "prefix"))
    rows = heads // kv * tokens
    q = s["q"].float().view(batch, tokens, kv, heads // kv, dim).permute(2, 0, 3, 1, 4).reshape(kv, batch * rows, dim)
    pool = [[x[table.long()].float().movedim(-3, 0).flatten(-3, -2) for x in (s["k"], s["v"])] for table in (s["prefix_table"], s["table"])]
    (k0, v0), (k1, v1) = pool
    k0, v0 = k0.reshape(kv, -1, dim)[:, :prefix], v0.reshape(kv, -1, dim)[:, :prefix]
    k1, v1 = k1.reshape(kv, batch, -1, dim), v1.reshape(kv, batch, -1, dim)
    x0 = (q @ k0.transpose(1, 2)).mul_(dim ** -0.5).view(kv, batch, rows, -1)
    x1 = (q.view(kv, batch, rows, dim) @ k1.transpose(2, 3)).mul_(dim ** -0.5)
    n = x1.shape[-1]
    t = torch.arange(tokens, device="cuda")
    sees = (s["lens"].long()[:, None] + t)[:, None, :, None]  # last own position of query t
    mask = (torch.arange(n, device="cuda") <= sees).expand(batch, heads // kv, tokens, n).reshape(batch, rows, n)
    x1 = x1.masked_fill(~mask, -float("inf"))
    top = torch.maximum(x0.amax(-1, keepdim=True), x1.amax(-1, keepdim=True))
    p0, p1 = x0.sub_(top).exp_(), x1.sub_(top).exp_()
    total = p0.sum(-1, keepdim=True) + p1.sum(-1, keepdim=True)
    stale = torch.arange(n, device="cuda") < s["all"].long()[:, None]
    v1 = torch.where(stale[None, :, :, None], v1, torch.zeros_like(v1))
    y = ((p0.view(kv, batch * rows, -1) @ v0).view(kv, batch, rows, dim) + p1 @ v1) / total
    y = y.view(kv, batch, heads // kv, tokens, dim).permute(1, 3, 0, 2, 4).reshape(batch, tokens, heads, dim)
    live = t < s["new"].long()[:, None]
    return {"out": torch.where(live[..., None, None], y.to(s["q"].dtype), s["out"])}


def _plain_sample(s):
    vocab = s["case"]["vocab"]
    x, order = torch.sort(s["x"].float(), dim=-1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    greedy = ~(t > 0)
    w = torch.exp((x - x[:, :1].double()) / torch.where(greedy, torch.ones_like(t), t))
    k = s["top_k"].long()[:, None]
    cut = torch.where((k > 0) & (k < vocab), k, torch.full_like(k, vocab))
    at = torch.arange(vocab, device="cuda")
    mass = torch.cumsum(torch.where(at < cut, w, torch.zeros_like(w)), -1)
    top_p = s["top_p"].double()[:, None]
    by_p = torch.where(top_p < 1, 1 + (mass < top_p * mass[:, -1:]).sum(-1, keepdim=True), cut)
    by_m = (w >= s["min_p"].double()[:, None]).sum(-1, keepdim=True)
    kept = torch.minimum(torch.minimum(cut, by_p), by_m).clamp(min=1)
    total = torch.gather(mass, 1, kept - 1)
    pick = torch.minimum((mass <= s["u"].double()[:, None] * total).sum(-1, keepdim=True), kept - 1)
    pick, kept = torch.where(greedy, 0, pick), torch.where(greedy, 1, kept)
    prob = torch.where(greedy, 1.0, torch.gather(w, 1, pick) / total)
    return {"token": torch.gather(order, 1, pick)[:, 0].int(), "kept": kept[:, 0].int(), "prob": prob[:, 0].float()}


def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    if op == "rotary":
        return _turn(s["x"], s["pos"], s).to(s["x"].dtype)
    if op == "append":
        return _plain_append(s)
    return _plain_attention(s) if op == "attention" else _plain_sample(s)


# ----------------------------------------------------------------------------- the framework's calls
def _handle(s, op):
    """The cache handle, the rotary and the workspace that a program keeps beside its buffers."""
    from n730_b200 import kv16
    c = s["case"]
    if op != "attention":
        s["turn"] = kv16.Rotary(s["freq"].data_ptr(), c["part"], layout=c["layout"], factor=s["factor"])
    if op != "rotary":
        s["cache"] = kv16.KV16Cache(s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(), n_pages=s["k"].shape[0],
                                    max_pages=s["table"].shape[1], n_kv=c["kv"], head_dim=c["dim"], page_size=c["page"],
                                    dtype="f16" if c["dtype"] == "f16" else "bf16", prefix_table=s["prefix_table"].data_ptr(),
                                    prefix_pages=s["prefix_table"].numel(), prefix_len=s["prefix"].data_ptr())
    if op == "attention":
        need = s["cache"].attention_workspace(c["batch"], c["tokens"], c["heads"])
        s["ws"] = torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda")
    s["ready"] = True


def _own(s, op):
    c = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "sample":
        from n730_b200 import sampling
        sampling.sample_rows(s["x"].data_ptr(), c["dtype"], c["batch"], c["vocab"], s["u"].data_ptr(), s["token"].data_ptr(),
                             temperature=s["temperature"].data_ptr(), top_k=s["top_k"].data_ptr(), top_p=s["top_p"].data_ptr(),
                             min_p=s["min_p"].data_ptr(), prob=s["prob"].data_ptr(), kept=s["kept"].data_ptr(), stream=stream)
        return {"token": s["token"], "kept": s["kept"], "prob": s["prob"]}
    if "ready" not in s:
        _handle(s, op)
    if op == "rotary":
        s["turn"].apply(s["x"].data_ptr(), s["y"].data_ptr(), c["dtype"], c["rows"], c["heads"], c["dim"], s["pos"].data_ptr(),
                        stream=stream)
        return s["y"]
    if op == "append":
        s["cache"].append(s["x_k"].data_ptr(), s["x_v"].data_ptr(), c["dtype"], c["batch"], c["tokens"], s["lens"].data_ptr(),
                          new=s["new"].data_ptr(), rotary=s["turn"], q=s["q"].data_ptr(), q_out=s["out"].data_ptr(),
                          heads=c["heads"], stream=stream)
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    s["cache"].attention(s["q"].data_ptr(), s["out"].data_ptr(), c["batch"], c["tokens"], c["heads"], s["lens"].data_ptr(),
                         new=s["new"].data_ptr(), ws=s["ws"].data_ptr(), ws_bytes=s["ws"].numel(), stream=stream)
    return {"out": s["out"]}


# ----------------------------------------------------------------------------- floors
def work(case):
    """Expected bytes and operations of one pass (ragged lengths by their mean)."""
    op, io = case["op"], BYTES[case["dtype"]]
    if op == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": n * io + 32 * case["batch"], "flops": 4 * n}
    if op == "rotary":
        n = case["rows"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * io + 4 * case["rows"], "flops": 3 * n * case["part"]}
    batch, tokens, ctx, kv, dim, heads = (case[k] for k in ("batch", "tokens", "ctx", "kv", "dim", "heads"))
    new = batch * tokens * (0.5 + 0.5 / tokens if case["ragged"] else 1)
    if op == "append":
        return {"bytes": new * dim * (2 * heads * io + 2 * kv * (io + 2)), "flops": 3 * new * (heads + kv) * case["part"]}
    mean = ctx * (9 / 16 if case["ragged"] else 1)
    return {"bytes": 2 * kv * dim * 2 * (case["prefix"] + batch * mean) + 2 * new * heads * dim * io,
            "flops": 4 * dim * heads * new * (case["prefix"] + max(1.0, mean - tokens / 2 + 0.5))}


# ----------------------------------------------------------------------------- 64 bits
def _exact_turn(x, pos, s):
    """The rotation as a product of complex numbers."""
    c = s["case"]
    part = c["part"]
    x = x.double()
    a = torch.exp(1j * (pos.double()[..., None, None] * s["freq"])) * s["factor"]
    if c["layout"] == "half":
        z = torch.complex(x[..., :part // 2], x[..., part // 2:part]) * a
        head = torch.cat([z.real, z.imag], -1)
    else:
        head = torch.view_as_real(torch.view_as_complex(x[..., :part].unflatten(-1, (-1, 2)).contiguous()) * a).flatten(-2)
    return torch.cat([head, x[..., part:]], -1)


def _exact_append(s):
    c = s["case"]
    q, k, v = s["out"].double(), s["k"].double(), s["v"].double()
    lens, new, table = s["lens"].tolist(), s["new"].tolist(), s["table"].long()
    for b in range(c["batch"]):
        at = lens[b] + torch.arange(new[b], device="cuda")
        q[b, :new[b]] = _exact_turn(s["q"][b, :new[b]], at + c["prefix"], s)
        k[table[b, at // c["page"]], :, at % c["page"]] = _exact_turn(s["x_k"][b, :new[b]], at + c["prefix"], s)
        v[table[b, at // c["page"]], :, at % c["page"]] = s["x_v"][b, :new[b]].double()
    return {"q": q, "k": k, "v": v}


def _exact_attention(s):
    c = s["case"]
    kv, page, dim, prefix = c["kv"], c["page"], c["dim"], c["prefix"]
    group = c["heads"] // kv
    out = s["out"].double()
    lens, new = s["lens"].tolist(), s["new"].tolist()
    p = torch.arange(prefix, device="cuda")
    for h in range(kv):
        first = [x[s["prefix_table"].long()[p // page], h, p % page].double() for x in (s["k"], s["v"])]
        for b in range(c["batch"]):
            at = torch.arange(lens[b] + new[b], device="cuda")
            k, v = (torch.cat([f, x[s["table"][b].long()[at // page], h, at % page].double()])
                    for f, x in zip(first, (s["k"], s["v"])))
            q = s["q"][b, :new[b], h * group:(h + 1) * group].double()
            x = torch.einsum("tgd,nd->gtn", q, k) / dim ** 0.5
            x += torch.triu(torch.full((new[b], k.shape[0]), -float("inf"), dtype=torch.float64, device="cuda"), prefix + lens[b] + 1)
            out[b, :new[b], h * group:(h + 1) * group] = torch.einsum("gtn,nd->tgd", torch.softmax(x, -1), v)
    return {"out": out}


def _exact_sample(s):
    prob = np.ones(s["case"]["batch"])
    x = s["x"].float().cpu().numpy().astype(np.float64)
    t, k, p, m, u = (s[n].cpu().numpy().astype(np.float64) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    for r in range(len(prob)):
        if t[r] <= 0:
            continue
        w = np.sort(np.exp((x[r] - x[r].max()) / t[r]))[::-1]
        w = w[:int(k[r])] if k[r] > 0 else w
        mass = np.cumsum(w)
        n = min(len(w), int(np.searchsorted(mass, p[r] * mass[-1])) + 1) if p[r] < 1 else len(w)
        n = max(1, min(n, int((w >= m[r]).sum())))
        prob[r] = w[min(np.searchsorted(mass[:n], u[r] * mass[n - 1], "right"), n - 1)] / mass[n - 1]
    return {"token": None, "kept": None, "prob": prob}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_turn(s["x"], s["pos"], s)
    if case["op"] == "append":
        return _exact_append(s)
    return _exact_attention(s) if case["op"] == "attention" else _exact_sample(s)
