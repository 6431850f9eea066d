"""The sequence operators as measured cases: a bucketed relative-position bias, the attention that reads it, and the norms around a block.

``run`` computes each operator in its plain form (torch products, sums and exponentials in 32 bits, rounded once at the end) or, where ``own``
is true, through ``cellvit_amd.seqops``.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}


# ---------------------------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------------------------
def _bias(name, dtype, heads, q_len, k_len, buckets, span, both, batch):
    return {"name": name, "op": "bias", "dtype": dtype, "heads": heads, "q_len": q_len, "k_len": k_len, "buckets": buckets, "span": span,
            "both": both, "batch": batch}


def _attn(name, mode, dtype, seqs, q_len, k_len, heads, kv_heads, dim, causal, ragged, buckets, span):
    return {"name": name, "op": "attn", "mode": mode, "dtype": dtype, "seqs": seqs, "q_len": q_len, "k_len": k_len, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "causal": causal, "ragged": ragged, "buckets": buckets, "span": span}


def _norm(name, train, dtype, rows, cols, kind, post, gate, alpha):
    return {"name": name, "op": "norm", "train": train, "dtype": dtype, "rows": rows, "cols": cols, "kind": kind, "post": post, "gate": gate,
            "alpha": alpha}


def listed():
    return [
        # the bias plane of one short tile sequence with a class token (256-pixel tile: 16 x 16 + 1 tokens, six heads): latency counts
        _bias("bias_small", "f16", 6, 257, 257, 32, 128, True, 0),
        # a decoder's bias plane shared by its layers and the gradient summed over a batch, 1024-pixel tiles: 4096 tokens, odd key count
        _bias("bias_train", "bf16", 16, 2048, 4097, 32, 128, False, 2),
        # one new token a sequence against a short context: the smallest call
        _attn("token_small", "token", "f16", 4, 1, 257, 6, 6, 64, True, False, 32, 128),
        # one new token a sequence against long ragged contexts, four query heads to a key head
        _attn("token_long", "token", "bf16", 16, 1, 32768, 16, 4, 128, True, True, 32, 128),
        # the tokens of 256-pixel tiles through a six-head layer
        _attn("tiles_small", "forward", "f16", 16, 257, 257, 6, 6, 64, False, False, 32, 128),
        # 1024-pixel tiles, sixteen heads of 80 (the widest encoder's geometry)
        _attn("tiles_large", "forward", "f16", 8, 4096, 4096, 16, 16, 80, False, False, 32, 128),
        # cell tokens of a slide region, ragged numbers of cells a tile, packed rows, training step
        _attn("cells_train", "train", "bf16", 24, 1500, 1500, 12, 12, 64, False, True, 32, 128),
        # causal decoder training on long sequences, shared key heads, buckets that reach far
        _attn("causal_train", "train", "f16", 2, 4096, 4096, 16, 8, 128, True, False, 64, 2048),
        # the parity engine's type
        _attn("parity_train", "train", "f32", 2, 577, 577, 6, 6, 64, False, False, 32, 128),
        # one short tile's tokens between two blocks: latency
        _norm("norm_small", False, "f16", 257, 384, "layer", True, "column", 1.0),
        # eight 1024-pixel tiles between two blocks of the widest encoder
        _norm("norm_large", False, "f16", 65536, 1280, "layer", True, "column", 1.0),
        # training with a gate a tile and a residual scale, rms norms
        _norm("norm_train", True, "bf16", 32784, 1280, "rms", True, "tile", 0.75),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    op = rng.choice(["bias", "attn", "attn", "attn", "norm"])
    dtype = rng.choice(["f16", "f16", "bf16", "bf16", "f32"])
    buckets, span = rng.choice([(32, 128), (16, 64), (64, 500), (32, 1024), (128, 2048)])
    if op == "bias":
        q, k = _log(rng, 1, 2048), _log(rng, 1, 4096)
        return _bias("", dtype, rng.randint(1, 16), q, k, buckets, span, rng.random() < 0.5, rng.choice([0, 1, 2]))
    if op == "attn":
        mode = rng.choice(["forward", "train", "token"])
        kv = rng.choice([1, 2, 4, 6, 8])
        heads, dim = kv * rng.choice([1, 1, 2, 4]), rng.choice([32, 64, 64, 72, 80, 96, 128])
        if mode == "token":
            seqs, k = rng.randint(1, 16), _log(rng, 1, 32768)
            q = min(k, rng.choice([1, 1, 1, 2, 5]))
        else:
            k = _log(rng, 17, 4096 if dtype != "f32" else 1024)
            q = k if rng.random() < 0.8 else rng.randint(1, k)
            seqs = rng.randint(1, max(1, min(24, (2 * 4096 * 4096) // (k * k * max(1, heads // 8)))))
        return _attn("", mode, dtype, seqs, q, k, heads, kv, dim, mode == "token" or rng.random() < 0.5, rng.random() < 0.5, buckets, span)
    cols = rng.choice([384, 768, 1024, 1280, 2048, 100, 250, 999, 4096])
    return _norm("", rng.random() < 0.5, dtype, min(_log(rng, 1, 65536), 80_000_000 // cols), cols, rng.choice(["layer", "rms"]), rng.random() < 0.7,
                 rng.choice(["none", "column", "tile"]), rng.choice([1.0, 0.75, 2.0]))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _lengths(case):
    """(query lengths, key lengths) a sequence; ragged ones are fixed by the case: some short, one empty, the first full."""
    n, q, k = case["seqs"], case["q_len"], case["k_len"]
    if not case["ragged"]:
        return [q] * n, [k] * n
    ks = [k if s == 0 else 0 if s == 3 else 1 + (s * 2654435761 + 12345) % 4294967296 * k // 4294967296 for s in range(n)]
    return [min(q, x) for x in ks], ks


def _pairs(case):
    """Visible (query, key) pairs of one head."""
    total = 0
    for q, k in zip(*_lengths(case)):
        total += q * k - q * (q - 1) // 2 if case["causal"] else q * k
    return total


def work(case):
    es = BYTES[case["dtype"]]
    if case["op"] == "bias":
        n = case["heads"] * case["q_len"] * case["k_len"]
        return {"bytes": n * es * (1 + case["batch"]), "flops": n * case["batch"]}
    if case["op"] == "attn":
        qs, ks = _lengths(case)
        h, g, d = case["heads"], case["kv_heads"], case["dim"]
        rows_q, rows_k, pairs = sum(qs) * h * d, sum(ks) * g * d, _pairs(case)
        if case["mode"] == "train":
            return {"bytes": es * (4 * rows_q + 4 * rows_k), "flops": 14 * pairs * h * d}
        return {"bytes": es * (2 * rows_q + 2 * rows_k), "flops": 4 * pairs * h * d}
    n = case["rows"] * case["cols"]
    if case["train"]:
        return {"bytes": n * (16 + 4 * es), "flops": 40 * n}
    return {"bytes": n * (8 + 2 * es), "flops": 14 * n}


# ---------------------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------------------
def _map(buckets, span, both):
    """Bucket of every offset -span .. span (key minus query position): half of the buckets of a side exact, the others spaced by the logarithm
    up to `span`; integers only, so that no border depends on a rounding."""
    side = buckets // 2 if both else buckets
    exact_n = side // 2
    steps = side - exact_n

    def near(n):
        if n < exact_n:
            return n
        k = 0
        while k + 1 < steps and span ** (k + 1) * exact_n ** (steps - k - 1) <= n ** steps:
            k += 1
        return exact_n + k

    return [(side + near(o) if o > 0 else near(-o)) if both else near(max(-o, 0)) for o in range(-span, span + 1)]


def _gate_rows(case):
    return 1 if case["gate"] == "column" else -(-case["rows"] // _tile_rows(case))


def _tile_rows(case):
    return 4096 if case["rows"] >= 8192 else 17


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def rand(*shape, dtype=dt, by=1.0, plus=0.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * by + plus).to(dtype)

    st = {"case": dict(case)}
    if case["op"] in ("bias", "attn"):
        st["table"] = rand(case["buckets"], case["heads"], dtype=torch.float32)
        both = case["both"] if case["op"] == "bias" else not case["causal"]
        st["map"] = torch.tensor(_map(case["buckets"], case["span"], both), dtype=torch.int32, device="cuda")
    if case["op"] == "bias":
        if case["batch"]:
            st["dbias"] = rand(case["batch"], case["heads"], case["q_len"], case["k_len"])
        return st
    if case["op"] == "attn":
        qs, ks = _lengths(case)
        h, n, d = case["heads"], case["kv_heads"], case["dim"]
        if case["ragged"]:
            st["q"], st["k"], st["v"] = rand(sum(qs), h, d), rand(sum(ks), n, d), rand(sum(ks), n, d)
            for name, lens in (("q_off", qs), ("k_off", ks)):
                st[name] = torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
        else:
            s = case["seqs"]
            st["q"], st["k"], st["v"] = rand(s, qs[0], h, d), rand(s, ks[0], n, d), rand(s, ks[0], n, d)
        if case["mode"] == "train":
            st["dout"] = rand(*st["q"].shape)
        return st
    m, c = case["rows"], case["cols"]
    st["x"] = rand(m, c, dtype=torch.float32, by=2.0, plus=0.25)
    st["y"] = rand(m, c, plus=0.1)
    if case["post"]:
        st["post_w"] = rand(c, dtype=torch.float32, by=0.2, plus=1.0)
        if case["kind"] == "layer":
            st["post_b"] = rand(c, dtype=torch.float32, by=0.1)
    st["pre_w"] = rand(c, dtype=torch.float32, by=0.2, plus=1.0)
    if case["kind"] == "layer":
        st["pre_b"] = rand(c, dtype=torch.float32, by=0.1)
    if case["gate"] != "none":
        st["gate"] = rand(_gate_rows(case), c, dtype=torch.float32, by=0.3, plus=0.5)
    if case["train"]:
        st["dx_out"], st["dz"] = rand(m, c, dtype=torch.float32), rand(m, c)
    return st


# ---------------------------------------------------------------------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------------------------------------------------------------------
def run(st):
    return {"bias": _run_bias, "attn": _run_attn, "norm": _run_norm}[st["case"]["op"]](st)


def _offset_index(st, q_len, k_len, shift):
    """Row of the table for every (query, key) pair of padded sequences: [.., q, k]; `shift` [..] is the first query's position."""
    span = st["case"]["span"]
    at = torch.arange(k_len, device="cuda") - torch.arange(q_len, device="cuda")[:, None] - shift[..., None, None]
    return st["map"].long()[at.clamp(-span, span) + span]


def _run_bias(st):
    c = st["case"]
    if own:
        from cellvit_amd import seqops
        out = {"bias": seqops.rel_bias(st["table"], st["map"], c["q_len"], c["k_len"], dtype=TYPES[c["dtype"]])}
        if c["batch"]:
            out["dtable"] = seqops.rel_bias_grad(st["dbias"], st["map"], c["buckets"])
        return out
    shift = torch.full((1,), c["k_len"] - c["q_len"], device="cuda")
    which = _offset_index(st, c["q_len"], c["k_len"], shift)[0]
    out = {"bias": st["table"].t()[:, which].to(TYPES[c["dtype"]])}
    if c["batch"]:
        out["dtable"] = _by_bucket(st, st["dbias"].float().sum(0, keepdim=True), shift)
    return out


def _by_bucket(st, d, shift):
    """Sums over the pairs of a bucket, [buckets, heads], of d [seqs, heads, q, k]: along the diagonals first (all their pairs share an offset), in
    64 bits, since these sums are long."""
    c = st["case"]
    n, h, q, k = d.shape
    # rows last to first, q zeros behind each; read again in rows one shorter, column q - 1 - i + j holds the offset j - i
    d = torch.nn.functional.pad(d.flip(2), (0, q)).reshape(n, h, q * (q + k))[..., : q * (q + k - 1)].reshape(n, h, q, q + k - 1)
    d = d.sum(2, dtype=torch.float64)
    span = c["span"]
    at = torch.arange(q + k - 1, device="cuda") - (q - 1) - shift[:, None]
    which = st["map"].long()[at.clamp(-span, span) + span].reshape(-1)
    total = torch.zeros(c["buckets"], h, device="cuda", dtype=torch.float64)
    return total.index_add_(0, which, d.transpose(1, 2).reshape(-1, h)).float()


def _pad(x, off, most):
    """Packed rows [T, h, d] -> [seqs, most, h, d] in 32 bits and a truth value for every place; dense rows pass."""
    if off is None:
        return x.float(), torch.ones(x.shape[:2], dtype=torch.bool, device="cuda")
    at = off[:-1, None].long() + torch.arange(most, device="cuda")
    valid = at < off[1:, None]
    rows = x.float()[at.clamp(max=max(0, x.shape[0] - 1))]
    return rows * valid[..., None, None], valid


def _unpad(x, off, rows):
    """[seqs, most, ..] -> packed rows [T, ..]."""
    if off is None:
        return x
    t = torch.arange(rows, device="cuda", dtype=torch.int32)
    s = torch.searchsorted(off, t, right=True) - 1
    return x[s, (t - off[s]).long()]


def _run_attn(st):
    c = st["case"]
    q_off, k_off, dt = st.get("q_off"), st.get("k_off"), TYPES[c["dtype"]]
    scale = c["dim"] ** -0.5
    if own:
        from cellvit_amd import seqops
        kw = dict(scale=scale, causal=c["causal"], q_offsets=q_off, k_offsets=k_off, max_q=c["q_len"], max_k=c["k_len"])
        if c["mode"] != "train":
            return {"out": seqops.rel_attention(st["q"], st["k"], st["v"], st["table"], st["map"], **kw)}
        out, saved = seqops.rel_attention_train(st["q"], st["k"], st["v"], st["table"], st["map"], **kw)
        dq, dk, dv, dtable = seqops.rel_attention_grad(saved, st["dout"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}
    h, n, d = c["heads"], c["kv_heads"], c["dim"]
    q, vq = _pad(st["q"], q_off, c["q_len"])
    k, vk = _pad(st["k"], k_off, c["k_len"])
    v, _ = _pad(st["v"], k_off, c["k_len"])
    heads = lambda x: x.transpose(1, 2)  # noqa: E731  [s, h, len, d]
    spread = lambda x: heads(x).repeat_interleave(h // n, 1)  # noqa: E731
    q, k, v = heads(q), spread(k), spread(v)
    shift = vk.sum(1) - vq.sum(1)
    which = _offset_index(st, c["q_len"], c["k_len"], shift)                    # [s, q, k]
    hide = ~vk[:, None, :]
    if c["causal"]:
        at = torch.arange(c["k_len"], device="cuda") - torch.arange(c["q_len"], device="cuda")[:, None] - shift[:, None, None]
        hide = hide | (at > 0)
    hide = hide[:, None]
    s = q @ k.transpose(2, 3).contiguous() * scale + st["table"].t()[:, which].transpose(0, 1)
    s = s.masked_fill(hide, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = p @ v
    rows = st["q"].shape[0]
    out = {"out": _unpad(o.transpose(1, 2), q_off, rows).to(dt)}
    if c["mode"] != "train":
        return out
    do = heads(_pad(st["dout"], q_off, c["q_len"])[0])
    dv = p.transpose(2, 3).contiguous() @ do
    dp = do @ v.transpose(2, 3).contiguous()
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    dq = ds @ k * scale
    dk = ds.transpose(2, 3).contiguous() @ q * scale
    gather = lambda x: x.reshape(x.shape[0], n, h // n, *x.shape[2:]).sum(2).transpose(1, 2)  # noqa: E731
    krows = st["k"].shape[0]
    out["dq"] = _unpad(dq.transpose(1, 2), q_off, rows).to(dt)
    out["dk"], out["dv"] = (_unpad(gather(x), k_off, krows).to(dt) for x in (dk, dv))
    out["dtable"] = _by_bucket(st, ds, shift)
    return out


def _normed(x, kind, w, b):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    hat = x * r
    out = hat * w
    return (out if b is None else out + b), hat, r


def _normed_grad(d, hat, r, kind, w):
    """Gradient of a norm's input and the column sums of its weight and bias."""
    dw, db = (d * hat).sum(0), d.sum(0)
    d = d * w
    d = d - hat * (d * hat).mean(-1, keepdim=True) - (d.mean(-1, keepdim=True) if kind == "layer" else 0.0)
    return d * r, dw, db


def _run_norm(st):
    c, dt = st["case"], TYPES[st["case"]["dtype"]]
    per = _tile_rows(c) if c["gate"] == "tile" else 0
    if own:
        from cellvit_amd import seqops
        post = (st["post_w"], st.get("post_b")) if c["post"] else None
        kw = dict(post=post, pre=(st["pre_w"], st.get("pre_b")), gate=st.get("gate"), rows_per_gate=per or None, alpha=c["alpha"], kind=c["kind"], eps=1e-6)
        if not c["train"]:
            x, z = seqops.block_norm(st["x"], st["y"], **kw)
            return {"x": x, "z": z}
        x, z, saved = seqops.block_norm_train(st["x"], st["y"], **kw)
        grads = seqops.block_norm_grad(saved, st["dx_out"], st["dz"])
        return {"x": x, "z": z, **{k: v for k, v in grads.items() if v is not None}}
    y = st["y"].float()
    if c["post"]:
        u, hat_y, r_y = _normed(y, c["kind"], st["post_w"], st.get("post_b"))
    else:
        u = y
    gate = st.get("gate")
    if gate is not None:
        gate = gate[0] if not per else gate.repeat_interleave(per, 0)[: c["rows"]]
    x = c["alpha"] * st["x"] + (u if gate is None else gate * u)
    z, hat_x, r_x = _normed(x, c["kind"], st["pre_w"], st.get("pre_b"))
    out = {"x": x, "z": z.to(dt)}
    if not c["train"]:
        return out
    d, out["pre_w"], db = _normed_grad(st["dz"].float(), hat_x, r_x, c["kind"], st["pre_w"])
    if c["kind"] == "layer":
        out["pre_b"] = db
    d = d + st["dx_out"]
    out["dx"] = c["alpha"] * d
    du = d if gate is None else d * gate
    if gate is not None:
        dg = d * u
        if per:
            most = _gate_rows(c)
            dg = torch.nn.functional.pad(dg, (0, 0, 0, most * per - c["rows"])).reshape(most, per, -1).sum(1)
        else:
            dg = dg.sum(0, keepdim=True)
        out["gate"] = dg
    if c["post"]:
        dy, out["post_w"], db = _normed_grad(du, hat_y, r_y, c["kind"], st["post_w"])
        if c["kind"] == "layer":
            out["post_b"] = db
    else:
        dy = du
    out["dy"] = dy.to(dt)
    return out


# ---------------------------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    return {"bias": _exact_bias, "attn": _exact_attn, "norm": _exact_norm}[case["op"]](prepare(case, seed), case)


def _which(st, q_len, k_len):
    """Table rows of the pairs of one sequence, [q_len, k_len]."""
    span = (st["map"].numel() - 1) // 2
    position = torch.arange(k_len - q_len, k_len, device="cuda").unsqueeze(1)
    away = torch.arange(k_len, device="cuda").unsqueeze(0) - position
    return st["map"].long().index_select(0, (away.sign() * away.abs().clamp(max=span) + span).reshape(-1)).reshape(q_len, k_len)


def _exact_bias(st, case):
    which = _which(st, case["q_len"], case["k_len"])
    t = st["table"].double()
    out = {"bias": torch.stack([t[:, h][which] for h in range(case["heads"])])}
    if case["batch"]:
        d = torch.zeros(case["buckets"], case["heads"], dtype=torch.float64, device="cuda")
        for h in range(case["heads"]):
            plane = st["dbias"][:, h].double().sum(0)
            for b in range(case["buckets"]):
                d[b, h] = plane[which == b].sum()
        out["dtable"] = d
    return out


def _exact_attn(st, case):
    train = case["mode"] == "train"
    qs, ks = _lengths(case)
    h, n = case["heads"], case["kv_heads"]
    q, k, v = (st[x].double().reshape(-1, *st[x].shape[-2:]) for x in ("q", "k", "v"))
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dtable = torch.zeros_like(st["table"], dtype=torch.float64)
    do = st["dout"].double().reshape(q.shape) if train else None
    a = b = 0
    for lq, lk in zip(qs, ks):
        if lq and lk:
            which = _which(st, lq, lk)
            seen = None
            if case["causal"]:
                seen = torch.arange(lk, device="cuda")[None, :] <= torch.arange(lq, device="cuda")[:, None] + (lk - lq)
            for i in range(h):
                m = i // (h // n)
                qi, ki, vi, ti = q[a:a + lq, i], k[b:b + lk, m], v[b:b + lk, m], st["table"][:, i].double()
                if train:
                    qi, ki, vi = (x.clone().requires_grad_(True) for x in (qi, ki, vi))
                with torch.set_grad_enabled(train):
                    s = torch.matmul(qi, ki.t().contiguous()) / math.sqrt(case["dim"]) + ti[which]
                    if seen is not None:
                        s = s.where(seen, torch.full_like(s, -1e300))
                    w = torch.softmax(s, -1)
                    o = torch.matmul(w, vi)
                out[a:a + lq, i] = o.detach()
                if train:
                    g = torch.autograd.grad(o, (qi, ki, vi, s), do[a:a + lq, i])
                    dq[a:a + lq, i] = g[0]
                    dk[b:b + lk, m] += g[1]
                    dv[b:b + lk, m] += g[2]
                    for bucket in range(case["buckets"]):
                        dtable[bucket, i] += (g[3] * (which == bucket)).sum()
        a, b = a + lq, b + lk
    shaped = {"out": out.reshape(st["q"].shape)}
    if train:
        shaped |= {"dq": dq.reshape(st["q"].shape), "dk": dk.reshape(st["k"].shape), "dv": dv.reshape(st["v"].shape), "dtable": dtable}
    return shaped


def _exact_norm(st, case):
    names = ["x", "y", "post_w", "post_b", "gate", "pre_w", "pre_b"]
    p = {k: st[k].double().requires_grad_(case["train"]) for k in names if k in st}

    def norm(t, w, b):
        mean = t.mean(-1, keepdim=True) if case["kind"] == "layer" else 0.0
        var = ((t - mean) ** 2).mean(-1, keepdim=True)
        t = (t - mean) / torch.sqrt(var + 1e-6) * w
        return t if b is None else t + b

    with torch.set_grad_enabled(case["train"]):
        u = norm(p["y"], p["post_w"], p.get("post_b")) if case["post"] else p["y"]
        if "gate" in p:
            rows = torch.arange(case["rows"], device="cuda") // (_tile_rows(case) if case["gate"] == "tile" else case["rows"])
            u = p["gate"].index_select(0, rows) * u
        x = case["alpha"] * p["x"] + u
        z = norm(x, p["pre_w"], p.get("pre_b"))
    out = {"x": x.detach(), "z": z.detach()}
    if case["train"]:
        keys = list(p)
        g = torch.autograd.grad([x, z], [p[k] for k in keys], [st["dx_out"].double(), st["dz"].double()])
        out |= {{"x": "dx", "y": "dy"}.get(k, k): t for k, t in zip(keys, g)}
    return out
