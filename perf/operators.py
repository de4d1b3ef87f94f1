"""Cases of the chunk-serving operators: rope_and_cache, chunk_attention, verify_draft_tokens.

``run`` computes a case in its plain form (elementary torch operations in 32 bits), or with ``own`` set
by the calls a serving program makes of this package; ``exact`` computes it in 64 bits, on its own.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the smallest prefill chunk: a short follow-up turn of one user
        dict(name="chunk_short", op="chunk", batch=1, q_lo=16, q_hi=16, ctx_lo=400, ctx_hi=400, singles=0, heads=32,
             kv_heads=8, dim=128, block=16, dtype="bf16", int8=False, layout=0, window=0),
        # a whole prompt in one chunk: the largest product
        dict(name="chunk_prompt_8k", op="chunk", batch=1, q_lo=8192, q_hi=8192, ctx_lo=8192, ctx_hi=8192, singles=0,
             heads=32, kv_heads=8, dim=128, block=128, dtype="bf16", int8=False, layout=0, window=0),
        # chunked prefill late in a long prompt
        dict(name="chunk_512_over_32k", op="chunk", batch=1, q_lo=512, q_hi=512, ctx_lo=32768, ctx_hi=32768, singles=0,
             heads=32, kv_heads=8, dim=128, block=64, dtype="fp16", int8=False, layout=1, window=0),
        # a mixed step: most sequences decode one token, a few bring ragged chunks
        dict(name="chunk_mixed", op="chunk", batch=32, q_lo=61, q_hi=256, ctx_lo=300, ctx_hi=4096, singles=27, heads=32,
             kv_heads=8, dim=128, block=32, dtype="bf16", int8=False, layout=0, window=0),
        # single tokens over long contexts
        dict(name="chunk_single_64k", op="chunk", batch=8, q_lo=1, q_hi=1, ctx_lo=20001, ctx_hi=65536, singles=0,
             heads=64, kv_heads=8, dim=128, block=128, dtype="bf16", int8=False, layout=0, window=0),
        # head_dim 64, an odd group of 7, a sliding window
        dict(name="chunk_window_d64", op="chunk", batch=3, q_lo=700, q_hi=1501, ctx_lo=1600, ctx_hi=6001, singles=0,
             heads=56, kv_heads=8, dim=64, block=16, dtype="fp16", int8=False, layout=0, window=1024),
        # chunks over the int8 cache
        dict(name="chunk_int8", op="chunk", batch=4, q_lo=257, q_hi=400, ctx_lo=3000, ctx_hi=8192, singles=0, heads=32,
             kv_heads=8, dim=128, block=128, dtype="bf16", int8=True, layout=0, window=0),
        # a decode step: one new token per sequence
        dict(name="rope_decode", op="rope", tokens=64, heads=32, kv_heads=8, dim=128, rotary=128, block=128,
             dtype="bf16", int8=False, layout=0, interleaved=False, norm=False, fused=True, pad=0.0),
        # a prefill step with norms of queries and keys, rows of a fused projection, some of them padding
        dict(name="rope_prefill_norm", op="rope", tokens=16384, heads=32, kv_heads=8, dim=128, rotary=128, block=128,
             dtype="bf16", int8=False, layout=0, interleaved=False, norm=True, fused=True, pad=0.05),
        # an odd number of rows, neighbouring pairs, half of the head rotated, quantised on the way
        dict(name="rope_int8", op="rope", tokens=4097, heads=32, kv_heads=8, dim=128, rotary=64, block=16,
             dtype="fp16", int8=True, layout=0, interleaved=True, norm=False, fused=False, pad=0.0),
        # one user, a few drafted tokens
        dict(name="verify_one", op="verify", batch=1, drafts=4, vocab=32000, given=True, ragged=False, dtype="fp32"),
        # a full batch over a large vocabulary, ragged numbers of drafts
        dict(name="verify_batch", op="verify", batch=64, drafts=5, vocab=128256, given=True, ragged=True,
             dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "chunk", "rope", "verify"])
    if op == "rope":
        dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        int8 = rng.random() < 0.3
        return dict(op="rope", tokens=_log(rng, 1, 16384), heads=kv_heads * rng.choice([1, 2, 3, 4, 7]),
                    kv_heads=kv_heads, dim=dim, rotary=rng.choice([dim, dim // 2]), block=rng.choice([16, 32, 64, 128]),
                    dtype=rng.choice(["bf16", "fp16"]), int8=int8, layout=0 if int8 else rng.choice([0, 1]),
                    interleaved=rng.random() < 0.5, norm=rng.random() < 0.5, fused=rng.random() < 0.5,
                    pad=rng.choice([0.0, 0.1]))
    if op == "verify":
        batch, drafts, vocab = _log(rng, 1, 64), rng.randint(1, 5), _log(rng, 1000, 128256)
        return dict(op="verify", batch=batch, drafts=drafts, vocab=vocab, given=rng.random() < 0.8,
                    ragged=rng.random() < 0.5, dtype=rng.choice(["fp32", "fp32", "bf16"]))
    dim, kv_heads, group = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8])
    int8 = dim == 128 and rng.random() < 0.25
    q_hi, past, batch = _log(rng, 1, 4096), _log(rng, 1, 32768), _log(rng, 1, 32)
    ctx_hi = q_hi + past
    while batch > 1 and (batch * kv_heads * group * q_hi * ctx_hi > 2 ** 30 or batch * kv_heads * ctx_hi > 2 ** 21):
        batch = (batch + 1) // 2
    while kv_heads * group * q_hi * ctx_hi > 2 ** 30:
        q_hi = (q_hi + 1) // 2
        ctx_hi = q_hi + past
    return dict(op="chunk", batch=batch, q_lo=max(1, q_hi // 3), q_hi=q_hi, ctx_lo=max(1, q_hi // 2), ctx_hi=ctx_hi,
                singles=batch // 2, heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                block=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "fp16"]), int8=int8,
                layout=0 if int8 else rng.choice([0, 1]),
                window=_log(rng, 16, 4096) if rng.random() < 0.25 else 0)


# ---------------------------------------------------------------------------------------------- inputs
def _lens(c):
    """New and cached tokens of every sequence, on the host; the cached ones include the new ones.  A case has
    its lengths whatever the seed, so that its outputs have one shape."""
    g = torch.Generator().manual_seed(c["q_hi"] + c["ctx_hi"])
    b = c["batch"]
    q = torch.randint(c["q_lo"], c["q_hi"] + 1, (b,), generator=g)
    ctx = torch.randint(c["ctx_lo"], c["ctx_hi"] + 1, (b,), generator=g)
    order = torch.randperm(b, generator=g)
    q[order[:c["singles"]]] = 1
    ctx = torch.maximum(ctx, q)
    ctx[order[-1]] = c["ctx_hi"]
    q[order[-1]] = c["q_hi"]
    return q.to(torch.int32), ctx.to(torch.int32)


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _prepare_chunk(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q_lens, ctx = _lens(c)
    bs, kvh, d, dtype = c["block"], c["kv_heads"], c["dim"], DTYPES[c["dtype"]]
    need = (ctx.long() + bs - 1) // bs
    total, width = int(need.sum()), int(need.max())
    blocks = total + max(1, total // 10)
    pool = torch.randperm(blocks, generator=g, device="cuda")[:total].to(torch.int32)
    # the blocks of a sequence stand at the front of its table row, the rest of the row is 0
    need = need.cuda()
    col = torch.arange(width, device="cuda")
    used = col[None, :] < need[:, None]
    tables = torch.zeros(c["batch"], width, dtype=torch.int32, device="cuda")
    tables[used] = pool
    shape = (blocks, kvh, bs, d) if c["layout"] == 1 else (blocks, bs, kvh, d)
    s = dict(case=c, q_lens=q_lens, ctx=ctx, tables=tables, q_lens_dev=q_lens.cuda(), ctx_dev=ctx.cuda(),
             query=_normal(g, (int(q_lens.sum()), c["heads"], d), dtype), scale=1.0 / math.sqrt(d))
    if c["int8"]:
        s["kc"] = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
        s["vc"] = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
        # values of about unit variance: 127 steps of an int8 stand for 1.7 standard deviations
        s["kd"] = 0.01 + 0.007 * torch.rand(kvh * d, generator=g, device="cuda")
        s["vd"] = 0.01 + 0.007 * torch.rand(kvh * d, generator=g, device="cuda")
    else:
        s["kc"], s["vc"] = _normal(g, shape, dtype), _normal(g, shape, dtype)
        s["kd"] = s["vd"] = None
    return s


def _prepare_rope(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, h, kvh, d, dtype = c["tokens"], c["heads"], c["kv_heads"], c["dim"], DTYPES[c["dtype"]]
    if c["fused"]:  # rows of one projection of queries, keys and values
        rows = _normal(g, (t, h + 2 * kvh, d), dtype)
        q, k, v = rows[:, :h], rows[:, h:h + kvh], rows[:, h + kvh:]
    else:
        q, k, v = _normal(g, (t, h, d), dtype), _normal(g, (t, kvh, d), dtype), _normal(g, (t, kvh, d), dtype)
    blocks = (t + t // 8) // c["block"] + 1
    shape = (blocks, kvh, c["block"], d) if c["layout"] == 1 else (blocks, c["block"], kvh, d)
    slots = torch.randperm(blocks * c["block"], generator=g, device="cuda")[:t].to(torch.int32)
    if c["pad"]:  # padding rows of the step: no slot
        slots[torch.rand(t, generator=g, device="cuda") < c["pad"]] = -1
    far = 32768
    positions = torch.randint(0, far, (t,), generator=g, device="cuda", dtype=torch.int32)
    r = c["rotary"]
    inv = 10000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
    ang = torch.arange(far, device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
    s = dict(case=c, q=q, k=k, v=v, slots=slots, positions=positions, eps=1e-6,
             cos_sin=torch.cat([ang.cos(), ang.sin()], dim=1).float())
    if c["int8"]:
        s["kc"] = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
        s["vc"] = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
        s["kd"] = 0.02 + 0.02 * torch.rand(kvh * d, generator=g, device="cuda")
        s["vd"] = 0.02 + 0.02 * torch.rand(kvh * d, generator=g, device="cuda")
    else:
        s["kc"], s["vc"] = _normal(g, shape, dtype), _normal(g, shape, dtype)
        s["kd"] = s["vd"] = None
    s["qw"] = (1 + 0.2 * _normal(g, (d,), torch.float32)).to(dtype) if c["norm"] else None
    s["kw"] = (1 + 0.2 * _normal(g, (d,), torch.float32)).to(dtype) if c["norm"] else None
    return s


def _prepare_verify(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, k, v = c["batch"], c["drafts"], c["vocab"]
    dtype = torch.float32 if c["dtype"] == "fp32" else DTYPES[c["dtype"]]
    # a draft model that is near its target: the same logits and some noise
    logits = 3.0 * torch.randn(b, k + 1, v, generator=g, device="cuda")
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits[:, :k] + 0.7 * torch.randn(b, k, v, generator=g, device="cuda"), -1).to(dtype)
    tokens = torch.multinomial(draft.reshape(b * k, v).float(), 1, generator=g).view(b, k).to(torch.int32)
    lens = torch.full((b,), k, dtype=torch.int32, device="cuda")
    if c["ragged"]:
        lens = torch.randint(0, k + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    return dict(case=c, target=target, draft=draft if c["given"] else None, tokens=tokens, lens=lens,
                uniform=torch.rand(b, k + 1, generator=g, device="cuda"))


def prepare(case, seed):
    return {"chunk": _prepare_chunk, "rope": _prepare_rope, "verify": _prepare_verify}[case["op"]](case, seed)


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_chunk(s):
    c = s["case"]
    bs, kvh, d = c["block"], c["kv_heads"], c["dim"]
    b, grp = c["batch"], c["heads"] // kvh
    max_q, max_ctx = int(s["q_lens"].max()), int(s["ctx"].max())
    q_lens, ctx = s["q_lens_dev"].long(), s["ctx_dev"].long()
    dev = s["query"].device
    # the rows of every sequence, padded to the longest
    j = torch.arange(max_ctx, device=dev)
    block = s["tables"].long()[:, :(max_ctx + bs - 1) // bs].repeat_interleave(bs, 1)[:, :max_ctx]
    if c["layout"] == 1:
        keys, values = s["kc"][block, :, j % bs], s["vc"][block, :, j % bs]
    else:
        keys, values = s["kc"][block, j % bs], s["vc"][block, j % bs]
    keys, values = keys.float(), values.float()
    if c["int8"]:
        keys, values = keys * s["kd"].view(kvh, d), values * s["vd"].view(kvh, d)
    first = torch.cumsum(q_lens, 0) - q_lens
    i = torch.arange(max_q, device=dev)
    live = i[None, :] < q_lens[:, None]
    row = (first[:, None] + i[None, :])[live]
    q = torch.zeros(b, max_q, c["heads"], d, device=dev)
    q[live] = s["query"].float()[row]
    q = q.view(b, max_q, kvh, grp, d).permute(0, 2, 3, 1, 4).reshape(b, kvh, grp * max_q, d)
    score = torch.matmul(q, keys.permute(0, 2, 3, 1)).mul_(s["scale"]).view(b, kvh, grp, max_q, max_ctx)
    pos = (ctx - q_lens)[:, None] + i[None, :]
    seen = j[None, None, :] <= pos[:, :, None]
    if c["window"]:
        seen &= j[None, None, :] > pos[:, :, None] - c["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, kvh, grp * max_q, max_ctx), values.permute(0, 2, 1, 3))
    out = out.view(b, kvh, grp, max_q, d) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, max_q, c["heads"], d)
    return out[live].to(s["query"].dtype)


def _turn(x, cos, sin, rotary, interleaved):
    a, b = (x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved else (x[..., :rotary // 2], x[..., rotary // 2:rotary])
    cos, sin = cos[:, None], sin[:, None]
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([r, x[..., rotary:]], -1)


def _stored(s):
    """The caches as the values they stand for, in the model's type."""
    if s["kd"] is None:
        return s["kc"], s["vc"]
    shape, dtype = (s["case"]["kv_heads"], s["case"]["dim"]), s["q"].dtype
    return (s["kc"] * s["kd"].view(shape)).to(dtype), (s["vc"] * s["vd"].view(shape)).to(dtype)


def _plain_rope(s):
    c = s["case"]
    r, bs = c["rotary"], c["block"]
    table = s["cos_sin"][s["positions"].long()]
    cos, sin = table[:, :r // 2], table[:, r // 2:]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + s["eps"]) * s["qw"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + s["eps"]) * s["kw"].float()
    q, k = _turn(q, cos, sin, r, c["interleaved"]), _turn(k, cos, sin, r, c["interleaved"])
    live = s["slots"] >= 0
    slots = s["slots"][live].long()
    k, v = k[live], v[live]
    if c["int8"]:
        shape = (c["kv_heads"], c["dim"])
        k = torch.clamp(torch.round(k / s["kd"].view(shape)), -128, 127)
        v = torch.clamp(torch.round(v / s["vd"].view(shape)), -128, 127)
    k, v = k.to(s["kc"].dtype), v.to(s["vc"].dtype)
    if c["layout"] == 1:
        s["kc"][slots // bs, :, slots % bs] = k
        s["vc"][slots // bs, :, slots % bs] = v
    else:
        s["kc"][slots // bs, slots % bs] = k
        s["vc"][slots // bs, slots % bs] = v
    return (q.to(s["q"].dtype), *_stored(s))


def _plain_verify(s):
    c = s["case"]
    b, k = c["batch"], c["drafts"]
    rows, lens = torch.arange(b, device="cuda"), s["lens"].long()
    i = torch.arange(k, device="cuda")
    tok = s["tokens"].long()[:, :, None]
    p = s["target"][:, :k].gather(2, tok)[..., 0].double()
    q = s["draft"].gather(2, tok)[..., 0].double() if c["given"] else torch.ones_like(p)
    ok = (s["uniform"][:, :k].double() * q < p) & (i[None, :] < lens[:, None])
    taken = torch.cumprod(ok.long(), 1).sum(1)
    row = s["target"][rows, taken].double()
    at = torch.clamp(taken, max=k - 1)
    if c["given"]:
        less = s["draft"][rows, at].double()
    else:
        less = torch.zeros_like(row).scatter_(1, s["tokens"].long()[rows, at][:, None], 1.0)
    rest = torch.where((taken < lens)[:, None], torch.clamp(row - less, min=0.0), row)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, row)
    run_sum = torch.cumsum(rest, 1)
    over = run_sum > s["uniform"][:, k:].double() * run_sum[:, -1:]
    last = torch.argmax(over.to(torch.int8), 1)
    out = torch.where(i[None, :] < taken[:, None], s["tokens"].long(), -1)
    out = torch.cat([out, torch.full_like(out[:, :1], -1)], 1).scatter_(1, taken[:, None], last[:, None])
    return out.to(torch.int32), taken.to(torch.int32)


def run(state):
    c = state["case"]
    if own:
        import ms_custom_ops_b200 as ops
        if c["op"] == "chunk":
            return ops.chunk_attention(state["query"], state["kc"], state["vc"], state["tables"], state["q_lens"],
                                       state["ctx"], qk_scale=state["scale"], window_size=c["window"],
                                       input_layout=c["layout"], k_descale=state["kd"], v_descale=state["vd"])
        if c["op"] == "rope":
            q = ops.rope_and_cache(state["q"], state["k"], state["v"], state["kc"], state["vc"], state["slots"],
                                   state["positions"], state["cos_sin"], q_weight=state["qw"], k_weight=state["kw"],
                                   eps=state["eps"], interleaved=c["interleaved"], input_layout=c["layout"],
                                   k_descale=state["kd"], v_descale=state["vd"])
            return (q, *_stored(state))
        return ops.verify_draft_tokens(state["target"], state["draft"], state["tokens"], state["uniform"],
                                       draft_lens=state["lens"])
    return {"chunk": _plain_chunk, "rope": _plain_rope, "verify": _plain_verify}[c["op"]](state)


# ---------------------------------------------------------------------------------------------- what a pass needs
def _pairs(q, ctx, window):
    """(query, key) pairs of one sequence that the causal mask and the window leave."""
    lo, hi = ctx - q + 1, ctx  # keys that the first and the last query see without a window
    if not window or hi <= window:
        return (lo + hi) * q // 2
    if lo >= window:
        return window * q
    return (lo + window - 1) * (window - lo) // 2 + window * (hi - window + 1)


def work(case):
    c = case
    if c["op"] == "chunk":
        d, h, kvh = c["dim"], c["heads"], c["kv_heads"]
        seqs = list(zip(*(v.tolist() for v in _lens(c))))
        pairs = sum(_pairs(a, b, c["window"]) for a, b in seqs)
        keys = sum(min(b, a + c["window"] - 1) if c["window"] else b for a, b in seqs)
        tokens = sum(a for a, b in seqs)
        return {"bytes": keys * kvh * d * 2 * (1 if c["int8"] else 2) + tokens * h * d * 4, "flops": 4 * d * h * pairs}
    if c["op"] == "rope":
        t, d, h, kvh = c["tokens"], c["dim"], c["heads"], c["kv_heads"]
        wrote = t * (1 - c["pad"]) * 2 * kvh * d * (1 if c["int8"] else 2)
        return {"bytes": t * (h + 2 * kvh) * d * 2 + t * h * d * 2 + wrote + t * (c["rotary"] * 4 + 8),
                "flops": t * (h + kvh) * d * (8 if c["norm"] else 4)}
    size = 4 if c["dtype"] == "fp32" else 2
    # a row of the target, and the draft's where one of its tokens is turned down (about one in four is)
    turned = 1 - 0.75 ** (c["drafts"] / 2 if c["ragged"] else c["drafts"])
    rows = c["batch"] * (1 + (turned if c["given"] else 0))
    return {"bytes": rows * c["vocab"] * size + c["batch"] * c["drafts"] * 20, "flops": 3 * rows * c["vocab"]}


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_chunk(s):
    c = s["case"]
    bs, kvh, grp, d = c["block"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, (ql, cl) in enumerate(zip(s["q_lens"].tolist(), s["ctx"].tolist())):
        ids = s["tables"][b, :(cl + bs - 1) // bs].long()
        for h in range(kvh):
            if c["layout"] == 1:
                k, v = s["kc"][ids, h], s["vc"][ids, h]
            else:
                k, v = s["kc"][ids][:, :, h], s["vc"][ids][:, :, h]
            k, v = k.reshape(-1, d)[:cl].double(), v.reshape(-1, d)[:cl].double()
            if c["int8"]:
                k, v = k * s["kd"][h * d:(h + 1) * d].double(), v * s["vd"][h * d:(h + 1) * d].double()
            key_at = torch.arange(cl, device="cuda")
            for lo in range(0, ql, 2048):
                n = min(2048, ql - lo)
                here = torch.arange(cl - ql + lo, cl - ql + lo + n, device="cuda")
                hide = key_at[None, :] > here[:, None]
                if c["window"]:
                    hide |= key_at[None, :] + c["window"] <= here[:, None]
                q = s["query"][at + lo:at + lo + n, h * grp:(h + 1) * grp].double()
                x = torch.einsum("nge,ce->gnc", q, k) * s["scale"]
                x = torch.softmax(x.masked_fill(hide[None], -math.inf), -1)
                out[at + lo:at + lo + n, h * grp:(h + 1) * grp] = torch.einsum("gnc,ce->nge", x, v)
        at += ql
    return out


def _exact_rope(s):
    c = s["case"]
    d, r, bs = c["dim"], c["rotary"], c["block"]
    table = s["cos_sin"].double()[s["positions"].long()]
    # the rotation as complex numbers
    turn = torch.complex(table[:, :r // 2], table[:, r // 2:])[:, None, :]
    first = torch.arange(r // 2, device="cuda") * (2 if c["interleaved"] else 1)
    second = first + (1 if c["interleaved"] else r // 2)

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + s["eps"]) * w.double()
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        x = x.clone()
        x[..., first], x[..., second] = z.real, z.imag
        return x

    q, k, v = turned(s["q"], s["qw"]), turned(s["k"], s["kw"]), s["v"].double()
    shape = (c["kv_heads"], d)
    kc, vc = s["kc"].double(), s["vc"].double()
    if c["int8"]:
        kd, vd = s["kd"].double().view(shape), s["vd"].double().view(shape)
        k, v = (k / kd).round().clamp(-128, 127) * kd, (v / vd).round().clamp(-128, 127) * vd
        kc, vc = kc * kd, vc * vd
    if c["layout"] == 1:
        kc, vc = kc.transpose(1, 2).contiguous(), vc.transpose(1, 2).contiguous()
    kept = torch.nonzero(s["slots"] >= 0)[:, 0]
    where = s["slots"][kept].long()
    kc.view(-1, *shape).index_copy_(0, where, k[kept])
    vc.view(-1, *shape).index_copy_(0, where, v[kept])
    if c["layout"] == 1:
        kc, vc = kc.transpose(1, 2).contiguous(), vc.transpose(1, 2).contiguous()
    return q, kc, vc


def _exact_verify(s):
    c = s["case"]
    k = c["drafts"]
    tokens, lens, u = s["tokens"].tolist(), s["lens"].tolist(), s["uniform"].double().tolist()
    out, count = [], []
    for b in range(c["batch"]):
        n = 0
        while n < lens[b]:
            t = tokens[b][n]
            q = float(s["draft"][b, n, t]) if c["given"] else 1.0
            if not u[b][n] * q < float(s["target"][b, n, t]):
                break
            n += 1
        weights = s["target"][b, n].double()
        if n < lens[b]:
            less = weights.clone()
            if c["given"]:
                less -= s["draft"][b, n].double()
            else:
                less[tokens[b][n]] = 0.0
            less = torch.relu(less)
            weights = less if float(less.sum()) > 0 else weights
        total = torch.cumsum(weights, 0)
        t = int(torch.searchsorted(total, u[b][k] * total[-1], right=True))
        out.append(tokens[b][:n] + [t] + [-1] * (k - n))
        count.append(n)
    return torch.tensor(out, dtype=torch.int32), torch.tensor(count, dtype=torch.int32)


def exact(case, seed):
    return {"chunk": _exact_chunk, "rope": _exact_rope, "verify": _exact_verify}[case["op"]](prepare(case, seed))
