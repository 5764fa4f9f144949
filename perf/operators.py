"""The cases by which the 8-bit key/value cache and windowed attention are measured, with their plain forms.

Three operators over the paged key/value pools of this package, as they follow one another in a serving loop:

  append   the position rotation of Q and K, and the append of K and V to pools that hold 8 bits an element
           (e4m3) and one power-of-two scale for each (block of tokens, KV head)
  decode   attention of one query token per sequence over such pools, or over half-precision ones, optionally
           through a sliding window behind a few first tokens that stay visible
  prefill  the same for a run of query tokens of one sequence (a chunk of a prompt, a few draft tokens)

`run` computes them in elementary torch operations or, where `own` is true, through granite_amd.HipCompute.
"""
import math

import torch

own = False

F8 = torch.float8_e4m3fn
F8_MAX = 448.0            # largest e4m3 value; 448 = 0.875 * 2^9
SCALE_EXPONENTS = (-96, 120)
DTYPES = {"f32": torch.float32, "f16": torch.float16}


# ------------------------------------------------------------------ the cases

def _append(name, tokens, start, heads, kv_heads, dim, block, src, q_out, steps=False):
    return {"name": name, "op": "append", "tokens": tokens, "start": start, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "block": block, "src": src, "q_out": q_out, "steps": steps}


def _decode(name, batch, ctx_min, ctx_max, heads, kv_heads, dim, block, kv, q, window=0, sinks=0):
    return {"name": name, "op": "decode", "batch": batch, "ctx_min": ctx_min, "ctx_max": ctx_max, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "block": block, "kv": kv, "q": q, "window": window, "sinks": sinks}


def _prefill(name, tokens, start, heads, kv_heads, dim, block, kv, q, window=0, sinks=0):
    return {"name": name, "op": "prefill", "tokens": tokens, "start": start, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "block": block, "kv": kv, "q": q, "window": window, "sinks": sinks}


def listed():
    return [
        # one step of a batched decode: every sequence appends one token to its own block
        _append("append step 64", 64, 8192, 32, 8, 128, 16, "f32", "f16", steps=True),
        # the chunk of a long prompt that the chunked prefill appends (64 heads over 8, blocks of 32)
        _append("append chunk 512 at 32768", 512, 32768, 64, 8, 128, 32, "f32", "f16"),
        # a whole prompt behind a short prefix, half projections; both ends lie inside a block
        _append("append run 8187 at 5", 8187, 5, 32, 8, 128, 16, "f16", "f32"),
        # one sequence, a short context: latency
        _decode("decode 8-bit 1 x 512", 1, 512, 512, 32, 8, 128, 16, "f8", "f32"),
        # the batched decode step of the benchmark, its cache in 8 bits
        _decode("decode 8-bit 64 x 8192", 64, 256, 8192, 32, 8, 128, 16, "f8", "f16"),
        # few sequences of a long context: the keys have to be split
        _decode("decode 8-bit 2 x 131072", 2, 120001, 131072, 64, 8, 128, 32, "f8", "f16"),
        # the same step on half pools with a short window
        _decode("decode window 1024 64 x 8192", 64, 256, 8192, 32, 8, 128, 16, "f16", "f16", 1024, 4),
        # a streaming service: long sequences, a window and sinks, 8 bits
        _decode("decode 8-bit window 4096", 16, 8192, 32768, 32, 8, 128, 16, "f8", "f32", 4096, 16),
        # a chunk of a long prompt over the cache in 8 bits
        _prefill("prefill 8-bit 512 at 32768", 512, 32768, 64, 8, 128, 32, "f8", "f16"),
        # a few tokens at once (drafts to be verified), float queries and outputs
        _prefill("prefill 8-bit 37 at 4096", 37, 4096, 32, 8, 128, 16, "f8", "f32"),
        # a whole prompt under a window, contiguous half cache
        _prefill("prefill window 512 2048", 2048, 0, 32, 8, 128, 0, "f16", "f16", 512, 4),
        # a large chunk of a long prompt under a window, head size 64, 8 bits
        _prefill("prefill 8-bit window 4096", 4096, 12288, 32, 8, 64, 16, "f8", "f16", 4096, 4),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefill", "prefill"])
    heads, kv_heads = rng.choice([(32, 8), (64, 8), (16, 16), (28, 4), (12, 2), (24, 8), (40, 5), (48, 1)])
    dim, block = rng.choice([64, 128]), rng.choice([8, 16, 20, 32, 64, 128])
    if op == "append":
        steps = rng.random() < 0.5
        tokens = _log_int(rng, 1, 256) if steps else _log_int(rng, 1, 8000)
        start = _log_int(rng, 1, 16384) if steps else _log_int(rng, 1, 32768) - 1
        c = _append("", tokens, start, heads, kv_heads, dim, block, rng.choice(["f32", "f16"]), rng.choice(["f32", "f16"]), steps)
    else:
        kv = rng.choice(["f8", "f8", "f16"])
        windowed = kv == "f16" or rng.random() < 0.4
        window, sinks = (_log_int(rng, 1, 8192), rng.choice([0, 0, 1, 4, 4, 16, 100])) if windowed else (0, 0)
        if op == "decode":
            batch = _log_int(rng, 1, 64)
            high = _log_int(rng, 1, max(1, min(65536, 8 * 270000 // (batch * kv_heads))))
            low = rng.randint(1, high)
            if kv == "f16" and rng.random() < 0.3:  # one sequence of a contiguous cache
                batch, block = 1, 0
            c = _decode("", batch, low, high, heads, kv_heads, dim, block, kv, rng.choice(["f32", "f16"]), window, sinks)
        else:
            tokens = _log_int(rng, 2, 4096)
            start = _log_int(rng, 1, max(1, min(32768, 64 * 512 * 33000 // (heads * tokens) - tokens))) - 1
            if kv == "f16" and rng.random() < 0.3:
                block = 0
            c = _prefill("", tokens, start, heads, kv_heads, dim, block, kv, rng.choice(["f32", "f16"]), window, sinks)
    del c["name"]
    return c


# ------------------------------------------------------------------ the inputs

def _lengths(case):
    """Sequence lengths of a decode case: spread evenly from ctx_min to ctx_max (the seed only permutes them)."""
    n, low, high = case["batch"], case["ctx_min"], case["ctx_max"]
    return [high if n == 1 else low + (high - low) * i // (n - 1) for i in range(n)]


def _positions(case):
    """Positions that the tokens of a batched append step take, up to `start`."""
    n, high = case["tokens"], case["start"]
    return [high if n == 1 else high * (i + 1) // n for i in range(n)]


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _power_of_two(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _scale_of(top):
    """The smallest power of two s with top <= 448 s, inside SCALE_EXPONENTS."""
    m, x = torch.frexp(top)
    e = x - 9 + (m > 0.875).to(x.dtype)
    e = torch.where(top > 0, e, torch.full_like(e, SCALE_EXPONENTS[0]))
    return _power_of_two(e.clamp(*SCALE_EXPONENTS))


def _pools(gen, blocks, case, spread):
    """K and V pools of `blocks` blocks: a factor of its own for every (head, channel), as trained keys have."""
    shape = (blocks, case["block"] or 1, case["kv_heads"], case["dim"])
    channel = torch.exp(0.5 * _normal(gen, 1, 1, *shape[2:])) * spread
    k, v = _normal(gen, *shape).mul_(channel), _normal(gen, *shape).mul_(0.5)
    if case.get("kv", "f8") == "f16":
        return (k.to(torch.float16).view(-1, *shape[2:]), v.to(torch.float16).view(-1, *shape[2:])), None
    k_scale, v_scale = _scale_of(k.abs().amax((1, 3))), _scale_of(v.abs().amax((1, 3)))
    k = k.div_(k_scale[:, None, :, None]).to(F8).view(-1, *shape[2:])
    v = v.div_(v_scale[:, None, :, None]).to(F8).view(-1, *shape[2:])
    return (k, v), (k_scale, v_scale)


def _tables(gen, used, capacity, extra=1.25):
    """Block tables of len(used) sequences over a shuffled pool; entries beyond a sequence's last block are zero."""
    total = max(1, int(sum(used) * extra))
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(used), capacity, dtype=torch.int32, device="cuda")
    slot = torch.arange(capacity, device="cuda")[None] < torch.tensor(used, device="cuda")[:, None]
    table[slot] = order[: sum(used)]
    return table, total


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case, "scale": 1.0 / math.sqrt(case["dim"])}
    bs, hq, hkv, dim = case["block"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        n = case["tokens"]
        if case["steps"]:
            at = torch.tensor(_positions(case), device="cuda", dtype=torch.int32)
            at = at[torch.randperm(n, generator=gen, device="cuda")]
            used = (at // bs + 1).tolist()
            s["positions"], last = at, case["start"]
        else:
            used = [(case["start"] + n + bs - 1) // bs]
            s["positions"], last = None, case["start"] + n - 1
        s["table"], s["blocks"] = _tables(gen, used, max(used))
        # what is there already is smaller than most of what comes: some scales have to grow
        (s["k_pool"], s["v_pool"]), (s["k_scale"], s["v_scale"]) = _pools(gen, s["blocks"], case, 0.25)
        angle = torch.arange(last + 1, device="cuda", dtype=torch.float64)[:, None] * (
            10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim))
        s["cos"], s["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        src = DTYPES[case["src"]]
        s["q"], s["k"], s["v"] = (_normal(gen, n, h, dim, dtype=src) for h in (hq, hkv, hkv))
        s["q_out"] = torch.zeros(n, hq, dim, device="cuda", dtype=DTYPES[case["q_out"]])
        return s
    if case["op"] == "decode":
        n, lens = case["batch"], torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
        lens = lens[torch.randperm(n, generator=gen, device="cuda")]
        s["lens"], longest = lens, case["ctx_max"]
        used = ((lens + bs - 1) // bs).tolist() if bs else None
        q, rows = (n, hq, dim), (n, hq)
    else:
        longest = case["start"] + case["tokens"]
        used = [(longest + bs - 1) // bs] if bs else None
        q, rows = (case["tokens"], hq, dim), (hq, case["tokens"])
    s["length"] = longest
    if bs:
        s["table"], s["blocks"] = _tables(gen, used, (longest + bs - 1) // bs)
        pools, scales = _pools(gen, s["blocks"], case, 1.0)
        s["k_pool"], s["v_pool"] = pools
        s["k_scale"], s["v_scale"] = scales or (None, None)
    else:  # contiguous: [kv_heads, tokens, dim]
        pools, _ = _pools(gen, longest, case, 1.0)
        s["k_pool"], s["v_pool"] = (p.transpose(0, 1).contiguous() for p in pools)
        s["table"] = s["k_scale"] = s["v_scale"] = None
        s["blocks"] = 0
    s["q"] = _normal(gen, *q, dtype=DTYPES[case["q"]])
    s["out"] = torch.zeros(q, device="cuda", dtype=torch.float32 if case["op"] == "decode" else DTYPES[case["q"]])
    s["lse"] = torch.zeros(rows, device="cuda")
    return s


# ------------------------------------------------------------------ the plain forms

def _rotate(x, cos, sin):
    """Pairs (2i, 2i+1) of x [n, heads, dim] by the angles of their token; every product and sum rounded to float."""
    x = x.float()
    a, b, c, s = x[..., 0::2], x[..., 1::2], cos[:, None], sin[:, None]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def _store(rows_new, pool, scale, phys, offset, count):
    """Appends to len(phys) blocks: rows_new [blocks, block, heads, dim] holds `count` new rows of each block from
    row `offset` on. A block that already holds rows keeps them, with its scale grown where the new rows ask for it."""
    blocks, size, heads, dim = rows_new.shape
    slot = torch.arange(size, device=pool.device)[None]
    new = (slot >= offset[:, None]) & (slot < (offset + count)[:, None])
    kept = slot < offset[:, None]
    rows = phys.long()[:, None] * size + slot
    codes = pool.view(torch.uint8)
    before = scale[phys.long()] * (offset > 0)[:, None]
    top = (rows_new.abs() * new[:, :, None, None]).amax((1, 3))
    after = torch.maximum(before, _scale_of(top))
    old = codes[rows].view(F8).float() * before[:, None, :, None]
    value = torch.where(new[:, :, None, None], rows_new, old) / after[:, None, :, None]
    written = new | (kept & (before > 0).any(1)[:, None])
    codes[rows[written]] = value[written].to(F8).view(torch.uint8)
    scale[phys.long()] = after


def _plain_append(s):
    case, n, bs = s["case"], s["case"]["tokens"], s["case"]["block"]
    at = s["positions"].long() if case["steps"] else case["start"] + torch.arange(n, device="cuda")
    cos, sin = s["cos"][at], s["sin"][at]
    q, k, v = _rotate(s["q"], cos, sin), _rotate(s["k"], cos, sin), s["v"].float()
    if case["steps"]:
        phys = s["table"].gather(1, (at // bs)[:, None])[:, 0]
        offset, count = at % bs, torch.ones_like(at)
        block, slot = torch.arange(n, device="cuda"), at % bs
    else:
        first, last = case["start"] // bs, (case["start"] + n - 1) // bs
        phys = s["table"][0, first: last + 1]
        begin = torch.arange(first, last + 1, device="cuda") * bs
        offset = (case["start"] - begin).clamp(min=0)
        count = (case["start"] + n - begin).clamp(max=bs) - offset
        block, slot = at // bs - first, at % bs
    rows_k, rows_v = (torch.zeros(len(phys), bs, *k.shape[1:], device="cuda") for _ in range(2))
    rows_k[block, slot], rows_v[block, slot] = k, v
    _store(rows_k, s["k_pool"], s["k_scale"], phys, offset, count)
    _store(rows_v, s["v_pool"], s["v_scale"], phys, offset, count)
    return _append_outputs(s, q.to(s["q_out"].dtype))


def _append_outputs(s, q):
    return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _gather(s, pool, scale, at):
    """Rows of the tokens at positions `at` [sequences, tokens], as float [sequences, kv_heads, tokens, dim]."""
    bs = s["case"]["block"]
    if not bs:
        return pool[:, at[0]].float()[None]
    entry = s["table"].long().gather(1, at // bs)
    x = pool.view(torch.uint8 if scale is not None else pool.dtype)[entry * bs + at % bs]
    x = x.view(F8).float() * scale[entry][..., None] if scale is not None else x.float()
    return x.transpose(1, 2)


def _attend(q, k, v, visible, scale):
    """q [..., rows, dim], k and v [..., tokens, dim], visible broadcast to [..., rows, tokens]: output and log-sum-exp."""
    x = (q @ k.transpose(-1, -2)) * scale
    x = x.masked_fill_(~visible, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    return (x @ v) / total, (total.log() + top)[..., 0]


def _plain_decode(s):
    case = s["case"]
    n, hq, hkv, dim = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    lens, window, sinks = s["lens"].long()[:, None], case["window"], case["sinks"]
    if window and window + sinks < s["length"]:  # the first tokens, then those of the window
        at = torch.arange(sinks + window, device="cuda")[None].expand(n, -1)
        start = (lens - window).clamp(min=0)
        at = torch.where(at < sinks, at, at - sinks + start)
        first = torch.arange(sinks + window, device="cuda")[None] < sinks
        visible = torch.where(first, at < start, at < lens)
        at = torch.minimum(at, lens - 1)
    else:
        at = torch.arange(s["length"], device="cuda")[None].expand(n, -1)
        visible = at < lens
        if window:
            visible = visible & ((at >= lens - window) | (at < sinks))
        at = torch.minimum(at, lens - 1)
    k, v = _gather(s, s["k_pool"], s["k_scale"], at), _gather(s, s["v_pool"], s["v_scale"], at)
    q = s["q"].float().view(n, hkv, hq // hkv, dim)
    out, lse = _attend(q, k, v, visible[:, None, None], s["scale"])
    return {"out": out.reshape(n, hq, dim), "lse": lse.reshape(n, hq)}


def _causal(case, length):
    """visible [queries, tokens]: key k to the query at position p iff k <= p, and k > p - window or k < sinks."""
    p = case["start"] + torch.arange(case["tokens"], device="cuda")[:, None]
    k = torch.arange(length, device="cuda")[None]
    visible = k <= p
    return visible & ((k > p - case["window"]) | (k < case["sinks"])) if case["window"] else visible


def _plain_prefill(s):
    case = s["case"]
    n, hq, hkv, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    at = torch.arange(s["length"], device="cuda")[None]
    k, v = _gather(s, s["k_pool"], s["k_scale"], at)[0], _gather(s, s["v_pool"], s["v_scale"], at)[0]
    q = s["q"].float().view(n, hkv, hq // hkv, dim).permute(1, 2, 0, 3)
    out, lse = _attend(q.reshape(hkv, -1, dim), k, v, _causal(case, s["length"]).repeat(hq // hkv, 1), s["scale"])
    out = out.view(hkv, hq // hkv, n, dim).permute(2, 0, 1, 3).reshape(n, hq, dim)
    return {"out": out.to(s["out"].dtype), "lse": lse.view(hq, n)}


# ------------------------------------------------------------------ one pass

def _code(t):
    from granite_amd import F16, F32, F8E4M3

    return {torch.float32: F32, torch.float16: F16, F8: F8E4M3}[t.dtype]


def _at(t):
    return None if t is None else t.data_ptr()


def _own(s):
    from granite_amd import MASK_CAUSAL, get_hip_compute

    gpu, case = get_hip_compute(0), s["case"]
    hq, hkv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        gpu.rope_append_q8(
            q=_at(s["q"]), q_out=_at(s["q_out"]), q_out_dtype=_code(s["q_out"]), k=_at(s["k"]), v=_at(s["v"]),
            src_dtype=_code(s["q"]), k_cache=_at(s["k_pool"]), v_cache=_at(s["v_pool"]), k_scale=_at(s["k_scale"]),
            v_scale=_at(s["v_scale"]), block_table=_at(s["table"]), cos_table=_at(s["cos"]), sin_table=_at(s["sin"]),
            table_positions=s["cos"].shape[0], num_heads_q=hq, num_heads_k=hkv, head_dim=dim, seq_len=case["tokens"],
            start_pos=0 if case["steps"] else case["start"], positions=_at(s["positions"]),
            table_stride=s["table"].shape[1], block_size=case["block"], num_blocks=s["blocks"],
            max_blocks_per_seq=s["table"].shape[1])
        return _append_outputs(s, s["q_out"])
    cache = dict(k_cache=_at(s["k_pool"]), v_cache=_at(s["v_pool"]), kv_dtype=_code(s["k_pool"]), k_scale=_at(s["k_scale"]),
                 v_scale=_at(s["v_scale"]), block_size=case["block"], num_blocks=s["blocks"], window=case["window"],
                 num_sinks=case["sinks"], num_heads=hq, num_kv_heads=hkv, head_dim=dim, scale=s["scale"],
                 max_seq=0 if case["block"] else s["length"])
    if case["op"] == "decode":
        gpu.decode_attention_ex(
            q=_at(s["q"]), q_dtype=_code(s["q"]), out=_at(s["out"]), lse=_at(s["lse"]), batch_size=case["batch"],
            block_tables=_at(s["table"]), seq_lens=_at(s["lens"]),
            max_blocks_per_seq=s["table"].shape[1] if case["block"] else 0, **cache)
    else:
        gpu.attention_ex(
            q=_at(s["q"]), q_dtype=_code(s["q"]), q_tok_stride=hq * dim, q_head_stride=dim, out=_at(s["out"]),
            out_dtype=_code(s["out"]), out_tok_stride=hq * dim, out_head_stride=dim, lse=_at(s["lse"]),
            seq_q=case["tokens"], cache_len=s["length"], start_pos=case["start"], block_table=_at(s["table"]),
            mask_mode=MASK_CAUSAL, **cache)
    return {"out": s["out"], "lse": s["lse"]}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill}[state["case"]["op"]](state)


# ------------------------------------------------------------------ the work

def _seen(position, window, sinks):
    """Keys that the query at `position` sees."""
    return position + 1 if not window else min(position + 1, window + min(sinks, max(0, position + 1 - window)))


def work(case):
    hq, hkv, dim, bs = case["heads"], case["kv_heads"], case["dim"], case["block"]
    size = {"f32": 4, "f16": 2, "f8": 1}
    if case["op"] == "append":
        n = case["tokens"]
        blocks = n if case["steps"] else (case["start"] + n - 1) // bs - case["start"] // bs + 1
        moved = n * dim * (hq * (size[case["src"]] + size[case["q_out"]]) + 2 * hkv * (size[case["src"]] + 1))
        return {"bytes": moved + n * dim * 4 + blocks * (4 + 2 * hkv * 8), "flops": 3 * n * dim * (hq + hkv)}
    row = 2 * hkv * dim * size[case["kv"]] + ((2 * hkv * 4 * (case["kv"] == "f8") + 4) / bs if bs else 0)
    window, sinks = case["window"], case["sinks"]
    if case["op"] == "decode":
        pairs = sum(_seen(p - 1, window, sinks) for p in _lengths(case))
        tokens, queries, out = pairs, case["batch"], 4
    else:
        n, start = case["tokens"], case["start"]
        pairs = sum(_seen(start + i, window, sinks) for i in range(n))
        first = max(0, start + 1 - window) if window else 0
        tokens, queries, out = start + n - first + min(sinks, first), n, size[case["q"]]
    return {"bytes": tokens * row + queries * hq * (dim * (size[case["q"]] + out) + 4), "flops": 4 * hq * dim * pairs}


# ------------------------------------------------------------------ the operators in 64 bits

def _exact_rotate(x, cos, sin, rounded):
    x, c, s = x.double(), cos.double()[:, None, :], sin.double()[:, None, :]
    cut = (lambda t: t.float().double()) if rounded else (lambda t: t)
    y = torch.empty_like(x)
    y[..., 0::2] = cut(cut(x[..., 0::2] * c) - cut(x[..., 1::2] * s))
    y[..., 1::2] = cut(cut(x[..., 0::2] * s) + cut(x[..., 1::2] * c))
    return y


def _exact_f8(x):
    """The nearest e4m3 value, ties to an even mantissa; |x| <= 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _token_positions(s):
    case = s["case"]
    return s["positions"].long() if case["steps"] else case["start"] + torch.arange(case["tokens"], device="cuda")


def _exact_rows(s, name, sequence, at):
    """[kv_heads, tokens, dim] in 64 bits: the tokens at positions `at` of one sequence."""
    bs, pool, scale = s["case"]["block"], s[name + "_pool"], s[name + "_scale"]
    if not bs:
        return pool[:, at].double()
    entry = s["table"][sequence].long()[at // bs]
    x = pool[entry * bs + at % bs].float().double()
    if scale is not None:
        x = x * scale[entry].double()[:, :, None]
    return x.permute(1, 0, 2)


def exact(case, seed):
    s = prepare(case, seed)

    def append():
        n, bs = case["tokens"], case["block"]
        out = {"q": _exact_rotate(s["q"], *(t[_token_positions(s)] for t in (s["cos"], s["sin"])), False)}
        # keys are stored from their float rotation: its roundings belong to the definition
        k = _exact_rotate(s["k"], *(t[_token_positions(s)] for t in (s["cos"], s["sin"])), True)
        at = _token_positions(s).tolist()
        table = s["table"].tolist()
        runs = []  # (physical block, first row, first token, tokens)
        if case["steps"]:
            runs = [(table[i][p // bs], p % bs, i, 1) for i, p in enumerate(at)]
        else:
            i = 0
            while i < n:
                take = min(bs - at[i] % bs, n - i)
                runs.append((table[0][at[i] // bs], at[i] % bs, i, take))
                i += take
        for name, x in (("k", k), ("v", s["v"].double())):
            pool, scale = s[name + "_pool"].float().double(), s[name + "_scale"].double()
            for block, row, token, take in runs:
                fresh = x[token: token + take]
                top = fresh.abs().amax((0, 2))
                need = torch.exp2(torch.ceil(torch.log2((top / F8_MAX).clamp(min=2.0 ** -200))).clamp(*SCALE_EXPONENTS))
                grown = torch.maximum(scale[block], need) if row else need
                lo = block * bs
                if row:
                    pool[lo: lo + row] = _exact_f8(pool[lo: lo + row] * (scale[block] / grown)[None, :, None])
                pool[lo + row: lo + row + take] = _exact_f8(fresh / grown[None, :, None])
                scale[block] = grown
            out[name + "_pool"], out[name + "_scale"] = pool, scale
        return out

    if case["op"] == "append":
        return append()
    hq, hkv = case["heads"], case["kv_heads"]
    group, window, sinks = hq // hkv, case["window"], case["sinks"]
    out, lse = torch.empty(s["out"].shape, device="cuda", dtype=torch.float64), torch.empty(s["lse"].shape, device="cuda", dtype=torch.float64)

    def attend(q, k, v, hidden):  # one head: q [rows, dim]
        w = (q @ k.T) / math.sqrt(case["dim"])
        w[hidden] = -math.inf
        total = torch.logsumexp(w, 1)
        return torch.exp(w - total[:, None]) @ v, total

    if case["op"] == "decode":
        for b, length in enumerate(s["lens"].tolist()):
            at = torch.arange(length, device="cuda")
            if window:
                at = at[(at >= length - window) | (at < sinks)]
            k, v = _exact_rows(s, "k", b, at), _exact_rows(s, "v", b, at)
            for h in range(hkv):
                q = s["q"][b, h * group: (h + 1) * group].double()
                out[b, h * group: (h + 1) * group], lse[b, h * group: (h + 1) * group] = attend(q, k[h], v[h], torch.zeros(group, len(at), dtype=torch.bool, device="cuda"))
        return {"out": out, "lse": lse}
    at = torch.arange(s["length"], device="cuda")
    k, v = _exact_rows(s, "k", 0, at), _exact_rows(s, "v", 0, at)
    p = case["start"] + torch.arange(case["tokens"], device="cuda")
    hidden = at[None] > p[:, None]
    if window:
        hidden |= (at[None] + window <= p[:, None]) & (at[None] >= sinks)
    for h in range(hq):
        out[:, h], lse[h] = attend(s["q"][:, h].double(), k[h // group], v[h // group], hidden)
    return {"out": out, "lse": lse}
