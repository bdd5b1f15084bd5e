"""The operators around windowed attention over the paged cache, as one serving step uses them: the
step's tables, rotary positions with the cache write, and attention with a sliding window and a few
first tokens that stay visible (decode and prefill).

A case is a dict of plain values.  `prepare` makes what a program has in hand before the call, `run`
is one call and its outputs -- in plain torch operations, or, where `own` is set, through the
framework's entry points -- `exact` is the operator's definition in 64 bits and `work` what a call
cannot do without.  Lengths come from the case alone, values from the seed.

Caches have the framework's layout: keys [blocks, kv_heads, head_size / 8, 16, 8], values
[blocks, kv_heads, head_size, 16], 16 tokens to a block.
"""
import math
import random

import numpy as np
import torch

own = False

BLOCK = 16
HEAD = 128  # head size of the attention operators
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # the tables of a decode step: 64 requests, one new token each
        step("step_tables decode 64", 64, 0, 1, 4096, 1),
        # a step of a large batch that takes in 64 chunks of prompts beside its decode tokens
        step("step_tables 2048 with 64 chunks", 2048, 64, 1024, 8192, 2),
        # the decode step of 64 sequences, 32 heads: rotate the new tokens and write them to the cache
        rotary("rotary+cache decode 64", [1] * 64, 32, 32, 128, 128, True, "bf16", "f32", 4096, 3),
        # a prompt batch through a model that rotates half of each head, pairs side by side
        rotary("rotary+cache prompts 16384", [2048] * 6 + [4095, 1], 64, 8, 128, 64, False, "f16", "f32", 32768, 4),
        # the table of a model with a context of 4096
        table("cos/sin table 4096", 4096, 128, 10000.0, "none", 1.0, 4096, "f32"),
        # the table of a context stretched eight times by wavelength bands
        table("cos/sin table 131072 yarn", 131072, 128, 500000.0, "yarn", 8.0, 16384, "f32"),
        # one user: a single sequence far beyond the window, where latency counts
        decode("window decode 1 of 16384", [16384], 32, 8, 1024, 4, "bf16", 5),
        # batch 64 of a model without grouped heads, contexts 512-4096
        decode("window decode 64 mha", uniform(64, 512, 4096, 6), 32, 32, 2048, 4, "bf16", 6),
        # the decode part of a mixed step: 192 sequences, contexts 256-16384
        decode("window decode 192 gqa", uniform(192, 256, 16384, 7), 32, 8, 4096, 16, "f16", 7),
        # four short prompts packed together, a window shorter than most of them
        prefill("window prefill 4 short", [64, 128, 256, 512], [64, 128, 256, 512], 32, 32, 128, 4, "bf16", False, 8),
        # chunks of 512 new tokens on 7680 cached ones, read from the paged cache
        prefill("window chunks 8 x 512 paged", [512] * 8, [8192] * 8, 32, 8, 1024, 4, "f16", True, 9),
        # two long prompts
        prefill("window prefill 2 x 32768", [32768] * 2, [32768] * 2, 64, 8, 4096, 4, "bf16", False, 10),
    ]


def step(name, requests, chunks, chunk, max_ctx, lens):
    return {"name": name, "op": "step", "requests": requests, "chunks": chunks, "chunk": chunk, "max_ctx": max_ctx, "lens": lens}


def rotary(name, runs, heads, kv_heads, head, rot, neox, type_, table_, positions, lens):
    return {"name": name, "op": "rotary", "runs": " ".join(map(str, runs)), "heads": heads, "kv_heads": kv_heads, "head": head, "rot": rot,
            "neox": neox, "type": type_, "table": table_, "positions": positions, "lens": lens}


def table(name, positions, rot, base, scaling, factor, original, type_):
    return {"name": name, "op": "table", "positions": positions, "rot": rot, "base": base, "scaling": scaling, "factor": factor,
            "original": original, "type": type_}


def decode(name, ctx, heads, kv_heads, window, sinks, type_, lens):
    return {"name": name, "op": "decode", "ctx": " ".join(map(str, ctx)), "heads": heads, "kv_heads": kv_heads, "window": window,
            "sinks": sinks, "type": type_, "lens": lens}


def prefill(name, lens_q, lens_k, heads, kv_heads, window, sinks, type_, paged, lens):
    return {"name": name, "op": "prefill", "lens_q": " ".join(map(str, lens_q)), "lens_k": " ".join(map(str, lens_k)), "heads": heads,
            "kv_heads": kv_heads, "window": window, "sinks": sinks, "type": type_, "paged": paged, "lens": lens}


def uniform(n, lo, hi, seed):
    r = random.Random(seed)
    return [r.randint(lo, hi) for _ in range(n)]


def numbers(text):
    return [int(x) for x in text.split()]


def log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "rotary", "table", "decode", "decode", "prefill", "prefill"])
    lens = rng.randrange(1 << 30)
    type_ = rng.choice(["bf16", "f16"])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    window = log_between(rng, 1, 8192)
    sinks = rng.choice([0, 0, 1, 4, 16, rng.randint(2, 300)])
    if op == "step":
        chunks = rng.choice([0, rng.randint(1, 64)])
        return unnamed(step("", max(chunks, log_between(rng, 1, 2048)), chunks, log_between(rng, 2, 1024), log_between(rng, 16, 8192), lens))
    if op == "rotary":
        head = rng.choice([64, 80, 96, 128, 128, 128, 256])
        rot = rng.choice([head, 16 * rng.randint(1, head // 16)])
        tokens = log_between(rng, 1, 16384 * 128 * 72 // (head * (heads + kv_heads)) if head * (heads + kv_heads) > 128 * 72 else 16384)
        runs = [1] * tokens if rng.random() < 0.3 and tokens <= 512 else split(rng, tokens)
        return unnamed(rotary("", runs, heads, kv_heads, head, rot, rng.random() < 0.5, type_, rng.choice(["f32", type_]), 40000, lens))
    if op == "table":
        return unnamed(table("", log_between(rng, 1, 131072), 16 * rng.randint(1, 8), rng.choice([10000.0, 500000.0, 1e6]),
                             rng.choice(["none", "linear", "ntk", "yarn"]), rng.choice([1.0, 2.0, 3.5, 8.0, 16.0]),
                             rng.choice([2048, 4096, 8192, 32768]), rng.choice(["f32", "f32", "bf16", "f16"])))
    if op == "decode":
        seqs, most = log_between(rng, 1, 192), log_between(rng, 1, 16384)
        ctx = [rng.randint(0 if rng.random() < 0.1 else (most + 1) // 2, most) for _ in range(seqs)]
        return unnamed(decode("", ctx, heads, kv_heads, window, sinks, type_, lens))
    lens_q = split(rng, log_between(rng, 1, 16384))
    paged = rng.random() < 0.5
    lens_k = [q + rng.choice([0, 0, rng.randint(1, 4096)]) for q in lens_q]
    return unnamed(prefill("", lens_q, lens_k, heads, kv_heads, min(window, 4096), sinks, type_, paged, lens))


def unnamed(case):
    del case["name"]
    return case


def split(rng, total):
    """`total` tokens as one to eight runs of uneven lengths."""
    cuts = sorted(rng.randint(0, total) for _ in range(rng.randint(0, 7)))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


# ---- inputs ------------------------------------------------------------------------------------------

def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, type_, *shape):
    return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).to(TYPES[type_])


def ints(values, type_=torch.int32):
    return torch.tensor(values, dtype=type_).to("cuda")


def running_sum(lens):
    return ints([sum(lens[:i]) for i in range(len(lens) + 1)])


def scattered_blocks(lens, seed, g):
    """Each sequence's blocks somewhere in a pool a little larger than all of them: table, and pool size."""
    counts = [-(-n // BLOCK) for n in lens]
    pool = sum(counts) + 8
    order = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
    width = max(max(counts, default=0), 1)
    starts = ints([sum(counts[:i]) for i in range(len(counts))], torch.int64)
    column = torch.arange(width, device="cuda")
    at = (starts[:, None] + column).clamp_(max=pool - 1)
    return torch.where(column < ints(counts)[:, None], order[at], 0).to(torch.int32).contiguous(), pool


def step_lens(case):
    r = random.Random(case["lens"])
    n = case["requests"]
    news = [r.randint(max(1, case["chunk"] // 2), case["chunk"]) if i < case["chunks"] else 1 for i in range(n)]
    r.shuffle(news)
    return news, [r.randint(0, case["max_ctx"]) for _ in range(n)]


def prepare(case, seed):
    g = generator(seed)
    op = case["op"]
    s = {"case": case}
    if op == "step":
        news, ctx = step_lens(case)
        counts = [-(-c // BLOCK) for c in ctx]
        width = max(-(-(c + q) // BLOCK) for c, q in zip(ctx, news))
        held = sum(counts)
        pool = sum(-(-(c + q) // BLOCK) for c, q in zip(ctx, news)) + 100
        order = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
        column = torch.arange(width, device="cuda")
        starts = ints([sum(counts[:i]) for i in range(len(counts))], torch.int64)
        at = (starts[:, None] + column).clamp_(max=pool - 1)
        s["block_tables"] = torch.where(column < ints(counts)[:, None], order[at], 0).to(torch.int32).contiguous()
        s["free_blocks"] = order[held:].contiguous()
        s["free_count"] = ints([pool - held])
        s["query_lens"], s["context_lens"] = ints(news), ints(ctx)
        s["num_blocks"], s["max_tokens"] = pool, sum(news)
        return s
    if op == "table":
        # a table is a function of its sizes; the seed picks the base within a tenth of a per cent
        s["base"] = case["base"] * (1 + 1e-3 * random.Random(seed).random())
        return s
    if op == "rotary":
        runs, H, Hk, D = numbers(case["runs"]), case["heads"], case["kv_heads"], case["head"]
        r = random.Random(case["lens"])
        T = sum(runs)
        begins = [r.randint(0, case["positions"] - n) for n in runs]
        qkv = normal(g, case["type"], T, (H + 2 * Hk) * D)
        s["query"], s["key"], s["value"] = qkv[:, :H * D], qkv[:, H * D:(H + Hk) * D], qkv[:, (H + Hk) * D:]
        tables, pool = scattered_blocks([b % BLOCK + n for b, n in zip(begins, runs)], case["lens"], g)
        seq = torch.repeat_interleave(torch.arange(len(runs), device="cuda"), ints(runs, torch.int64), output_size=T)
        first = running_sum(runs)[:-1].to(torch.int64)
        begin = ints(begins, torch.int64)
        s["positions"] = begin[seq] + torch.arange(T, device="cuda") - first[seq]
        inside = s["positions"] - (begin[seq] // BLOCK) * BLOCK
        s["slot_mapping"] = (tables[seq, inside // BLOCK] * BLOCK + inside % BLOCK).to(torch.int32)
        angle = torch.arange(case["positions"], device="cuda", dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).to(TYPES[case["table"]])
        s["key_cache"] = normal(g, case["type"], pool, Hk, D // 8, BLOCK, 8)
        s["value_cache"] = normal(g, case["type"], pool, Hk, D, BLOCK)
        return s
    H, Hk = case["heads"], case["kv_heads"]
    s["scale"] = 1 / math.sqrt(HEAD)
    if op == "decode":
        ctx = numbers(case["ctx"])
        s["block_tables"], pool = scattered_blocks(ctx, case["lens"], g)
        s["context_lens"], s["max_ctx"] = ints(ctx), max(ctx)
        s["query"] = normal(g, case["type"], len(ctx), H, HEAD)
        s["out"] = torch.empty_like(s["query"])
    else:
        lens_q, lens_k = numbers(case["lens_q"]), numbers(case["lens_k"])
        s["lens_q"], s["lens_k"] = lens_q, lens_k
        s["seqlens_q"] = running_sum(lens_q)
        s["max_q"], s["max_k"] = max(lens_q), max(lens_k)
        if not case["paged"]:
            s["seqlens_k"] = running_sum(lens_k)
            if lens_q == lens_k:  # slices of one projection, as a model has them
                qkv = normal(g, case["type"], sum(lens_q), H + 2 * Hk, HEAD)
                s["query"], s["key"], s["value"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
            else:
                s["query"] = normal(g, case["type"], sum(lens_q), H, HEAD)
                s["key"] = normal(g, case["type"], sum(lens_k), Hk, HEAD)
                s["value"] = normal(g, case["type"], sum(lens_k), Hk, HEAD)
            return s
        s["query"] = normal(g, case["type"], sum(lens_q), H, HEAD)
        s["block_tables"], pool = scattered_blocks(lens_k, case["lens"], g)
        s["context_lens"] = ints(lens_k)
    s["key_cache"] = normal(g, case["type"], pool, Hk, HEAD // 8, BLOCK, 8)
    s["value_cache"] = normal(g, case["type"], pool, Hk, HEAD, BLOCK)
    return s


# ---- one pass ----------------------------------------------------------------------------------------

def run(s):
    return (run_own if own else run_plain)(s)


def run_own(s):
    from aici_b200 import batch_info, tch_cuda
    case = s["case"]
    op = case["op"]
    if op == "step":
        t = batch_info.step_tables(s["query_lens"], s["context_lens"], s["block_tables"], s["free_blocks"], s["free_count"],
                                   s["num_blocks"], s["max_tokens"])
        return [t.seqlens_q, t.positions, t.slot_mapping, t.logit_idxs, t.context_lens, t.free_count, s["block_tables"]]
    if op == "table":
        return tch_cuda.rotary_cos_sin_cache(case["positions"], case["rot"], s["base"], TYPES[case["type"]], torch.device("cuda", torch.cuda.current_device()),
                                             scaling=case["scaling"], factor=case["factor"], original_context=case["original"])
    if op == "rotary":
        tch_cuda.rotary_embedding_and_cache(s["positions"], s["query"], s["key"], s["value"], case["head"], s["cos_sin"], case["neox"],
                                            s["key_cache"], s["value_cache"], s["slot_mapping"])
        return [s["query"], s["key"], s["key_cache"], s["value_cache"]]
    if op == "decode":
        tch_cuda.paged_attention_window(s["out"], s["query"], s["key_cache"], s["value_cache"], case["kv_heads"], s["scale"],
                                        s["block_tables"], s["context_lens"], BLOCK, s["max_ctx"], case["window"], case["sinks"])
        return s["out"]
    if case["paged"]:
        return tch_cuda.flash_attn_varlen_paged_window(s["query"], s["key_cache"], s["value_cache"], s["seqlens_q"], s["context_lens"],
                                                       s["block_tables"], s["max_q"], s["max_k"], s["scale"], case["window"], case["sinks"])
    return tch_cuda.flash_attn_varlen_window(s["query"], s["key"], s["value"], s["seqlens_q"], s["seqlens_k"], s["max_q"], s["max_k"],
                                             s["scale"], case["window"], case["sinks"])


def run_plain(s):
    return {"step": plain_step, "table": plain_table, "rotary": plain_rotary, "decode": plain_decode, "prefill": plain_prefill}[s["case"]["op"]](s)


def plain_step(s):
    """New tokens t of request i get positions ctx_i, ctx_i + 1, ...; a position that begins a block takes the
    next block from the end of the free list; slot = block * 16 + position % 16."""
    q, ctx, tables, free, count = (s[k] for k in ("query_lens", "context_lens", "block_tables", "free_blocks", "free_count"))
    cu = torch.nn.functional.pad(q.cumsum(0), (1, 0))
    t = torch.arange(s["max_tokens"], device=q.device)
    req = torch.searchsorted(cu[1:], t, right=True)
    pos = ctx[req].long() + t - cu[req]
    fresh = pos % BLOCK == 0
    rank = (fresh.cumsum(0) - 1).clamp(min=0)
    taken = free[count - 1 - rank]
    blk = pos // BLOCK
    at = torch.where(fresh, req * tables.shape[1] + blk, tables.numel())  # one place behind the table takes what is not written
    grown = torch.cat([tables.flatten(), tables.new_zeros(1)]).scatter(0, at, taken)
    tables.copy_(grown[:-1].view_as(tables))
    slots = tables[req, blk] * BLOCK + (pos % BLOCK).int()
    last = torch.where(q > 0, cu[1:] - 1, -1)
    return [cu.int(), pos, slots, last.int(), ctx + q, (count - fresh.sum()).int(), tables]


def frequencies(case, base):
    """Angle per position of each pair, in 64 bits (yarn: wavelengths below original / 32 keep theirs, those
    above original are stretched, the ones between are mixed), and the factor on cosine and sine."""
    rot, s = case["rot"], case["factor"]
    i = torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot
    if case["scaling"] == "ntk":
        return (base * s ** (rot / max(rot - 2, 1))) ** -i, 1.0
    f = base ** -i
    if case["scaling"] == "linear":
        return f / s, 1.0
    if case["scaling"] == "yarn":
        keep = ((case["original"] * f / (2 * math.pi) - 1) / (32 - 1)).clamp(0, 1)
        return f * (keep + (1 - keep) / s), 0.1 * math.log(s) + 1
    return f, 1.0


def plain_table(s):
    f, by = frequencies(s["case"], s["base"])
    angle = torch.arange(s["case"]["positions"], device="cuda", dtype=torch.float64)[:, None] * f
    return torch.cat([angle.cos() * by, angle.sin() * by], 1).to(TYPES[s["case"]["type"]])


def rotated(x, cos, sin, neox, rot):
    """x [tokens, heads, head_size] in 32 or 64 bits; cos and sin [tokens, rot / 2]."""
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if neox else (x[..., 0:rot:2], x[..., 1:rot:2])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([u, v], -1) if neox else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def plain_rotary(s):
    case = s["case"]
    D, rot = case["head"], case["rot"]
    cs = s["cos_sin"][s["positions"]].float()
    cos, sin = cs[:, :rot // 2], cs[:, rot // 2:]
    q, k, v = (s[n].unflatten(1, (-1, D)) for n in ("query", "key", "value"))
    q.copy_(rotated(q.float(), cos, sin, case["neox"], rot))
    k.copy_(rotated(k.float(), cos, sin, case["neox"], rot))
    blk, off = s["slot_mapping"].long() // BLOCK, s["slot_mapping"].long() % BLOCK
    s["key_cache"][blk, :, :, off] = k.unflatten(2, (D // 8, 8))
    s["value_cache"][blk, :, :, off] = v
    return [s["query"], s["key"], s["key_cache"], s["value_cache"]]


def cached(cache, blk, off):
    """Tokens of a cache as [..., kv_heads, head_size], in 32 bits."""
    x = cache[blk, :, :, off].float()
    return x.flatten(-2) if cache.dim() == 5 else x


def plain_decode(s):
    """A query at position ctx - 1 sees the tokens t < ctx with t >= ctx - window or t < sinks."""
    case = s["case"]
    ctx = s["context_lens"].long()
    n, H, Hk = len(ctx), case["heads"], case["kv_heads"]
    begin = (ctx - case["window"]).clamp(min=0)
    first = begin.clamp(max=case["sinks"])
    j = torch.arange(max(1, min(s["max_ctx"], case["window"] + case["sinks"])), device=ctx.device)
    t = torch.where(j < first[:, None], j, begin[:, None] + j - first[:, None])
    seen = t < ctx[:, None]
    blk = s["block_tables"].gather(1, (t // BLOCK).clamp(max=s["block_tables"].shape[1] - 1)).long()
    k, v = cached(s["key_cache"], blk, t % BLOCK), cached(s["value_cache"], blk, t % BLOCK)
    q = s["query"].float().view(n, Hk, H // Hk, HEAD)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)) * s["scale"]
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = (score - top).exp()
    o = torch.matmul(p, v.transpose(1, 2)) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    s["out"].copy_(o.view(n, H, HEAD))
    return s["out"]


ROWS = 2048  # rows of one product of the plain prefill


def plain_prefill(s):
    """Row r of a sequence is the token at position lens_k - lens_q + r; it sees the tokens t at or before its
    own with t > its position - window or t < sinks."""
    case = s["case"]
    H, Hk, W, S = case["heads"], case["kv_heads"], case["window"], case["sinks"]
    out = torch.zeros(s["query"].shape, dtype=s["query"].dtype, device="cuda")
    q0 = k0 = 0
    for i, (lq, lk) in enumerate(zip(s["lens_q"], s["lens_k"])):
        for r in range(0, lq, ROWS):
            rows = min(ROWS, lq - r)
            own_pos = torch.arange(r, r + rows, device="cuda") + lk - lq
            begin, end = max(0, lk - lq + r - W + 1), lk - lq + r + rows
            t = torch.cat([torch.arange(min(S, begin), device="cuda"), torch.arange(begin, end, device="cuda")])
            if case["paged"]:
                blk = s["block_tables"][i, t // BLOCK].long()
                k, v = cached(s["key_cache"], blk, t % BLOCK), cached(s["value_cache"], blk, t % BLOCK)
            else:
                k, v = s["key"][k0 + t].float(), s["value"][k0 + t].float()
            q = s["query"][q0 + r:q0 + r + rows].float().view(rows, Hk, H // Hk, HEAD).permute(1, 2, 0, 3)
            score = torch.matmul(q, k.permute(1, 2, 0)[:, None]).mul_(s["scale"])
            seen = (t <= own_pos[:, None]) & ((t > own_pos[:, None] - W) | (t < S))
            score.masked_fill_(~seen, -math.inf)
            score.sub_(score.amax(-1, keepdim=True)).exp_()
            o = torch.matmul(score, v.transpose(0, 1)[:, None]) / score.sum(-1, keepdim=True)
            out[q0 + r:q0 + r + rows] = o.permute(2, 0, 1, 3).reshape(rows, H, HEAD)
        q0, k0 = q0 + lq, k0 + lk
    return out


# ---- in 64 bits, apart from the plain forms ------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"step": exact_step, "table": exact_table, "rotary": exact_rotary, "decode": exact_decode, "prefill": exact_prefill}[case["op"]](s)


def exact_step(s):
    return None  # whole numbers: compared with the plain form's


def exact_table(s):
    """In the host's longest floats, one pair at a time."""
    case, rot, factor = s["case"], s["case"]["rot"], np.longdouble(s["case"]["factor"])
    at = np.arange(case["positions"], dtype=np.longdouble)
    out = np.empty((case["positions"], rot))
    by = 1.0
    for i in range(rot // 2):
        base = np.longdouble(s["base"])
        if case["scaling"] == "ntk":
            base *= factor ** (np.longdouble(rot) / max(rot - 2, 1))
        f = base ** (np.longdouble(-2 * i) / rot)
        if case["scaling"] == "linear":
            f /= factor
        if case["scaling"] == "yarn":
            turns = case["original"] * f / (2 * np.longdouble("3.14159265358979323846264338327950288"))
            kept = min(max((turns - 1) / 31, 0), 1)
            f = kept * f + (1 - kept) * (f / factor)
            by = 0.1 * math.log(case["factor"]) + 1
        out[:, i] = np.cos(at * f) * by
        out[:, rot // 2 + i] = np.sin(at * f) * by
    return torch.from_numpy(out)


def exact_rotary(s):
    """Each pair as a complex number times cos + i sin."""
    case = s["case"]
    D, rot = case["head"], case["rot"]
    cs = s["cos_sin"].double()[s["positions"]]
    turn = torch.complex(cs[:, :rot // 2], cs[:, rot // 2:])[:, None]

    def turned(x):
        x = x.double().reshape(x.shape[0], -1, D)
        pairs = x[..., :rot].reshape(*x.shape[:2], 2, rot // 2).transpose(2, 3) if case["neox"] else x[..., :rot].reshape(*x.shape[:2], rot // 2, 2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        y = x.clone()
        y[..., :rot] = (z.transpose(2, 3) if case["neox"] else z).reshape(*x.shape[:2], rot)
        return y

    q, k = turned(s["query"]), turned(s["key"])
    kc, vc = s["key_cache"].double(), s["value_cache"].double()
    slot = s["slot_mapping"].long()
    rows = kc.permute(0, 3, 1, 2, 4).reshape(-1, case["kv_heads"], D)  # one row to a slot
    rows[slot] = k
    kc = rows.view(kc.shape[0], BLOCK, case["kv_heads"], D // 8, 8).permute(0, 2, 3, 1, 4)
    rows = vc.permute(0, 3, 1, 2).reshape(-1, case["kv_heads"], D)
    rows[slot] = s["value"].double().reshape(len(slot), -1, D)
    vc = rows.view(vc.shape[0], BLOCK, case["kv_heads"], D).permute(0, 2, 3, 1)
    return [q.flatten(1), k.flatten(1), kc.contiguous(), vc.contiguous()]


def slots_of(table_row, n):
    t = torch.arange(n, device="cuda")
    return table_row[t // BLOCK].long() * BLOCK + t % BLOCK


def exact_rows(query, k, v, positions, case, scale):
    """Softmax attention of rows at `positions` over the tokens 0 .. len(k) - 1, the mask written out."""
    H, Hk = case["heads"], case["kv_heads"]
    t = torch.arange(len(k), device="cuda")
    p = positions[:, None]
    hidden = (t > p) | ((t <= p - case["window"]) & (t >= case["sinks"]))
    out = torch.empty(len(query), H, HEAD, dtype=torch.float64, device="cuda")
    some = torch.nonzero(~hidden.all(0)).flatten()  # tokens that no row sees count for nothing
    hidden = hidden[:, some]
    for h in range(Hk):
        kk, vv = k[some, h].double(), v[some, h].double()
        qq = query[:, h * (H // Hk):(h + 1) * (H // Hk)].double().transpose(0, 1)
        w = (qq @ kk.T * scale).masked_fill(hidden, -math.inf)
        w = torch.exp(w - torch.logsumexp(w, -1, keepdim=True)).nan_to_num(0.0)
        out[:, h * (H // Hk):(h + 1) * (H // Hk)] = (w @ vv).transpose(0, 1)
    return out


def exact_decode(s):
    case, ctx = s["case"], numbers(s["case"]["ctx"])
    out = torch.zeros(len(ctx), case["heads"], HEAD, dtype=torch.float64, device="cuda")
    for i, n in enumerate(ctx):
        if n == 0:
            continue
        t = torch.arange(n, device="cuda")
        t = t[(t >= n - case["window"]) | (t < case["sinks"])]
        slot = s["block_tables"][i, t // BLOCK].long() * BLOCK + t % BLOCK
        k = s["key_cache"][slot // BLOCK, :, :, slot % BLOCK].reshape(len(t), case["kv_heads"], HEAD)
        v = s["value_cache"][slot // BLOCK, :, :, slot % BLOCK]
        all_seen = dict(case, window=len(t), sinks=0)
        out[i:i + 1] = exact_rows(s["query"][i:i + 1], k, v, ints([len(t) - 1], torch.int64), all_seen, s["scale"])
    return out


def exact_prefill(s):
    case = s["case"]
    parts, q0, k0 = [], 0, 0
    for i, (lq, lk) in enumerate(zip(s["lens_q"], s["lens_k"])):
        if case["paged"]:
            slot = slots_of(s["block_tables"][i], lk)
            k = s["key_cache"][slot // BLOCK, :, :, slot % BLOCK].reshape(lk, case["kv_heads"], HEAD)
            v = s["value_cache"][slot // BLOCK, :, :, slot % BLOCK]
        else:
            k, v = s["key"][k0:k0 + lk], s["value"][k0:k0 + lk]
        for r in range(0, lq, 4096):
            n = min(4096, lq - r)
            at = torch.arange(r, r + n, device="cuda") + lk - lq
            parts.append(exact_rows(s["query"][q0 + r:q0 + r + n], k, v, at, case, s["scale"]))
        q0, k0 = q0 + lq, k0 + lk
    return torch.cat(parts) if parts else None


# ---- what a call cannot do without ---------------------------------------------------------------------

def seen_by_row(position, window, sinks):
    """How many tokens a row at `position` sees."""
    begin = max(0, position + 1 - window)
    return position + 1 - begin + min(sinks, begin)


def work(case):
    op = case["op"]
    if op == "step":
        news, ctx = step_lens(case)
        n, T = case["requests"], sum(news)
        fresh = sum(-(-(c + q) // BLOCK) - -(-c // BLOCK) for c, q in zip(ctx, news))
        # lengths in and out, tokens' positions and slots, blocks taken and entered, one table entry for each block continued
        return {"bytes": 8 * n + 12 * n + 12 * T + 8 * fresh + 4 * sum(c % BLOCK > 0 for c in ctx), "flops": 0}
    if op == "table":
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": case["positions"] * case["rot"] * size, "flops": 0}
    H, Hk = case["heads"], case["kv_heads"]
    if op == "rotary":
        T, D, rot = sum(numbers(case["runs"])), case["head"], case["rot"]
        one = rot * (4 if case["table"] == "f32" else 2) + 12  # a row of the table, position and slot
        moved = 2 * H * rot * 2 + Hk * (rot * 2 + D * 2 + D * 2) + Hk * 2 * D * 2  # only the rotated part of a query moves
        return {"bytes": T * (one + moved), "flops": T * (H + Hk) * rot * 3}
    if op == "decode":
        ctx = numbers(case["ctx"])
        seen = sum(seen_by_row(c - 1, case["window"], case["sinks"]) for c in ctx if c)
        blocks = sum(-(-seen_by_row(c - 1, case["window"], case["sinks"]) // BLOCK) for c in ctx if c)
        return {"bytes": seen * Hk * HEAD * 4 + len(ctx) * (H * HEAD * 4 + 4) + 4 * blocks, "flops": 4 * HEAD * H * seen}
    lens_q, lens_k = numbers(case["lens_q"]), numbers(case["lens_k"])
    pairs = sum(seen_by_row(lk - lq + r, case["window"], case["sinks"]) for lq, lk in zip(lens_q, lens_k) for r in range(lq))
    some = sum(min(lk, lq - 1 + case["window"] + case["sinks"]) for lq, lk in zip(lens_q, lens_k) if lq)
    return {"bytes": sum(lens_q) * H * HEAD * 4 + some * Hk * HEAD * 4, "flops": 4 * HEAD * H * pairs}
