"""The operators around windowed attention in 64 bits, on the CPU, one token at a time where that is
the plainest way -- TEST INFRASTRUCTURE ONLY, like the rest of this folder."""
import math

import torch

BLOCK = 16


def step_tables(query_lens, context_lens, tables, free, count, max_tokens, num_blocks):
    """Lists of Python ints; returns (seqlens_q, positions, slots, logit_idxs, context, count, tables) of
    the step, or of a step without tokens if it does not fit, and the kind of refusal."""
    n, width = len(query_lens), len(tables[0])
    tables = [list(r) for r in tables]
    bad = count < 0 or count > len(free) or any(q < 0 or c < 0 or c + q > width * BLOCK
                                                for q, c in zip(query_lens, context_lens))
    need = 0 if bad else sum(-(-(c + q) // BLOCK) - -(-c // BLOCK) for q, c in zip(query_lens, context_lens))
    kind = "bad" if bad else "blocks" if need > count else "bad" if sum(query_lens) > max_tokens else None
    qs = [0] * n if kind else query_lens
    cu, pos, slots, logits, ctx = [0], [], [], [], []
    for i in range(n):
        for p in range(context_lens[i], context_lens[i] + qs[i]):
            if p % BLOCK == 0:
                count -= 1
                tables[i][p // BLOCK] = free[count]
            b = tables[i][p // BLOCK]
            pos.append(p)
            slots.append(b * BLOCK + p % BLOCK if 0 <= b < num_blocks else -1)
        cu.append(cu[-1] + qs[i])
        logits.append(cu[-1] - 1 if qs[i] else -1)
        ctx.append(context_lens[i] + qs[i])
    rest = max_tokens - len(pos)
    return cu, pos + [0] * rest, slots + [-1] * rest, logits, ctx, count, tables, kind


def cos_sin(positions, rot_dim, base, scaling, factor, original):
    """Cosines and sines [len(positions), rot_dim] in 64 bits."""
    j = torch.arange(rot_dim // 2, dtype=torch.float64)
    by = 1.0
    if scaling == "ntk":
        base = base * factor ** (rot_dim / (rot_dim - 2))
    f = torch.exp(-2 * j / rot_dim * math.log(base))
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        turns = original / (2 * math.pi / f)
        share = torch.clamp((turns - 1) / (32 - 1), 0, 1)
        f = share * f + (1 - share) * f / factor
        by = 0.1 * math.log(factor) + 1
    angle = torch.as_tensor(positions, dtype=torch.float64)[:, None] * f
    return torch.cat([torch.cos(angle), torch.sin(angle)], 1) * by


def rotate(x, cs, neox):
    """x [tokens, heads, head_size] of any type, cs [tokens, rot_dim]; returns 64 bits, and for each
    element the sum of the magnitudes of its two products."""
    rot = cs.shape[1]
    cs = cs.double()
    y, mag = x.double().clone(), x.double().abs()
    for j in range(rot // 2):
        a, b = (j, j + rot // 2) if neox else (2 * j, 2 * j + 1)
        c, s = cs[:, j, None], cs[:, rot // 2 + j, None]
        xa, xb = x[..., a].double(), x[..., b].double()
        y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
        mag[..., a], mag[..., b] = (xa * c).abs() + (xb * s).abs(), (xb * c).abs() + (xa * s).abs()
    return y, mag


def write_cache(key, value, key_cache, value_cache, slots):
    """In place; key / value [tokens, heads, head_size], caches of the framework's layout."""
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            b, o = divmod(s, BLOCK)
            key_cache[b, :, :, o] = key[t].view(key.shape[1], -1, 8).to(key_cache.dtype)
            value_cache[b, :, :, o] = value[t].to(value_cache.dtype)


def read_cache(key_cache, value_cache, table_row, n):
    """Tokens 0 .. n - 1 of a sequence as [n, heads, head_size]."""
    t = torch.arange(n)
    b, o = table_row[t // BLOCK].long(), t % BLOCK
    return key_cache[b, :, :, o].flatten(2), value_cache[b, :, :, o]


def visible(position, window, sinks):
    """The tokens that the query at `position` sees."""
    return [t for t in range(position + 1) if t > position - window or t < sinks]


def attention_row(q, k, v, position, window, sinks, scale):
    """q [heads, head_size], k and v [tokens, kv_heads, head_size]: the output [heads, head_size] in 64
    bits, the same with |v| in place of v, how many tokens count, and the largest sum of magnitudes of a
    score's products."""
    H, D = q.shape
    Hk = k.shape[1]
    t = visible(position, window, sinks)
    if not t:
        z = torch.zeros(H, D, dtype=torch.float64)
        return z, z, 0, 0.0
    kk, vv = k[t].double(), v[t].double()
    qq = q.double().view(Hk, H // Hk, D)
    s = torch.einsum("hgd,thd->hgt", qq, kk) * scale
    size = float(torch.einsum("hgd,thd->hgt", qq.abs(), kk.abs()).max()) * scale
    p = torch.softmax(s, -1)
    return (torch.einsum("hgt,thd->hgd", p, vv).reshape(H, D), torch.einsum("hgt,thd->hgd", p, vv.abs()).reshape(H, D),
            len(t), size)


def attention_bound(o, a, n, size, vmax, dtype, split=False):
    """How far a kernel's output may be from `o`: half a step of the 16-bit type for the output and one for
    each probability, the fp32 sums over n tokens, the fp32 scores of 128 products each (which reach both
    the probabilities and their sum), exp2 in fp32, and for f16 probabilities below its normal range.  With
    `split` a probability is its rounded value plus what the rounding left, rounded: half a step squared."""
    half = torch.finfo(dtype).eps / 2
    small = n * 2.0 ** -23 + 2 * (128 * 2.0 ** -24 * size * 1.4427 + 2.0 ** -21)
    under = n * 2.0 ** -25 * vmax if dtype == torch.float16 else 0.0
    return (half * o.abs() + (half * half if split else half) * a + small * a) * 1.01 + under + 1e-30
