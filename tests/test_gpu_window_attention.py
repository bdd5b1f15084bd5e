"""Attention with a sliding window and sinks -- decode over the paged cache, prefill over packed tensors
and over the cache -- against the definition in 64 bits, at the sizes and masks where it can go wrong."""
import math
import random

import pytest
import torch

from aici_b200 import _lib, tch_cuda
from oracle import window_ref as W

pytestmark = pytest.mark.gpu
D, SCALE = 128, 1 / math.sqrt(128)
NAN = float("nan")
TYPES = [torch.bfloat16, torch.float16]


def normal(g, dtype, *shape):
    return torch.randn(*shape, generator=g).to(dtype)


def paged(g, lens, Hk, dtype, extra_blocks=3):
    """Sequences in shuffled blocks: caches, table, and the tokens [n, Hk, D] of each.  Everything that is
    no token is NaN, and table entries that name no block are -1."""
    counts = [-(-n // 16) for n in lens]
    nblk = sum(counts) + extra_blocks
    perm = torch.randperm(nblk, generator=g).tolist()
    kc = torch.full((nblk, Hk, D // 8, 16, 8), NAN, dtype=dtype)
    vc = torch.full((nblk, Hk, D, 16), NAN, dtype=dtype)
    table = torch.full((len(lens), max(max(counts), 1) + 1), -1, dtype=torch.int32)
    ks, vs = [], []
    for i, n in enumerate(lens):
        row = [perm.pop() for _ in range(counts[i])]
        table[i, :len(row)] = torch.tensor(row, dtype=torch.int32)
        k, v = normal(g, dtype, n, Hk, D), normal(g, dtype, n, Hk, D)
        slots = torch.tensor([row[t // 16] * 16 + t % 16 for t in range(n)], dtype=torch.int64)
        W.write_cache(k, v, kc, vc, slots)
        ks.append(k)
        vs.append(v)
    return kc, vc, table, ks, vs


def hide_unseen(kc, vc, table, i, n, seen):
    """NaN into the tokens 0 .. n - 1 of sequence i that nobody sees; -1 into entries of unseen blocks."""
    for t in range(n):
        if t not in seen:
            b, o = int(table[i, t // 16]), t % 16
            kc[b, :, :, o] = NAN
            vc[b, :, :, o] = NAN
    for b in range(-(-n // 16)):
        if not any(t in seen for t in range(16 * b, 16 * b + 16)):
            table[i, b] = -1


def near(got, q, k, v, positions, window, sinks, dtype, scale=SCALE, split=False):
    worst = 0.0
    for r, p in enumerate(positions):
        o, a, n, size = W.attention_row(q[r], k, v, p, window, sinks, scale)
        vmax = float(v[W.visible(p, window, sinks)].abs().max()) if n else 0.0
        bound = W.attention_bound(o, a, n, size, vmax, dtype, split)
        d = (got[r].double() - o).abs()
        assert torch.isfinite(got[r]).all(), (r, p)
        worst = max(worst, float((d / bound).max()))
    assert worst <= 1, worst


# ---- decode -------------------------------------------------------------------------------------------
def decode(dev, q, kc, vc, table, ctx, window, sinks, scale=SCALE):
    out = torch.full((len(ctx), q.shape[1], D), NAN, dtype=q.dtype, device=dev)
    tch_cuda.paged_attention_window(out, q.to(dev), kc.to(dev), vc.to(dev), kc.shape[1], scale, table.to(dev),
                                    torch.tensor(ctx, dtype=torch.int32, device=dev), 16, max(max(ctx), 1), window, sinks)
    return out.cpu()


DECODES = [  # contexts, heads, kv heads, window, sinks
    ([1], 1, 1, 1, 0), ([0], 2, 1, 8, 4), ([16, 17, 15, 0, 1], 8, 2, 16, 0), ([33, 64, 100], 4, 4, 5, 3),
    ([200, 3, 47, 0, 129], 8, 1, 40, 17), ([300], 6, 2, 1, 1), ([500, 77], 16, 1, 100, 50), ([129, 128, 127], 15, 3, 128, 128),
    ([40, 41, 42, 43], 7, 1, 1000, 2), ([1025], 32, 8, 600, 0), ([700, 1, 0, 350], 5, 5, 64, 300), ([90], 24, 2, 33, 4000),
    ([2000, 1999], 12, 1, 1111, 31), ([260] * 40, 4, 1, 70, 4)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ctx,H,Hk,window,sinks", DECODES)
def test_decode(cuda_device, ctx, H, Hk, window, sinks, dtype):
    g = torch.Generator().manual_seed(sum(ctx) + H + window)
    kc, vc, table, ks, vs = paged(g, ctx, Hk, dtype)
    for i, n in enumerate(ctx):
        hide_unseen(kc, vc, table, i, n, set(W.visible(n - 1, window, sinks)))
    q = normal(g, dtype, len(ctx), H, D)
    got = decode(cuda_device, q, kc, vc, table, ctx, window, sinks)
    for i, n in enumerate(ctx):
        near(got[i:i + 1], q[i:i + 1], ks[i], vs[i], [n - 1], window, sinks, dtype, split=True)
    assert _lib.last_status() == 0


def test_decode_many_sequences(cuda_device):
    """More rows than the GPU has places for, some of them empty."""
    r = random.Random(4)
    ctx = [r.choice([0, 1, r.randint(1, 90), 40]) for _ in range(2500)]
    g = torch.Generator().manual_seed(4)
    kc, vc, table, ks, vs = paged(g, ctx, 2, torch.bfloat16)
    q = normal(g, torch.bfloat16, len(ctx), 4, D)
    got = decode(cuda_device, q, kc, vc, table, ctx, 24, 2)
    for i in r.sample(range(len(ctx)), 200) + [0, len(ctx) - 1]:
        near(got[i:i + 1], q[i:i + 1], ks[i], vs[i], [ctx[i] - 1], 24, 2, torch.bfloat16)
    assert _lib.last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_decode_uneven_scores(cuda_device, dtype):
    """One token far above the rest, at either end of the window and among the sinks."""
    g = torch.Generator().manual_seed(9)
    ctx = [400, 400, 400, 400]
    kc, vc, table, ks, vs = paged(g, ctx, 1, dtype)
    q = normal(g, dtype, 4, 4, D)
    for i, t in enumerate((2, 300, 399, 350)):
        ks[i][t] = (q[i, 0] * (6.0 if i else 30.0)).to(dtype)
        W.write_cache(ks[i][t:t + 1], vs[i][t:t + 1], kc, vc, table[i, t // 16:t // 16 + 1].long() * 16 + t % 16)
    got = decode(cuda_device, q, kc, vc, table, ctx, 100, 4)
    for i in range(4):
        near(got[i:i + 1], q[i:i + 1], ks[i], vs[i], [399], 100, 4, dtype, split=True)


def test_decode_strided_queries_and_infinite_masked_tokens(cuda_device):
    dev, dtype = cuda_device, torch.bfloat16
    g = torch.Generator().manual_seed(10)
    ctx = [70, 35]
    kc, vc, table, ks, vs = paged(g, ctx, 2, dtype)
    for i, n in enumerate(ctx):
        seen = set(W.visible(n - 1, 20, 3))
        for t in range(n):
            if t not in seen:
                kc[table[i, t // 16], :, :, t % 16] = float("inf")
                vc[table[i, t // 16], :, :, t % 16] = -float("inf")
    wide = normal(g, dtype, 2, 8 * D + 64)
    q = wide[:, :8 * D].unflatten(1, (8, D))
    out = torch.empty(2, 8, D, dtype=dtype, device=dev)
    wd = wide.to(dev)
    tch_cuda.paged_attention_window(out, wd[:, :8 * D].unflatten(1, (8, D)), kc.to(dev), vc.to(dev), 2, SCALE, table.to(dev),
                                    torch.tensor(ctx, dtype=torch.int32, device=dev), 16, 70, 20, 3)
    for i, n in enumerate(ctx):
        near(out.cpu()[i:i + 1], q[i:i + 1], ks[i], vs[i], [n - 1], 20, 3, dtype)


def test_decode_bad_visible_block_is_reported(cuda_device):
    g = torch.Generator().manual_seed(11)
    kc, vc, table, _, _ = paged(g, [100, 40], 1, torch.bfloat16)
    kc, vc = kc.nan_to_num(0.0), vc.nan_to_num(0.0)
    table[0, 6] = kc.shape[0]
    q = normal(g, torch.bfloat16, 2, 2, D)
    got = decode(cuda_device, q, kc, vc, table, [100, 40], 30, 0)
    assert torch.isfinite(got).all() and _lib.last_status() == 1
    decode(cuda_device, q, kc, vc, table, [100 + 16 * 30, 40], 30, 0)  # longer than its table row
    assert _lib.last_status() == 1


def test_decode_cache_offsets_past_32_bits(cuda_device):
    dev, Hk = cuda_device, 8
    nblk = (1 << 31) // (Hk * D * 16) + 64
    kc = torch.empty(nblk, Hk, D // 8, 16, 8, dtype=torch.bfloat16, device=dev)
    vc = torch.empty(nblk, Hk, D, 16, dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(12)
    k, v, ctx = normal(g, torch.bfloat16, 200, Hk, D), normal(g, torch.bfloat16, 200, Hk, D), 200
    row = torch.arange(nblk - 13, nblk, dtype=torch.int32)
    small_k, small_v = torch.zeros(13, Hk, 16, 16, 8, dtype=torch.bfloat16), torch.zeros(13, Hk, D, 16, dtype=torch.bfloat16)
    W.write_cache(k, v, small_k, small_v, torch.arange(200))
    kc[-13:], vc[-13:] = small_k.to(dev), small_v.to(dev)
    q = normal(g, torch.bfloat16, 1, 16, D)
    out = torch.empty(1, 16, D, dtype=torch.bfloat16, device=dev)
    tch_cuda.paged_attention_window(out, q.to(dev), kc, vc, Hk, SCALE, row.view(1, -1).to(dev),
                                    torch.tensor([ctx], dtype=torch.int32, device=dev), 16, ctx, 90, 2)
    near(out.cpu(), q, k, v, [ctx - 1], 90, 2, torch.bfloat16)
    o2 = tch_cuda.flash_attn_varlen_paged_window(q.to(dev), kc, vc, torch.tensor([0, 1], dtype=torch.int32, device=dev),
                                                 torch.tensor([ctx], dtype=torch.int32, device=dev), row.view(1, -1).to(dev),
                                                 1, ctx, SCALE, 90, 2)
    near(o2.cpu(), q, k, v, [ctx - 1], 90, 2, torch.bfloat16)
    assert _lib.last_status() == 0


def test_decode_two_graphs_at_once(cuda_device):
    """Two captured calls of different batches replayed on two streams: neither disturbs the other."""
    dev, dtype = cuda_device, torch.bfloat16
    jobs = []
    for seed, S, n in ((1, 3, 900), (2, 50, 300)):
        g = torch.Generator().manual_seed(seed)
        ctx = [n - 7 * i % 40 for i in range(S)]
        kc, vc, table, _, _ = paged(g, ctx, 4, dtype)
        q = normal(g, dtype, S, 8, D).to(dev)
        args = (q, kc.to(dev), vc.to(dev), 4, SCALE, table.to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev), 16, n, 500, 4)
        out, ref = torch.empty_like(q), torch.empty_like(q)
        tch_cuda.paged_attention_window(ref, *args)
        stream = torch.cuda.Stream(dev)
        stream.wait_stream(torch.cuda.current_stream(dev))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            tch_cuda.paged_attention_window(out, *args)
        jobs.append((graph, stream, out, ref))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream, out, _ in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, ref in jobs:
        assert torch.equal(out, ref)


def test_results_do_not_depend_on_the_run(cuda_device):
    g = torch.Generator().manual_seed(13)
    ctx = [1500, 20, 700]
    kc, vc, table, _, _ = paged(g, ctx, 2, torch.bfloat16)
    q = normal(g, torch.bfloat16, 3, 8, D)
    a = decode(cuda_device, q, kc, vc, table, ctx, 1200, 4)
    for _ in range(5):
        assert torch.equal(a, decode(cuda_device, q, kc, vc, table, ctx, 1200, 4))


# ---- prefill ------------------------------------------------------------------------------------------
PREFILLS = [  # query lengths, key lengths, heads, kv heads, window, sinks
    ([1], [1], 1, 1, 1, 0), ([5, 0, 1], [5, 0, 9], 2, 1, 3, 1), ([128], [128], 2, 2, 128, 0), ([127, 129], [127, 129], 4, 2, 16, 4),
    ([130], [300], 2, 1, 100, 20), ([300], [300], 3, 1, 1, 0), ([64, 200], [264, 200], 8, 2, 70, 0), ([140], [40], 2, 1, 30, 2),
    ([257], [257], 2, 2, 129, 130), ([100, 3], [1000, 700], 4, 1, 200, 5), ([260], [260], 6, 2, 5000, 0), ([40], [700], 10, 2, 64, 300),
    ([20, 150], [20, 10], 2, 2, 12, 0), ([384], [512], 4, 2, 256, 128), ([1, 1, 1], [600, 17, 128], 5, 1, 33, 1)]


def run_prefill(dev, g, lens_q, lens_k, H, Hk, window, sinks, dtype, is_paged, hide=True):
    seen = []
    for lq, lk in zip(lens_q, lens_k):
        s = set()
        for r in range(lq):
            s |= set(W.visible(lk - lq + r, window, sinks))
        seen.append(s)
    total = sum(lens_q)
    wide = normal(g, dtype, total, H + 3, D)
    q = wide[:, 1:H + 1]
    cu = lambda lens: torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)  # noqa: E731
    wd = wide.to(dev)
    if is_paged:
        kc, vc, table, ks, vs = paged(g, lens_k, Hk, dtype)
        for i, n in enumerate(lens_k):
            if hide:
                hide_unseen(kc, vc, table, i, n, seen[i])
        out = tch_cuda.flash_attn_varlen_paged_window(wd[:, 1:H + 1], kc.to(dev), vc.to(dev), cu(lens_q),
                                                      torch.tensor(lens_k, dtype=torch.int32, device=dev), table.to(dev),
                                                      max(lens_q), max(lens_k), SCALE, window, sinks)
    else:
        ks = [normal(g, dtype, n, Hk, D) for n in lens_k]
        vs = [normal(g, dtype, n, Hk, D) for n in lens_k]
        k2, v2 = [k.clone() for k in ks], [v.clone() for v in vs]
        for i, n in enumerate(lens_k):
            for t in range(n):
                if hide and t not in seen[i]:
                    k2[i][t], v2[i][t] = NAN, NAN
        kv = torch.cat([torch.cat(k2), torch.cat(v2)], 1).to(dev)  # strided keys and values
        out = tch_cuda.flash_attn_varlen_window(wd[:, 1:H + 1], kv[:, :Hk], kv[:, Hk:], cu(lens_q), cu(lens_k), max(lens_q),
                                                max(lens_k), SCALE, window, sinks)
    return out.cpu(), q, ks, vs


@pytest.mark.parametrize("is_paged", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens_q,lens_k,H,Hk,window,sinks", PREFILLS)
def test_prefill(cuda_device, lens_q, lens_k, H, Hk, window, sinks, dtype, is_paged):
    g = torch.Generator().manual_seed(sum(lens_q) * 3 + sum(lens_k) + window)
    out, q, ks, vs = run_prefill(cuda_device, g, lens_q, lens_k, H, Hk, window, sinks, dtype, is_paged)
    at = 0
    for i, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        near(out[at:at + lq], q[at:at + lq], ks[i], vs[i], range(lk - lq, lk), window, sinks, dtype)
        at += lq
    assert _lib.last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens_q,lens_k,H,Hk,window,sinks", [
    ([4], [900], 4, 1, 100, 3), ([16], [300], 2, 2, 7, 0), ([2, 0, 3, 1], [40, 50, 2, 1000], 8, 2, 64, 4), ([8], [8], 2, 1, 3, 1),
    ([16, 5], [700, 3], 1, 1, 10, 0), ([1] * 90, [70 + i for i in range(90)], 16, 1, 33, 17), ([3] * 40, [3 + 7 * i for i in range(40)], 5, 1, 90, 0),
    ([7, 8], [2000, 1990], 4, 2, 1 << 40, 0), ([2], [17], 16, 2, 16, 16), ([9, 16, 1], [500, 20, 800], 15, 3, 64, 5),
    ([300], [1500], 4, 2, 200, 33), ([40, 0, 61], [40, 9, 333], 28, 4, 50, 1), ([16] * 40, [30 + 9 * i for i in range(40)], 24, 8, 75, 2),
    ([33], [2222], 48, 1, 1000, 130), ([2048], [2048], 2, 1, 64, 0)])
def test_prefill_few_rows(cuda_device, lens_q, lens_k, H, Hk, window, sinks, dtype):
    """Chunks of at most 16 tokens, or with all items of 16 rows (tokens x heads of a kv head) resident at once,
    have a form of their own, which carries what rounding a probability left; the others round it."""
    items = len(lens_q) * Hk * -(-max(lens_q) * (H // Hk) // 16)
    split = max(lens_q) <= 16 or items <= 2 * torch.cuda.get_device_properties(cuda_device).multi_processor_count
    g = torch.Generator().manual_seed(sum(lens_k) + window % 1000)
    out, q, ks, vs = run_prefill(cuda_device, g, lens_q, lens_k, H, Hk, window, sinks, dtype, True)
    at = 0
    for i, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        near(out[at:at + lq], q[at:at + lq], ks[i], vs[i], range(lk - lq, lk), window, sinks, dtype, split=split)
        at += lq
    assert _lib.last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens_q,lens_k,H,Hk,window,sinks", [
    ([130, 1, 17, 0, 64], [130, 900, 17, 50, 333], 16, 8, 100, 3), ([300], [300], 24, 24, 1, 0), ([257, 3], [700, 2], 20, 10, 64, 130),
    ([129], [1400], 64, 2, 300, 33), ([140], [1200], 40, 40, 1000, 0), ([200, 150], [900, 2000], 32, 4, 800, 5),
    ([0, 128, 256], [3, 128, 255], 28, 28, 1 << 40, 2), ([60] * 20, [60 + 13 * i for i in range(20)], 8, 4, 129, 1)])
def test_prefill_paged_tiles(cuda_device, lens_q, lens_k, H, Hk, window, sinks, dtype):
    """Chunks too many for the form above: tiles of 128 rows over the paged cache."""
    assert max(lens_q) > 16 and len(lens_q) * Hk * -(-max(lens_q) * (H // Hk) // 16) > 2 * 148
    g = torch.Generator().manual_seed(sum(lens_k) + H)
    out, q, ks, vs = run_prefill(cuda_device, g, lens_q, lens_k, H, Hk, window, sinks, dtype, True)
    at = 0
    for i, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        rows = range(0, lq, 1 if lq < 70 else 3)
        near(out[at:at + lq][list(rows)], q[at:at + lq][list(rows)], ks[i], vs[i], [lk - lq + r for r in rows], window, sinks, dtype)
        at += lq
    assert _lib.last_status() == 0


@pytest.mark.parametrize("is_paged", [False, True])
@pytest.mark.parametrize("lens_q,lens_k,H,Hk,window,sinks", [
    ([2500], [2500], 4, 2, 700, 4), ([300, 900], [3500, 900], 8, 1, 2300, 200), ([700], [4400], 6, 6, 4096, 0),
    ([129], [2700], 3, 1, 1000, 33)])
def test_prefill_long(cuda_device, lens_q, lens_k, H, Hk, window, sinks, is_paged):
    """Long enough for the shapes that long sequences take; a sample of the rows."""
    dtype = torch.float16 if Hk == 1 else torch.bfloat16
    g = torch.Generator().manual_seed(sum(lens_k))
    out, q, ks, vs = run_prefill(cuda_device, g, lens_q, lens_k, H, Hk, window, sinks, dtype, is_paged, hide=len(lens_q) == 1)
    r, at = random.Random(1), 0
    for i, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        rows = sorted(set(r.sample(range(lq), 60) + [0, 1, 127, min(128, lq - 1), lq - 1]))
        near(out[at:at + lq][rows], q[at:at + lq][rows], ks[i], vs[i], [lk - lq + x for x in rows], window, sinks, dtype)
        at += lq
    assert _lib.last_status() == 0


@pytest.mark.parametrize("is_paged", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens_q,lens_k,H,Hk,window,sinks", [
    ([2800, 1], [2900, 2900], 8, 4, 2650, 130), ([700, 90], [3300, 2700], 16, 4, 1 << 40, 0), ([640], [5000], 12, 6, 2560, 1)])
def test_prefill_two_tile_shape(cuda_device, lens_q, lens_k, H, Hk, window, sinks, dtype, is_paged):
    """Windows of more than 2560 keys and an even number of heads to a kv head: two heads' tiles to a CTA."""
    assert min(window + sinks, max(lens_k)) > 2560 and H // Hk % 2 == 0
    assert len(lens_q) * Hk * -(-max(lens_q) * (H // Hk) // 16) > 2 * 148
    g = torch.Generator().manual_seed(sum(lens_k) + H)
    out, q, ks, vs = run_prefill(cuda_device, g, lens_q, lens_k, H, Hk, window, sinks, dtype, is_paged, hide=len(lens_q) == 1)
    r, at = random.Random(2), 0
    for i, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        rows = sorted(set(r.sample(range(lq), min(lq, 30)) + [x for x in (0, 1, 127, 128, lq - 129, lq - 2, lq - 1) if 0 <= x < lq]))
        near(out[at:at + lq][rows], q[at:at + lq][rows], ks[i], vs[i], [lk - lq + x for x in rows], window, sinks, dtype)
        at += lq
    assert _lib.last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(60, 0), (200, 3), (1000, 0)])
def test_prefill_uneven_scores(cuda_device, dtype, window, sinks):
    """Keys that outgrow each other along the sequence and against it, scores up to some hundreds."""
    dev = cuda_device
    g = torch.Generator().manual_seed(window)
    n, H = 520, 2
    for order in (1, -1):
        q, k, v = normal(g, dtype, n, H, D), normal(g, dtype, n, 1, D), normal(g, dtype, n, 1, D)
        by = torch.linspace(0.05, 30, n).view(n, 1, 1)
        by = by if order == 1 else by.flip(0)
        k = (k.float() * by).to(dtype)
        cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
        out = tch_cuda.flash_attn_varlen_window(q.to(dev), k.to(dev), v.to(dev), cu, cu, n, n, SCALE, window, sinks).cpu()
        near(out[::7], q[::7], k, v, range(0, n, 7), window, sinks, dtype)


def test_prefill_with_a_covering_window_is_causal_attention(cuda_device):
    dev, g = cuda_device, torch.Generator().manual_seed(3)
    q, k, v = (normal(g, torch.bfloat16, 700, h, D).to(dev) for h in (8, 2, 2))
    cu = torch.tensor([0, 300, 700], dtype=torch.int32, device=dev)
    a = tch_cuda.flash_attn_varlen_window(q, k, v, cu, cu, 400, 400, SCALE, 1 << 40).float()
    b = tch_cuda.flash_attn_varlen(q, k, v, cu, cu, 400, 400, SCALE, True).float()
    # both are within half a step of the output and one of each probability of the exact result
    assert float((a - b).abs().max()) <= 4 * 2.0 ** -8 * float(v.float().abs().max())


@pytest.mark.parametrize("is_paged", [False, True])
@pytest.mark.parametrize("window,sinks,offset", [(100, 0, 0), (128, 4, 37), (300, 20, 128)])
def test_prefill_tiles_that_do_not_see_a_token_do_not_meet_it(cuda_device, window, sinks, offset, is_paged):
    """NaN in one token: query tiles of 128 rows none of which sees it stay right."""
    dev, dtype, n, H = cuda_device, torch.bfloat16, 520, 2
    for bad in (0, 3, 19, 21, 130, 255, 256, 300, 511):
        g = torch.Generator().manual_seed(bad)
        lens_k = [n + offset]
        kc, vc, table, ks, vs = paged(g, lens_k, 1, dtype)
        q, k, v = normal(g, dtype, n, H, D), ks[0].clone(), vs[0].clone()
        k[bad], v[bad] = NAN, NAN
        kc[table[0, bad // 16], :, :, bad % 16] = NAN
        vc[table[0, bad // 16], :, :, bad % 16] = NAN
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        if is_paged:
            out = tch_cuda.flash_attn_varlen_paged_window(q.to(dev), kc.to(dev), vc.to(dev), i32([0, n]), i32(lens_k),
                                                          table.to(dev), n, n + offset, SCALE, window, sinks).cpu()
        else:
            out = tch_cuda.flash_attn_varlen_window(q.to(dev), k.to(dev), v.to(dev), i32([0, n]), i32([0, n + offset]), n,
                                                    n + offset, SCALE, window, sinks).cpu()
        for r0 in range(0, n, 128):
            rows = range(r0, min(r0 + 128, n))
            if not any(bad in W.visible(offset + r, window, sinks) for r in (rows[0], rows[-1], max(rows[0], min(rows[-1], bad - offset)))):
                some = [rows[0], rows[len(rows) // 2], rows[-1]]
                near(out[some], q[some], ks[0], vs[0], [offset + r for r in some], window, sinks, dtype)
    assert _lib.last_status() == 0


def test_prefill_of_single_tokens_is_decode(cuda_device):
    dev, dtype = cuda_device, torch.float16
    g = torch.Generator().manual_seed(14)
    ctx = [600, 17, 128, 1]
    kc, vc, table, ks, vs = paged(g, ctx, 2, dtype)
    q = normal(g, dtype, 4, 8, D)
    got = decode(dev, q, kc, vc, table, ctx, 100, 4)
    out = tch_cuda.flash_attn_varlen_paged_window(q.to(dev), kc.to(dev), vc.to(dev), torch.arange(5, dtype=torch.int32, device=dev),
                                                  torch.tensor(ctx, dtype=torch.int32, device=dev), table.to(dev), 1, 600,
                                                  SCALE, 100, 4).cpu()
    for i, n in enumerate(ctx):
        for o in (got, out):
            near(o[i:i + 1], q[i:i + 1], ks[i], vs[i], [n - 1], 100, 4, dtype)


def test_rows_behind_the_last_sequence_stay(cuda_device):
    """A batch padded for a captured step: query rows that no sequence owns are not written."""
    dev, g = cuda_device, torch.Generator().manual_seed(15)
    q, k, v = (normal(g, torch.bfloat16, 200, 2, D).to(dev) for _ in range(3))
    cu = torch.tensor([0, 130, 130], dtype=torch.int32, device=dev)
    L, p = _lib.lib(), lambda t: t.data_ptr()  # noqa: E731
    out = torch.full_like(q, 7.0)
    _lib.check("x", L.aici_mha_varlen_window_fwd(
        p(out), p(q), p(k), p(v), p(cu), p(cu), 2, 200, 200, 2, 2, D, 130, 130, 50, 0, *[256, 128] * 4, SCALE, 0,
        torch.cuda.current_stream().cuda_stream))
    near(out[:130].cpu(), q[:130].cpu(), k.cpu(), v.cpu(), range(130), 50, 0, torch.bfloat16)
    assert (out[130:] == 7.0).all()


@pytest.mark.parametrize("is_paged", [False, True])
@pytest.mark.parametrize("lens_q", [
    [3] * 40 + [700] + [0] * 5, [0, 0, 290] + [1, 0, 130] * 12, [900] + [17] * 31, [128] * 3 + [5] * 70 + [513] + [0] * 1000 + [129],
    [0] * 31 + [400]], ids=["long_in_the_middle", "empty_ones", "long_first", "a_thousand_empty", "long_last"])
def test_prefill_ragged_batches(cuda_device, lens_q, is_paged):
    """Batches in which one sequence has many more tiles than the others; the rows at the tiles' ends."""
    dtype, H, Hk, window, sinks = torch.bfloat16, 12, 6, 70, 3
    g = torch.Generator().manual_seed(len(lens_q))
    lens_k = [lq + i % 50 for i, lq in enumerate(lens_q)]
    out, q, ks, vs = run_prefill(cuda_device, g, lens_q, lens_k, H, Hk, window, sinks, dtype, is_paged)
    at = 0
    for i, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        rows = [r for r in range(lq) if r % 128 in (0, 1, 40, 127) or r == lq - 1]
        if rows:
            near(out[at:at + lq][rows], q[at:at + lq][rows], ks[i], vs[i], [lk - lq + r for r in rows], window, sinks, dtype)
        at += lq
    assert _lib.last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens_q,lens_k,H,Hk,window,sinks", [
    ([1] * 20 + [300], [37 * i + 1 for i in range(20)] + [900], 16, 4, 90, 2), ([0, 16, 17, 1, 600], [9, 500, 17, 1, 640], 24, 12, 130, 0),
    ([257] + [1] * 40, [257] + [11 * i + 3 for i in range(40)], 8, 8, 1 << 40, 0), ([2] * 7 + [400, 0], [3000 + i for i in range(7)] + [400, 7], 40, 8, 1000, 9),
    ([500, 3, 16, 0, 1], [2, 3, 10, 5, 1], 64, 4, 20, 1)])
def test_prefill_mixed_batches(cuda_device, lens_q, lens_k, H, Hk, window, sinks, dtype):
    """Steps of single tokens and chunks: sequences of at most 16 tokens take one form, the others another."""
    assert 2 * sum(lens_q) < len(lens_q) * max(lens_q) or sum(lens_q) < 17 * (len(lens_q) - 1) + max(lens_q)
    assert len(lens_q) * Hk * -(-max(lens_q) * (H // Hk) // 16) > 2 * 148
    g = torch.Generator().manual_seed(sum(lens_k) + H)
    out, q, ks, vs = run_prefill(cuda_device, g, lens_q, lens_k, H, Hk, window, sinks, dtype, True)
    at = 0
    for i, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        rows = [r for r in range(lq) if lq < 20 or r % 7 == 0 or r % 128 in (0, 127) or r == lq - 1]
        if rows:
            near(out[at:at + lq][rows], q[at:at + lq][rows], ks[i], vs[i], [lk - lq + r for r in rows], window, sinks, dtype,
                 split=lq <= 16)
        at += lq
    assert _lib.last_status() == 0


@pytest.mark.parametrize("lens_q", [[1] * 50 + [900], [1] * 50 + [0]])
def test_mixed_batches_end_before_what_follows(cuda_device, lens_q):
    """The two launches of a mixed step overlap: what comes behind them, on the stream or in a captured graph, sees
    the rows of both, and the inputs may be written again.  (The second batch leaves the later launch nothing.)"""
    dev, dtype, H, Hk = cuda_device, torch.bfloat16, 8, 2
    g = torch.Generator().manual_seed(21)
    lens_k = [2500 if lq < 2 else lq for lq in lens_q]
    kc, vc, table, _, _ = (x.to(dev) if torch.is_tensor(x) else x for x in paged(g, lens_k, Hk, dtype))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cu, ctx, total = i32([sum(lens_q[:i]) for i in range(len(lens_q) + 1)]), i32(lens_k), sum(lens_q)
    qs = [normal(g, dtype, total, H, D).to(dev) for _ in range(4)]
    q, got = qs[0].clone(), torch.zeros(4, total, H, D, dtype=dtype, device=dev)
    call = lambda x: tch_cuda.flash_attn_varlen_paged_window(x, kc, vc, cu, ctx, table, 900, 2500, SCALE, 2000, 4)  # noqa: E731
    want = []
    for x in qs:
        want.append(call(x))
        torch.cuda.synchronize()
    def steps():
        for i, x in enumerate(qs):
            q.copy_(x)
            got[i].copy_(call(q))
            q.fill_(NAN)
    for _ in range(5):
        got.zero_()
        steps()
        assert torch.equal(got, torch.stack(want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps()
    for _ in range(5):
        got.zero_()
        graph.replay()
        assert torch.equal(got, torch.stack(want))
    assert torch.isfinite(got).all() and _lib.last_status() == 0


def test_mixed_batches_see_what_came_before(cuda_device):
    """Lengths, block tables, queries and caches written by the kernels right before the call, at the same addresses
    with other contents each time."""
    dev, dtype, H, Hk, B = cuda_device, torch.bfloat16, 8, 2, 40
    g = torch.Generator().manual_seed(22)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    sets = []
    for s in range(4):
        lens_q = [1] * B
        lens_q[7 * s] = 700 - s
        lens_k = [900 + 13 * s + i for i in range(B)]
        kc, vc, table, _, _ = paged(g, [1000] * B, Hk, dtype)
        cu = i32([sum(lens_q[:i]) for i in range(B + 1)])
        sets.append([x.to(dev) for x in (normal(g, dtype, 739, H, D), kc, vc, cu, i32(lens_k), table)])
    call = lambda x: tch_cuda.flash_attn_varlen_paged_window(*x, 700, 1000, SCALE, 500, 4)  # noqa: E731
    want = []
    for x in sets:
        want.append(call(x)[:int(x[3][-1])].clone())
        torch.cuda.synchronize()
    now, got = [x.clone() for x in sets[0]], torch.zeros(4, 739, H, D, dtype=dtype, device=dev)
    def steps():
        for i, x in enumerate(sets):
            for a, b in zip(now, x):
                a.copy_(b)
            got[i].copy_(call(now))
    def check():
        for i, w in enumerate(want):
            assert torch.equal(got[i, :len(w)], w), i
    for _ in range(5):
        steps()
        check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps()
    for _ in range(10):
        got.zero_()
        graph.replay()
        check()
    assert _lib.last_status() == 0


def test_sizes_as_other_integers(cuda_device):
    """Sizes that come out of a tensor or an array."""
    dev, g = cuda_device, torch.Generator().manual_seed(16)
    q, k = normal(g, torch.bfloat16, 40, 2, D), normal(g, torch.bfloat16, 40, 2, D)
    cu = torch.tensor([0, 40], dtype=torch.int32, device=dev)
    out = tch_cuda.flash_attn_varlen_window(q.to(dev), k.to(dev), k.to(dev), cu, cu, cu.max(), cu[-1], SCALE, torch.tensor(9),
                                            torch.tensor(2)).cpu()
    near(out, q, k, k, range(40), 9, 2, torch.bfloat16)


def test_refuses_mismatched_tensors(cuda_device):
    dev = cuda_device
    q, i = torch.zeros(4, 2, D, dtype=torch.bfloat16, device=dev), torch.tensor([0, 4], dtype=torch.int32, device=dev)
    f = lambda **c: tch_cuda.flash_attn_varlen_window(**{**dict(  # noqa: E731
        q=q, k=q, v=q, seqlens_q=i, seqlens_k=i, max_seqlen_q=4, max_seqlen_k=4, softmax_scale=1.0, window=4), **c})
    for change, match in ((dict(k=q.half()), "same dtype"), (dict(v=q[:3]), "k and v"), (dict(seqlens_q=i.long()), "seqlens_q"),
                          (dict(seqlens_k=i[:1]), "seqlens_k"), (dict(q=q.float(), k=q.float(), v=q.float()), "only bf16 and f16"),
                          (dict(q=q.transpose(1, 2)), "contiguous last"), (dict(window=0), "window"), (dict(sinks=-1), "sinks"),
                          (dict(window=5 - (1 << 32)), "window"), (dict(sinks=-(1 << 40)), "sinks")):
        with pytest.raises(_lib.AiciError, match=match):
            f(**change)
    f()


def into(out, dev, q, kv, lens_q, lens_k, max_q, window, sinks, table=None, total=None, cu_q=None):
    """A windowed prefill through the C ABI into a buffer that is there before: `kv` is (keys, values) of the
    packed form, or the caches where there is a table."""
    p = lambda t: t.data_ptr()  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    sums = lambda lens: [sum(lens[:i]) for i in range(len(lens) + 1)]  # noqa: E731
    L, H, (a, b) = _lib.lib(), q.shape[1], kv
    cu = i32(cu_q or sums(lens_q))
    total, dt, s = total or q.shape[0], 0 if q.dtype == torch.bfloat16 else 1, torch.cuda.current_stream().cuda_stream
    if table is None:
        ck, Hk = i32(sums(lens_k)), a.shape[1]
        _lib.check("x", L.aici_mha_varlen_window_fwd(
            p(out), p(q), p(a), p(b), p(cu), p(ck), len(lens_q), total, a.shape[0], H, Hk, D, max_q, max(lens_k), window, sinks,
            H * D, D, Hk * D, D, Hk * D, D, H * D, D, SCALE, dt, s))
    else:
        ck, Hk = i32(lens_k), a.shape[1]
        _lib.check("x", L.aici_mha_varlen_paged_window_fwd(
            p(out), p(q), p(a), p(b), p(cu), p(ck), p(table), len(lens_q), total, H, Hk, D, 16, max_q, max(lens_k),
            table.shape[1], a.shape[0], window, sinks, H * D, D, H * D, D, a.stride(0), a.stride(1), SCALE, dt, s))
    torch.cuda.synchronize()


LIES = [  # paged, query lengths, the stated longest, heads, kv heads
    (False, [40, 300, 64], 130, 4, 2), (False, [300] + [5] * 9, 140, 4, 2), (False, [200] + [5] * 40, 140, 2, 2),
    (True, [3, 20, 1], 8, 4, 2), (True, [50, 90], 60, 2, 1), (True, [9, 2], 1, 24, 1), (True, [40, 300, 64], 130, 32, 32),
    (True, [1] * 20 + [300, 400], 300, 16, 4), (True, [17] + [1] * 40, 16, 8, 8)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("is_paged,lens_q,stated,H,Hk", LIES)
def test_prefill_of_a_sequence_longer_than_stated(cuda_device, is_paged, lens_q, stated, H, Hk, dtype):
    """Whatever form the call takes, the sequence's rows are zero and the status says so; the others are right."""
    dev, g = cuda_device, torch.Generator().manual_seed(sum(lens_q) + H)
    lens_k = [lq + 11 for lq in lens_q]
    q = normal(g, dtype, sum(lens_q), H, D)
    if is_paged:
        kc, vc, table, ks, vs = paged(g, lens_k, Hk, dtype)
        kv, table = (kc.to(dev), vc.to(dev)), table.to(dev)
    else:
        ks, vs = ([normal(g, dtype, n, Hk, D) for n in lens_k] for _ in range(2))
        kv, table = (torch.cat(ks).to(dev), torch.cat(vs).to(dev)), None
    out = torch.full_like(q, 7.0).to(dev)
    into(out, dev, q.to(dev), kv, lens_q, lens_k, stated, 50, 2, table)
    out, at = out.cpu(), 0
    for i, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        if lq > stated:
            assert not out[at:at + lq].any(), i
        else:
            near(out[at:at + lq], q[at:at + lq], ks[i], vs[i], range(lk - lq, lk), 50, 2, dtype)
        at += lq
    assert _lib.last_status() == 1


def test_prefill_of_no_tokens_gives_zeros(cuda_device):
    """A longest length of 0 over a padded tensor of rows: nobody's rows come back as zeros, not as what the memory held."""
    dev = cuda_device
    q = torch.full((40, 4, D), 7.0, dtype=torch.bfloat16, device=dev)
    cu, ctx, table = (torch.zeros(*s, dtype=torch.int32, device=dev) for s in ((3,), (2,), (2, 4)))
    kc, vc = torch.zeros(4, 2, 16, 16, 8, dtype=q.dtype, device=dev), torch.zeros(4, 2, D, 16, dtype=q.dtype, device=dev)
    for _ in range(3):
        junk = torch.full_like(q, 7.0)
        del junk
        assert not tch_cuda.flash_attn_varlen_window(q, q[:, :2], q[:, :2], cu, cu, 0, 0, SCALE, 9).any()
        assert not tch_cuda.flash_attn_varlen_paged_window(q, kc, vc, cu, ctx, table, 0, 0, SCALE, 9).any()
    assert _lib.last_status() == 0


@pytest.mark.parametrize("ends", ["behind", "before", "both"])
@pytest.mark.parametrize("is_paged,lens_q,H,Hk", [
    (False, [40, 90], 4, 2), (False, [140] + [3] * 12 + [90], 4, 2), (False, [140] + [3] * 45 + [90], 2, 2), (True, [3, 12], 4, 2),
    (True, [40, 90], 32, 32), (True, [1] * 20 + [300, 90], 16, 4)])
def test_prefill_rows_outside_the_query_tensor_are_not_touched(cuda_device, is_paged, lens_q, H, Hk, ends):
    """Running sums that begin before the tensor's first row or end behind its last: the buffer around the
    output stays, the status says so, and the sequences inside are right."""
    dev, dtype, around = cuda_device, torch.bfloat16, 200
    g = torch.Generator().manual_seed(sum(lens_q) + H)
    lens_k = [lq + 11 for lq in lens_q]
    cut0, cut1 = (0 if ends == "behind" else 2), (0 if ends == "before" else 5)
    if cut0:
        lens_q, lens_k = [30] + lens_q, [41] + lens_k
    cu = [sum(lens_q[:i]) - cut0 for i in range(len(lens_q) + 1)]
    total = cu[-1] - cut1
    q = normal(g, dtype, around + total + around, H, D)
    if is_paged:
        kc, vc, table, ks, vs = paged(g, lens_k, Hk, dtype)
        kv, table = (kc.to(dev), vc.to(dev)), table.to(dev)
    else:
        ks, vs = ([normal(g, dtype, n, Hk, D) for n in lens_k] for _ in range(2))
        kv, table = (torch.cat(ks).to(dev), torch.cat(vs).to(dev)), None
    out, qd = torch.full_like(q, 7.0).to(dev), q.to(dev)
    into(out[around:], dev, qd[around:], kv, lens_q, lens_k, max(lens_q), 50, 2, table, total=total, cu_q=cu)
    out = out.cpu()
    assert (out[:around] == 7).all() and (out[around + total:] == 7).all()
    out, q = out[around:around + total], q[around:around + total]
    for i, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        if cu[i] >= 0 and cu[i + 1] <= total:
            near(out[cu[i]:cu[i + 1]], q[cu[i]:cu[i + 1]], ks[i], vs[i], range(lk - lq, lk), 50, 2, dtype)
    assert _lib.last_status() == 1


@pytest.mark.parametrize("most", [1 << 31, 1 << 32, (1 << 32) + 5, 1 << 40])
def test_longest_lengths_beyond_32_bits(cuda_device, most):
    """A stated longest length may be any bound."""
    dev, dtype = cuda_device, torch.bfloat16
    g = torch.Generator().manual_seed(17)
    lens = [70, 200, 16]
    kc, vc, table, ks, vs = paged(g, lens, 2, dtype)
    q = normal(g, dtype, 286, 4, D)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cu, ctx, qd, k, v = i32([0, 70, 270, 286]), i32(lens), q.to(dev), torch.cat(ks).to(dev), torch.cat(vs).to(dev)
    outs = [tch_cuda.flash_attn_varlen_window(qd, k, v, cu, cu, most, most, SCALE, 30, 2).cpu(),
            tch_cuda.flash_attn_varlen_paged_window(qd, kc.to(dev), vc.to(dev), cu, ctx, table.to(dev), most, most, SCALE, 30, 2).cpu()]
    for i, (a, b) in enumerate(((0, 70), (70, 270), (270, 286))):
        for out in outs:
            near(out[a:b], q[a:b], ks[i], vs[i], range(b - a), 30, 2, dtype)
    out = torch.empty(3, 4, D, dtype=dtype, device=dev)
    tch_cuda.paged_attention_window(out, qd[:3], kc.to(dev), vc.to(dev), 2, SCALE, table.to(dev), ctx, 16, most, 30, 2)
    for i, n in enumerate(lens):
        near(out.cpu()[i:i + 1], q[i:i + 1], ks[i], vs[i], [n - 1], 30, 2, dtype)
    assert _lib.last_status() == 0


@pytest.mark.parametrize("stride", [1, 128, 1001])
def test_a_single_row_has_no_stride(cuda_device, stride):
    """One query token (or one key) whose first stride is what is left of another layout."""
    dev, dtype, H, Hk = cuda_device, torch.float16, 6, 2
    g = torch.Generator().manual_seed(18)
    kc, vc, table, ks, vs = paged(g, [50], Hk, dtype)
    q, k1, v1 = normal(g, dtype, 1, H, D), ks[0][-1:], vs[0][-1:]
    odd = lambda x: x.to(dev).as_strided(x.shape, (stride, D, 1))  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    assert odd(q).is_contiguous() and odd(q).stride(0) == stride
    out = torch.empty(1, H, D, dtype=dtype, device=dev)
    tch_cuda.paged_attention_window(out, odd(q), kc.to(dev), vc.to(dev), Hk, SCALE, table.to(dev), i32([50]), 16, 50, 20, 2)
    near(out.cpu(), q, ks[0], vs[0], [49], 20, 2, dtype)
    out = tch_cuda.flash_attn_varlen_paged_window(odd(q), kc.to(dev), vc.to(dev), i32([0, 1]), i32([50]), table.to(dev), 1, 50,
                                                  SCALE, 20, 2).cpu()
    near(out, q, ks[0], vs[0], [49], 20, 2, dtype)
    out = tch_cuda.flash_attn_varlen_window(odd(q), odd(k1), odd(v1), i32([0, 1]), i32([0, 1]), 1, 1, SCALE, 20, 2).cpu()
    near(out, q, k1, v1, [0], 20, 2, dtype)
    assert _lib.last_status() == 0


@pytest.mark.parametrize("H", [20, 2], ids=["tiles", "items"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks,offset", [(100, 0, 0), (128, 4, 37), (300, 20, 128)])
def test_paged_tiles_that_do_not_see_a_token_do_not_meet_it(cuda_device, window, sinks, offset, dtype, H):
    """NaN in one token of the cache that some rows see: with 20 heads the call takes tiles of 128 rows, with 2 items
    of 16, and those none of whose rows sees it stay right."""
    dev, n, rows_each = cuda_device, 520, 128 if H == 20 else 16
    assert (H * -(-n // 16) > 2 * 148) == (H == 20)
    for bad in (0, 3, 19, 21, 130, 255, 256, 300, 511):
        g = torch.Generator().manual_seed(bad)
        kc, vc, table, ks, vs = paged(g, [n + offset], H, dtype)
        q = normal(g, dtype, n, H, D)
        kc[table[0, bad // 16], :, :, bad % 16] = NAN
        vc[table[0, bad // 16], :, :, bad % 16] = NAN
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        out = tch_cuda.flash_attn_varlen_paged_window(q.to(dev), kc.to(dev), vc.to(dev), i32([0, n]), i32([n + offset]),
                                                      table.to(dev), n, n + offset, SCALE, window, sinks).cpu()
        kept = 0
        for r0 in range(0, n, rows_each):
            rows = range(r0, min(r0 + rows_each, n))
            if not any(bad in W.visible(offset + r, window, sinks) for r in rows):
                some = [rows[0], rows[len(rows) // 2], rows[-1]]
                near(out[some], q[some], ks[0], vs[0], [offset + r for r in some], window, sinks, dtype, split=H == 2)
                kept += 1
        assert kept >= (0 if bad < sinks else 1)
    assert _lib.last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(60, 0), (200, 3), (1000, 0)])
def test_paged_tiles_uneven_scores(cuda_device, dtype, window, sinks):
    """Keys of the cache that outgrow each other along the sequence and against it, in tiles of 128 rows."""
    dev, n, H, Hk = cuda_device, 520, 20, 10
    assert Hk * -(-n * 2 // 16) > 2 * 148
    for order in (1, -1):
        g = torch.Generator().manual_seed(window + order)
        kc, vc, table, ks, vs = paged(g, [n], Hk, dtype)
        by = torch.linspace(0.05, 30, n).view(n, 1, 1)
        k = (ks[0].float() * (by if order == 1 else by.flip(0))).to(dtype)
        W.write_cache(k, vs[0], kc, vc, torch.tensor([int(table[0, t // 16]) * 16 + t % 16 for t in range(n)]))
        q, i32 = normal(g, dtype, n, H, D), lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        out = tch_cuda.flash_attn_varlen_paged_window(q.to(dev), kc.to(dev), vc.to(dev), i32([0, n]), i32([n]), table.to(dev), n, n,
                                                      SCALE, window, sinks).cpu()
        near(out[::9], q[::9], k, vs[0], range(0, n, 9), window, sinks, dtype)
    assert _lib.last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["decode", "items", "paged tiles", "packed tiles"])
def test_the_error_is_that_of_its_roundings(cuda_device, form, dtype):
    """Root mean square over many rows.  A rounding's error is spread evenly over half a step u either way, so its
    square is u^2 / 3 of the value's on average at most: one for the output, and where a probability is rounded
    once (the tiles), one for each product p v.  Five per cent for fp32 sums, exp2 and chance."""
    dev, g, window, sinks, H, Hk = cuda_device, torch.Generator().manual_seed(30), 200, 4, 20, 10
    lens_q = {"decode": [1] * 60, "items": [10] * 12, "paged tiles": [520], "packed tiles": [520]}[form]
    lens_k = [lq + 190 + 7 * i for i, lq in enumerate(lens_q)]
    if form == "decode":
        kc, vc, table, ks, vs = paged(g, lens_k, Hk, dtype)
        q = normal(g, dtype, 60, H, D)
        out = decode(dev, q, kc, vc, table, lens_k, window, sinks)
    else:
        out, q, ks, vs = run_prefill(dev, g, lens_q, lens_k, H, Hk, window, sinks, dtype, form != "packed tiles")
    step, at, err, size, parts, count = torch.finfo(dtype).eps / 2, 0, 0.0, 0.0, 0.0, 0
    for i, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        for r in range(0, lq, 1 if lq < 20 else 7):
            seen = W.visible(lk - lq + r, window, sinks)
            kk, vv = ks[i][seen].double(), vs[i][seen].double()
            p = torch.softmax(torch.einsum("hgd,thd->hgt", q[at + r].double().view(Hk, H // Hk, D), kk) * SCALE, -1)
            o = torch.einsum("hgt,thd->hgd", p, vv).reshape(H, D)
            err += float((out[at + r].double() - o).square().sum())
            size += float(o.square().sum())
            parts += float(torch.einsum("hgt,thd->hgd", p.square(), vv.square()).sum())
            count += o.numel()
        at += lq
    assert count >= 60 * H * D
    bound = step / math.sqrt(3) * math.sqrt(size + (parts if "tiles" in form else 0.0)) * 1.05
    assert math.sqrt(err) <= bound, math.sqrt(err) / bound


@pytest.mark.parametrize("dtype", TYPES)
def test_paged_tiles_cache_offsets_past_32_bits(cuda_device, dtype):
    """Tiles of 128 rows over the last blocks of a pool of more than 2^31 elements."""
    dev, H, Hk, n = cuda_device, 16, 8, 330
    assert Hk * -(-n * 2 // 16) > 2 * 148
    nblk = (1 << 31) // (Hk * D * 16) + 64
    kc = torch.empty(nblk, Hk, D // 8, 16, 8, dtype=dtype, device=dev)
    vc = torch.empty(nblk, Hk, D, 16, dtype=dtype, device=dev)
    g = torch.Generator().manual_seed(19)
    k, v, q = normal(g, dtype, n, Hk, D), normal(g, dtype, n, Hk, D), normal(g, dtype, n, H, D)
    row = torch.arange(nblk - 21, nblk, dtype=torch.int32)
    small_k, small_v = torch.zeros(21, Hk, 16, 16, 8, dtype=dtype), torch.zeros(21, Hk, D, 16, dtype=dtype)
    W.write_cache(k, v, small_k, small_v, torch.arange(n))
    kc[-21:], vc[-21:] = small_k.to(dev), small_v.to(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    out = tch_cuda.flash_attn_varlen_paged_window(q.to(dev), kc, vc, i32([0, n]), i32([n]), row.view(1, -1).to(dev), n, n, SCALE,
                                                  90, 2).cpu()
    near(out[::5], q[::5], k, v, range(0, n, 5), 90, 2, dtype)
    assert _lib.last_status() == 0


@pytest.mark.parametrize("lens_q", [[60000, 60000], [130, 119300, 570]], ids=["even", "ragged"])
def test_prefill_rows_past_32_bits(cuda_device, lens_q):
    """Queries, keys and values as slices of rows so wide that the last tokens lie more than 2^31 elements behind the first."""
    dev, dtype, H, Hk, width, window, sinks = cuda_device, torch.bfloat16, 2, 1, 150, 20, 1
    total = sum(lens_q)
    assert (total - 1000) * width * D > 1 << 31
    wide = torch.zeros(total, width, D, dtype=dtype, device=dev)
    wide[:, -4:] = torch.randn(total, 4, D, device=dev, generator=torch.Generator(dev).manual_seed(20)).to(dtype)
    q, k, v = wide[:, -4:-2], wide[:, -2:-1], wide[:, -1:]
    cu = torch.tensor([sum(lens_q[:i]) for i in range(len(lens_q) + 1)], dtype=torch.int32, device=dev)
    out = tch_cuda.flash_attn_varlen_window(q, k, v, cu, cu, max(lens_q), max(lens_q), SCALE, window, sinks).cpu()
    q, k, v, at = q.cpu(), k.cpu(), v.cpu(), 0
    for n in lens_q:
        rows = [0, 1, n // 2, n - 130, n - 2, n - 1]
        for r in rows:  # the definition sees the sinks and the last tokens only
            seen = W.visible(r, window, sinks)
            near(out[at + r:at + r + 1], q[at + r:at + r + 1], k[at:at + n][seen], v[at:at + n][seen], [len(seen) - 1], 1 << 30, 0, dtype)
        at += n
    assert _lib.last_status() == 0


def test_calls_from_several_threads_on_one_stream(cuda_device):
    """Mixed steps, whose two launches may then lie apart on the stream, and decode calls between them."""
    import threading
    dev, dtype, H, Hk = cuda_device, torch.bfloat16, 8, 2
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    jobs = []
    for s in range(4):
        g = torch.Generator().manual_seed(40 + s)
        lens_q = [1] * 40 + [500 + s]
        lens_k = [700 + 13 * s + i for i in range(40)] + [600]
        kc, vc, table, _, _ = (x.to(dev) if torch.is_tensor(x) else x for x in paged(g, lens_k, Hk, dtype))
        q, cu, ctx = normal(g, dtype, 540 + s, H, D).to(dev), i32(list(range(41)) + [540 + s]), i32(lens_k)
        def mixed(q=q, kc=kc, vc=vc, cu=cu, ctx=ctx, table=table):
            return tch_cuda.flash_attn_varlen_paged_window(q, kc, vc, cu, ctx, table, 510, 800, SCALE, 300, 4)
        def single(q=q, kc=kc, vc=vc, ctx=ctx, table=table):
            out = torch.empty(41, H, D, dtype=dtype, device=dev)
            tch_cuda.paged_attention_window(out, q[:41], kc, vc, Hk, SCALE, table, ctx, 16, 800, 300, 4)
            return out
        jobs.append((mixed, mixed()) if s % 2 == 0 else (lambda a=mixed, b=single: torch.cat([a(), b()]), torch.cat([mixed(), single()])))
    torch.cuda.synchronize()
    wrong = []
    def work(call, want):
        for _ in range(60):
            if not torch.equal(call(), want):
                wrong.append(want.shape)
    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and _lib.last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk", [(17, 1), (48, 1), (96, 2)])
def test_single_tokens_of_larger_groups(cuda_device, H, Hk, dtype):
    """More than 16 query heads to a kv head, which the decode call refuses: the paged prefill with one token a sequence."""
    g, lens = torch.Generator().manual_seed(H), [1, 700, 16, 129]
    out, q, ks, vs = run_prefill(cuda_device, g, [1] * 4, lens, H, Hk, 100, 5, dtype, True)
    for i, n in enumerate(lens):
        near(out[i:i + 1], q[i:i + 1], ks[i], vs[i], [n - 1], 100, 5, dtype, split=True)
    assert _lib.last_status() == 0


FORMS = [(False, [40, 90], 4, 2), (False, [140] + [3] * 12 + [90], 4, 2), (True, [3, 0, 12], 4, 2), (True, [40, 90], 32, 32),
         (True, [1] * 20 + [300, 90], 16, 4)]  # paged, query lengths, heads, kv heads: each form of a call


def batch(g, dev, dtype, is_paged, lens_q, H, Hk, extra):
    """Queries with `extra` rows behind the last sequence, keys and values on the device, and the tokens."""
    lens_k = [lq + 11 for lq in lens_q]
    q = normal(g, dtype, sum(lens_q) + extra, H, D)
    if is_paged:
        kc, vc, table, ks, vs = paged(g, lens_k, Hk, dtype)
        return lens_k, q, (kc.to(dev), vc.to(dev)), table.to(dev), ks, vs
    ks, vs = ([normal(g, dtype, n, Hk, D) for n in lens_k] for _ in range(2))
    return lens_k, q, (torch.cat(ks).to(dev), torch.cat(vs).to(dev)), None, ks, vs


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("is_paged,lens_q,H,Hk", FORMS)
def test_padding_rows_stay_and_do_no_harm(cuda_device, is_paged, lens_q, H, Hk, dtype):
    """A batch padded for a captured step: NaN in the query rows that no sequence owns, whose output rows stay."""
    dev, g, total = cuda_device, torch.Generator().manual_seed(sum(lens_q)), sum(lens_q)
    lens_k, q, kv, table, ks, vs = batch(g, dev, dtype, is_paged, lens_q, H, Hk, 77)
    q[total:] = NAN
    out = torch.full_like(q, 7.0).to(dev)
    into(out, dev, q.to(dev), kv, lens_q, lens_k, max(lens_q), 50, 2, table)
    out, at = out.cpu(), 0
    assert (out[total:] == 7).all()
    for i, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        near(out[at:at + lq], q[at:at + lq], ks[i], vs[i], range(lk - lq, lk), 50, 2, dtype)
        at += lq
    assert _lib.last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("is_paged,lens_q,H,Hk", FORMS)
def test_a_query_row_of_nan_stays_alone(cuda_device, is_paged, lens_q, H, Hk, dtype):
    dev, g = cuda_device, torch.Generator().manual_seed(sum(lens_q) + 1)
    lens_k, q, kv, table, ks, vs = batch(g, dev, dtype, is_paged, lens_q, H, Hk, 0)
    bad = [(1, 0), (sum(lens_q) - 4, H - 1), (sum(lens_q) // 2, 1)]
    for row, head in bad:
        q[row, head, 5] = NAN
    out = torch.full_like(q, 7.0).to(dev)
    into(out, dev, q.to(dev), kv, lens_q, lens_k, max(lens_q), 50, 2, table)
    out, at = out.cpu(), 0
    for row, head in bad:
        assert torch.isnan(out[row, head]).all()
        q[row, head] = 0  # the definition of a row of zeros in its place
        seq = next(i for i in range(len(lens_q)) if sum(lens_q[:i + 1]) > row)
        pos = lens_k[seq] - lens_q[seq] + row - sum(lens_q[:seq])
        out[row, head] = W.attention_row(q[row], ks[seq], vs[seq], pos, 50, 2, SCALE)[0][head].to(dtype)
    for i, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        near(out[at:at + lq], q[at:at + lq], ks[i], vs[i], range(lk - lq, lk), 50, 2, dtype)
        at += lq


@pytest.mark.parametrize("dtype", TYPES)
def test_decode_writes_over_its_queries(cuda_device, dtype):
    """The output may be the query's own buffer, for rows of one CTA and of a cluster."""
    for ctx, H, Hk, window in (([900, 20], 16, 2, 800), ([60 + i for i in range(200)], 8, 4, 50), ([3000], 32, 2, 2500)):
        g = torch.Generator().manual_seed(len(ctx))
        kc, vc, table, ks, vs = paged(g, ctx, Hk, dtype)
        q = normal(g, dtype, len(ctx), H, D)
        want, dev = decode(cuda_device, q, kc, vc, table, ctx, window, 3), cuda_device
        x, i32 = q.to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev)
        args = kc.to(dev), vc.to(dev), Hk, SCALE, table.to(dev), i32, 16, max(ctx), window, 3
        for _ in range(5):
            x.copy_(q)
            tch_cuda.paged_attention_window(x, x, *args)
            assert torch.equal(x.cpu(), want)
