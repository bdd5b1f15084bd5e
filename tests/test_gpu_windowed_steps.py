"""The operators together, as a serving loop uses them: tables for the step, rotary positions with the
cache write, attention over the cache -- a chunk of prompt first, then single tokens, then both."""
import math

import pytest
import torch

from aici_b200 import _lib, batch_info, tch_cuda
from oracle import window_ref as W

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("dtype,neox,rot,H,Hk,window,sinks", [
    (torch.bfloat16, True, 128, 8, 2, 40, 4), (torch.float16, False, 64, 6, 2, 25, 0), (torch.bfloat16, False, 32, 4, 4, 500, 1)])
def test_steps_of_a_batch(cuda_device, dtype, neox, rot, H, Hk, window, sinks):
    dev, n, nblk, scale = cuda_device, 4, 60, 1 / math.sqrt(D)
    g = torch.Generator().manual_seed(rot + H)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cs = tch_cuda.rotary_cos_sin_cache(300, rot, 1e4, torch.float32, dev, scaling="yarn", factor=2.0, original_context=64)
    tables, free = torch.full((n, 20), -1, dtype=torch.int32, device=dev), i32(torch.randperm(nblk, generator=g).tolist())
    ctx, count = i32([0] * n), i32([nblk])
    kc = torch.full((nblk, Hk, 16, 16, 8), float("nan"), dtype=dtype, device=dev)
    vc = torch.full((nblk, Hk, D, 16), float("nan"), dtype=dtype, device=dev)
    keys, values = [torch.zeros(0, Hk, D)] * n, [torch.zeros(0, Hk, D)] * n
    for news in ([70, 33, 1, 130], [1, 1, 1, 1], [1, 45, 0, 1], [1, 1, 1, 1]):
        T = sum(news)
        x = torch.randn(T, H + 2 * Hk, D, generator=g).to(dtype)
        xd = x.to(dev)
        q, k, v = xd[:, :H], xd[:, H:H + Hk], xd[:, H + Hk:]
        step = batch_info.step_tables(i32(news), ctx, tables, free, count, nblk, T)
        tch_cuda.rotary_embedding_and_cache(step.positions, q, k, v, D, cs, neox, kc, vc, step.slot_mapping)
        ctx, count = step.context_lens, step.free_count
        if news == [1] * n:
            out = torch.empty(n, H, D, dtype=dtype, device=dev)
            tch_cuda.paged_attention_window(out, q, kc, vc, Hk, scale, tables, ctx, 16, 300, window, sinks)
        else:
            out = tch_cuda.flash_attn_varlen_paged_window(q, kc, vc, step.seqlens_q, ctx, tables, max(news), 300, scale,
                                                          window, sinks)
        out, at = out.cpu(), 0
        pos = step.positions.cpu()
        table = cs.cpu()[pos]
        for i, m in enumerate(news):
            rows = slice(at, at + m)
            # the kernel's own rotated keys are the reference's (the rotation has tests of its own): what is
            # checked here is that every token's key sits where attention looks for it
            wq, mag = W.rotate(x[rows, :H], table[rows], neox)
            half = torch.finfo(dtype).eps / 2
            assert ((q[rows].cpu().double() - wq).abs() <= half * 1.01 * wq.abs() + 2.0 ** -22 * mag + 2.0 ** -25).all()
            keys[i] = torch.cat([keys[i].to(dtype), k[rows].cpu()])
            values[i] = torch.cat([values[i].to(dtype), x[rows, H + Hk:]])
            for r in range(m):
                p = len(keys[i]) - m + r
                assert int(pos[at + r]) == p
                o, a, seen, size = W.attention_row(q[at + r].cpu(), keys[i], values[i], p, window, sinks, scale)
                vmax = float(values[i].abs().max())
                assert ((out[at + r].double() - o).abs() <= W.attention_bound(o, a, seen, size, vmax, dtype)).all(), (i, p)
            at += m
    assert ctx.tolist() == [73, 80, 3, 133] and count.tolist() == [nblk - 5 - 5 - 1 - 9] and _lib.last_status() == 0


def test_a_captured_decode_loop(cuda_device):
    """Tables, rotation, cache write and attention of a decode step in one graph whose state lives on the
    GPU: replayed step by step it gives what the same calls give eagerly."""
    dev, n, H, Hk, nblk, dtype, scale = cuda_device, 9, 8, 2, 80, torch.bfloat16, 1 / math.sqrt(D)
    g = torch.Generator().manual_seed(5)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cs = tch_cuda.rotary_cos_sin_cache(200, 128, 1e4, torch.float32, dev)
    ones, free = i32([1] * n), i32(torch.randperm(nblk, generator=g).tolist())
    xs = torch.randn(50, n, H + 2 * Hk, D, generator=g).to(dtype).to(dev)

    def fresh():
        return (torch.zeros(n, 8, dtype=torch.int32, device=dev), i32([0] * n), i32([nblk]),
                torch.zeros(nblk, Hk, 16, 16, 8, dtype=dtype, device=dev), torch.zeros(nblk, Hk, D, 16, dtype=dtype, device=dev))

    def one(x, state, out, st):
        tables, ctx, count, kc, vc = state
        batch_info.step_tables(ones, ctx, tables, free, count, nblk, n, out=st)
        q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
        tch_cuda.rotary_embedding_and_cache(st.positions, q, k, v, D, cs, True, kc, vc, st.slot_mapping)
        tch_cuda.paged_attention_window(out, q, kc, vc, Hk, scale, tables, ctx, 16, 128, 30, 2)

    def tensors(state):
        e = lambda k, t=torch.int32: torch.empty(k, dtype=t, device=dev)  # noqa: E731
        return batch_info.StepTables(e(n + 1), e(n, torch.int64), e(n), e(n), state[1], state[2])

    a, b = fresh(), fresh()
    sa, sb = tensors(a), tensors(b)
    eager, out, x = [], torch.empty(n, H, D, dtype=dtype, device=dev), xs[0].clone()
    for s in range(50):
        o = torch.empty(n, H, D, dtype=dtype, device=dev)
        one(xs[s].clone(), a, o, sa)
        eager.append(o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one(x, b, out, sb)
    for s in range(50):
        x.copy_(xs[s])
        graph.replay()
        assert torch.equal(out, eager[s]), s
    assert torch.equal(a[3], b[3]) and torch.equal(a[4], b[4]) and a[1].tolist() == b[1].tolist() == [50] * n
    assert _lib.last_status() == 0
