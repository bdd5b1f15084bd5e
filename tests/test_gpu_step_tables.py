"""The step's index tensors built on the GPU: equal, entry by entry, to the oracle's."""
import random

import pytest
import torch

from aici_b200 import _lib, batch_info
from oracle import window_ref as W

pytestmark = pytest.mark.gpu
I32 = torch.int32


def make(seed, n, most_new, most_ctx, pad_tokens=0, pad_free=3, width_extra=0):
    r = random.Random(seed)
    news = [r.choice([0, 1, 1, r.randint(0, most_new)]) for _ in range(n)]
    ctx = [r.randint(0, most_ctx) for _ in range(n)]
    width = max(1, max(-(-(c + q) // 16) for c, q in zip(ctx, news))) + width_extra
    need = sum(-(-(c + q) // 16) - -(-c // 16) for c, q in zip(ctx, news))
    held = sum(-(-c // 16) for c in ctx)
    ids = list(range(held + need + pad_free))
    r.shuffle(ids)
    it = iter(ids)
    tables = [[next(it) for _ in range(-(-c // 16))] for c in ctx]
    tables = [row + [-7] * (width - len(row)) for row in tables]
    free = list(it)
    return news, ctx, tables, free, len(free), sum(news) + pad_tokens, len(ids)


def call(dev, news, ctx, tables, free, count, max_tokens, num_blocks, out=None, t=None):
    d = lambda x: torch.tensor(x, dtype=I32, device=dev)  # noqa: E731
    bt = t if t is not None else d(tables)
    res = batch_info.step_tables(d(news), d(ctx), bt, d(free), d([count]), num_blocks, max_tokens, out=out)
    return res, bt


def check(res, bt, want):
    cu, pos, slots, logits, ctx, count, tables, _ = want
    assert res.seqlens_q.tolist() == cu
    assert res.positions.tolist() == pos
    assert res.slot_mapping.tolist() == slots
    assert res.logit_idxs.tolist() == logits
    assert res.context_lens.tolist() == ctx
    assert res.free_count.tolist() == [count]
    assert bt.tolist() == tables


@pytest.mark.parametrize("seed,n,most_new,most_ctx,pad", [
    (1, 1, 1, 0, 0), (2, 1, 1, 16, 3), (3, 1, 300, 15, 0), (4, 5, 40, 40, 1), (5, 64, 1, 700, 0), (6, 200, 70, 300, 5),
    (7, 513, 3, 50, 2), (8, 1025, 40, 33, 0), (9, 3000, 2, 100, 9), (10, 30, 2000, 2000, 0)])
def test_matches_oracle(cuda_device, seed, n, most_new, most_ctx, pad):
    args = make(seed, n, most_new, most_ctx, pad)
    res, bt = call(cuda_device, *args)
    check(res, bt, W.step_tables(*args))
    assert _lib.last_status() == 0


def test_most_requests(cuda_device):
    args = make(11, 16384, 1, 20)
    res, bt = call(cuda_device, *args)
    check(res, bt, W.step_tables(*args))
    assert _lib.last_status() == 0


def test_in_place_over_several_steps_and_strided_table(cuda_device):
    """State that advances in its own buffers, in a table whose rows lie further apart."""
    dev, n = cuda_device, 37
    d = lambda x: torch.tensor(x, dtype=I32, device=dev)  # noqa: E731
    r = random.Random(3)
    wide = torch.full((n, 40), -7, dtype=I32, device=dev)
    bt, ctx, free = wide[:, :33], d([0] * n), list(range(900))
    r.shuffle(free)
    count, free_d = d([900]), d(free)
    T = 150
    out = batch_info.StepTables(torch.empty(n + 1, dtype=I32, device=dev), torch.empty(T, dtype=torch.int64, device=dev),
                                torch.empty(T, dtype=I32, device=dev), torch.empty(n, dtype=I32, device=dev), ctx, count)
    state = ([0] * n, [[-7] * 33 for _ in range(n)], 900)
    for step in range(6):
        news = [r.randint(0, 7) for _ in range(n)]
        news = news if sum(news) <= T else [1] * n
        want = W.step_tables(news, state[0], state[1], free, state[2], T, 900)
        batch_info.step_tables(d(news), ctx, bt, free_d, count, 900, T, out=out)
        check(out, bt, want)
        state = (want[4], want[6], want[5])
    assert (wide[:, 33:] == -7).all() and _lib.last_status() == 0


@pytest.mark.parametrize("which", ["context", "count", "both"])
def test_in_place_with_many_tokens(cuda_device, which):
    """Large enough for several CTAs, which must all read the state before one of them writes it."""
    dev = cuda_device
    d = lambda x: torch.tensor(x, dtype=I32, device=dev)  # noqa: E731
    news, ctx, tables, free, count, T, num_blocks = make(31, 700, 160, 400)
    want = W.step_tables(news, ctx, tables, free, count, T, num_blocks)
    for _ in range(20):
        e = lambda k, t=I32: torch.empty(k, dtype=t, device=dev)  # noqa: E731
        ctx_d, count_d, bt = d(ctx), d([count]), d(tables)
        out = batch_info.StepTables(e(701), e(T, torch.int64), e(T), e(700), ctx_d if which != "count" else e(700),
                                    count_d if which != "context" else e(1))
        batch_info.step_tables(d(news), ctx_d, bt, d(free), count_d, num_blocks, T, out=out)
        check(out, bt, want)
    assert _lib.last_status() == 0


@pytest.mark.parametrize("change,status", [
    (lambda a: a[0].__setitem__(2, -1), 1), (lambda a: a[1].__setitem__(0, -5), 1), (lambda a: a[1].__setitem__(1, 1 << 30), 1),
    (lambda a: a[0].__setitem__(1, (1 << 31) - 1), 1), (lambda a: a.__setitem__(5, a[5] - 1), 1),
    (lambda a: a.__setitem__(4, 0), 16), (lambda a: a.__setitem__(4, -3), 1), (lambda a: a.__setitem__(4, a[4] + 1), 1)])
def test_a_step_that_does_not_fit_changes_nothing(cuda_device, change, status):
    args = list(make(21, 9, 50, 60, 0, 0))
    change(args)
    res, bt = call(cuda_device, *args)
    want = W.step_tables(*args)
    assert want[-1] == ("blocks" if status == 16 else "bad")
    check(res, bt, want)
    assert _lib.last_status() == status


def test_bad_block_ids_give_no_slot(cuda_device):
    args = list(make(22, 6, 30, 40))
    args[2][0][0], args[1][0], args[0][0] = 99999, 5, 4  # the block the first request continues
    args[6] = max(args[6], 1)
    args[5] = sum(args[0])
    args[3] = list(args[3]) + [5] * 4
    args[4] = len(args[3])
    res, bt = call(cuda_device, *args)
    check(res, bt, W.step_tables(*args))
    assert res.slot_mapping[:4].tolist() == [-1] * 4 and _lib.last_status() == 1


def test_captured_steps_advance_on_another_stream(cuda_device):
    """One new token per request and step, captured once and replayed."""
    dev, n = cuda_device, 20
    d = lambda x: torch.tensor(x, dtype=I32, device=dev)  # noqa: E731
    ctx0 = [3 * i for i in range(n)]
    free = list(range(100, 400))
    tables = [[i * 4 + j for j in range(-(-c // 16))] + [-7] * (8 - -(-c // 16)) for i, c in enumerate(ctx0)]
    ctx, bt, count, ones, free_d = d(ctx0), d(tables), d([300]), d([1] * n), d(free)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        keep = ctx.clone(), bt.clone(), count.clone()
        first = batch_info.step_tables(ones, ctx, bt, free_d, count, 400, n)
        out = batch_info.StepTables(first.seqlens_q, first.positions, first.slot_mapping, first.logit_idxs, ctx, count)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            batch_info.step_tables(ones, ctx, bt, free_d, count, 400, n, out=out)
        for t, k in zip((ctx, bt, count), keep):
            t.copy_(k)
        state = (ctx0, tables, 300)
        for _ in range(40):
            want = W.step_tables([1] * n, state[0], state[1], free, state[2], n, 400)
            graph.replay()
            state = (want[4], want[6], want[5])
        check(out, bt, want)
    assert _lib.last_status() == 0


def test_refuses_out_of_another_shape(cuda_device):
    args = make(30, 4, 5, 20)
    res, bt = call(cuda_device, *args)
    with pytest.raises(_lib.AiciError, match="out does not match"):
        call(cuda_device, *args[:5], args[5] + 1, args[6], out=res)
    for tokens in (-1, 1 << 30, 1 << 32):
        with pytest.raises(_lib.AiciError, match="max_tokens"):
            call(cuda_device, *args[:5], tokens, args[6])


def test_a_bad_id_of_the_free_list_stays_bad(cuda_device):
    """A block id outside the pool that the free list hands out is entered in the table: later tokens of that block
    meet it again, and none of them is written to the block that the entry named before."""
    dev = cuda_device
    args = [[3, 2], [16, 4], [[1, 6], [2, 6]], [5, 777], 2, 8, 10]
    res, bt = call(dev, *args)
    want = W.step_tables(*args)
    check(res, bt, want)
    assert bt.tolist()[0] == [1, 777] and res.slot_mapping[:3].tolist() == [-1] * 3 and _lib.last_status() == 1
    args = [[1, 0], want[4], want[6], [5, 777], want[5], 8, 10]
    res, bt = call(dev, *args)
    check(res, bt, W.step_tables(*args))
    assert res.slot_mapping[0].item() == -1 and _lib.last_status() == 1


def test_most_requests_in_place(cuda_device):
    """The largest call in its own buffers: one cluster of CTAs with all of their shared memory."""
    dev = cuda_device
    d = lambda x: torch.tensor(x, dtype=I32, device=dev)  # noqa: E731
    e = lambda k, t=I32: torch.empty(k, dtype=t, device=dev)  # noqa: E731
    news, ctx, tables, free, count, T, num_blocks = make(32, 16384, 5, 40)
    want = W.step_tables(news, ctx, tables, free, count, T, num_blocks)
    for _ in range(5):
        ctx_d, count_d, bt = d(ctx), d([count]), d(tables)
        out = batch_info.StepTables(e(16385), e(T, torch.int64), e(T), e(16384), ctx_d, count_d)
        batch_info.step_tables(d(news), ctx_d, bt, d(free), count_d, num_blocks, T, out=out)
        check(out, bt, want)
    assert _lib.last_status() == 0
