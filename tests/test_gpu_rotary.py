"""Rotary positions: the table, both pairings, part of the head, both 16-bit types, with and without the
cache write, against the definition in 64 bits."""
import math

import pytest
import torch

from aici_b200 import _lib, tch_cuda
from oracle import window_ref as W

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,rot,base,scaling,factor,original,dtype", [
    (1, 2, 1e4, "none", 1.0, 0, torch.float32), (33, 16, 1e4, "none", 1.0, 0, torch.float32),
    (257, 96, 1e4, "linear", 2.5, 0, torch.float32), (300, 128, 5e5, "ntk", 4.0, 0, torch.float32),
    (5000, 128, 1e6, "yarn", 8.0, 512, torch.float32), (70, 2, 1e4, "ntk", 2.0, 0, torch.float32),
    (129, 256, 1e4, "yarn", 1.0, 64, torch.bfloat16), (130, 66, 1e4, "none", 1.0, 0, torch.float16)])
def test_table(cuda_device, n, rot, base, scaling, factor, original, dtype):
    got = tch_cuda.rotary_cos_sin_cache(n, rot, base, dtype, cuda_device, scaling=scaling, factor=factor,
                                        original_context=original).cpu().double()
    if rot == 2 and scaling == "ntk":  # one pair turns by 1 per position whatever the base
        scaling = "none"
    want = W.cos_sin(range(n), rot, base, scaling, factor, original)
    # half a step of the type; the angle in 64 bits, off by some 2^-50 of itself at most
    under = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -149
    bound = torch.finfo(dtype).eps / 2 * want.abs() + n * 2.0 ** -49 + under
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max()


def test_table_far_positions(cuda_device):
    n, rot = 1 << 20, 16
    got = tch_cuda.rotary_cos_sin_cache(n, rot, 1e4, torch.float32, cuda_device)
    at = [0, 1, 65535, 65536, 99999, 524287, 524288, n - 2, n - 1]
    want = W.cos_sin(at, rot, 1e4, "none", 1.0, 0)
    assert ((got[at].cpu().double() - want).abs() <= 2.0 ** -24 * want.abs() + n * 2.0 ** -49 + 2.0 ** -60).all()


def inputs(seed, T, H, Hk, D, rot, dtype, table, gap=0):
    g = torch.Generator().manual_seed(seed)
    wide = torch.randn(T, (H + 2 * Hk) * D + gap, generator=g).to(dtype)
    cs = W.cos_sin(range(500), rot, 1e4, "none", 1.0, 0).to(table)
    pos = torch.randint(0, 500, (T,), generator=g)
    nblk = (T + 40) // 16 + 6
    slots = torch.randperm(nblk * 16 - 64, generator=g)[:T] + 64
    if T >= 40:  # a run that starts inside a block, as a chunk does, and one on a block's start
        slots[:21] = torch.arange(21) + 5
        slots[21:37] = torch.arange(16) + 32
    if T > 2:
        slots[2] = -1
    kc = torch.randn(nblk, Hk, D // 8, 16, 8, generator=g).to(dtype)
    vc = torch.randn(nblk, Hk, D, 16, generator=g).to(dtype)
    return wide, cs, pos, slots, kc, vc


def close(got, want, mag, dtype):
    """Half a step of the type, three fp32 roundings of the products' magnitudes; f16 below its normals."""
    under = 2.0 ** -25 if dtype == torch.float16 else 0.0
    bound = torch.finfo(dtype).eps / 2 * want.abs() * 1.01 + 2.0 ** -22 * mag + under
    d = (got.cpu().double() - want).abs()
    assert (d <= bound).all(), float((d / bound.clamp(min=1e-30)).max())


CASES = [(1, 1, 1, 16, 16, True), (1, 8, 2, 128, 128, True), (3, 5, 1, 64, 32, False), (16, 4, 4, 80, 32, True),
         (17, 6, 2, 96, 96, False), (40, 8, 8, 128, 64, False), (50, 7, 1, 128, 48, True), (41, 2, 2, 256, 256, False),
         (200, 32, 8, 128, 128, True), (64, 3, 3, 256, 16, True)]


@pytest.mark.parametrize("dtype,table", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
@pytest.mark.parametrize("T,H,Hk,D,rot,neox", CASES)
def test_with_cache_write(cuda_device, T, H, Hk, D, rot, neox, dtype, table):
    dev = cuda_device
    wide, cs, pos, slots, kc, vc = inputs(T * 7 + rot, T, H, Hk, D, rot, dtype, table, gap=8)
    x = wide.to(dev)
    q, k, v = x[:, :H * D], x[:, H * D:(H + Hk) * D], x[:, (H + Hk) * D:(H + 2 * Hk) * D]
    kc_d, vc_d = kc.to(dev), vc.to(dev)
    slot_d = slots.to(dev) if T % 2 else slots.to(torch.int32).to(dev)
    tch_cuda.rotary_embedding_and_cache(pos.to(dev), q, k, v, D, cs.to(dev), neox, kc_d, vc_d, slot_d)
    wq, mq = W.rotate(wide[:, :H * D].view(T, H, D), cs[pos], neox)
    wk, mk = W.rotate(wide[:, H * D:(H + Hk) * D].reshape(T, Hk, D), cs[pos], neox)
    close(q.reshape(T, H, D), wq, mq, dtype)
    close(k.reshape(T, Hk, D), wk, mk, dtype)
    assert torch.equal(x[:, (H + Hk) * D:].cpu(), wide[:, (H + Hk) * D:])  # values and what lies behind them
    W.write_cache(k.reshape(T, Hk, D).cpu(), v.reshape(T, Hk, D).cpu(), kc, vc, slots)
    assert torch.equal(kc_d.cpu().view(torch.int16), kc.view(torch.int16))
    assert torch.equal(vc_d.cpu().view(torch.int16), vc.view(torch.int16))
    assert _lib.last_status() == 0


@pytest.mark.parametrize("T,H,Hk,D,rot,neox", CASES)
def test_alone_gives_what_it_gives_with_the_cache(cuda_device, T, H, Hk, D, rot, neox):
    dev, dtype = cuda_device, torch.bfloat16
    wide, cs, pos, slots, kc, vc = inputs(T + 3 * D, T, H, Hk, D, rot, dtype, torch.float32)
    a, b = wide.to(dev), wide.to(dev)
    cut = lambda x: (x[:, :H * D], x[:, H * D:(H + Hk) * D], x[:, (H + Hk) * D:])  # noqa: E731
    tch_cuda.rotary_embedding(pos.to(dev), *cut(a)[:2], D, cs.to(dev), neox)
    tch_cuda.rotary_embedding_and_cache(pos.to(dev), *cut(b), D, cs.to(dev), neox, kc.to(dev), vc.to(dev), slots.to(dev))
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    h = wide.to(dev)  # the same rows as [tokens, heads, head_size]
    q3, k3 = h[:, :H * D].unflatten(1, (H, D)), h[:, H * D:(H + Hk) * D].unflatten(1, (Hk, D))
    tch_cuda.rotary_embedding(pos.to(dev), q3, k3, D, cs.to(dev), neox)
    assert torch.equal(a.view(torch.int16), h.view(torch.int16))


def test_bad_positions_and_slots_leave_their_tokens(cuda_device):
    dev, T, H, Hk, D = cuda_device, 20, 4, 2, 128
    wide, cs, pos, slots, kc, vc = inputs(5, T, H, Hk, D, 128, torch.bfloat16, torch.float32)
    pos[4], pos[11], slots[7] = 500, -1, kc.shape[0] * 16
    x, kc_d, vc_d = wide.to(dev), kc.to(dev), vc.to(dev)
    q, k, v = x[:, :H * D], x[:, H * D:(H + Hk) * D], x[:, (H + Hk) * D:]
    tch_cuda.rotary_embedding_and_cache(pos.to(dev), q, k, v, D, cs.to(dev), True, kc_d, vc_d, slots.to(dev))
    assert _lib.last_status() == 2
    for t in (4, 11):
        assert torch.equal(x[t].cpu(), wide[t])
    good = slots.clone()
    good[[4, 7, 11]] = -1
    W.write_cache(k.reshape(T, Hk, D).cpu(), v.reshape(T, Hk, D).cpu(), kc, vc, good)
    assert torch.equal(kc_d.cpu(), kc) and torch.equal(vc_d.cpu(), vc)


def test_cache_offsets_past_32_bits(cuda_device):
    """A pool of more than 2^31 elements; only its last blocks are written."""
    dev, Hk, D = cuda_device, 8, 128
    nblk = (1 << 31) // (Hk * D * 16) + 16
    kc = torch.zeros(nblk, Hk, D // 8, 16, 8, dtype=torch.float16, device=dev)
    vc = torch.zeros(nblk, Hk, D, 16, dtype=torch.float16, device=dev)
    wide, cs, pos, _, _, _ = inputs(6, 20, 8, Hk, D, 64, torch.float16, torch.float32)
    x = wide.to(dev)
    q, k, v = x[:, :8 * D], x[:, 8 * D:16 * D], x[:, 16 * D:]
    slots = torch.arange(20) + (nblk - 3) * 16 + 7
    tch_cuda.rotary_embedding_and_cache(pos.to(dev), q, k, v, D, cs.to(dev), False, kc, vc, slots.to(dev))
    want_k, want_v = torch.zeros(8, Hk, 16, 16, 8, dtype=torch.float16), torch.zeros(8, Hk, 128, 16, dtype=torch.float16)
    W.write_cache(k.reshape(20, Hk, D).cpu(), v.reshape(20, Hk, D).cpu(), want_k, want_v, slots - (nblk - 8) * 16)
    assert torch.equal(kc[-8:].cpu(), want_k) and torch.equal(vc[-8:].cpu(), want_v)
    assert not kc[:8].any() and not vc[:8].any() and _lib.last_status() == 0


def test_refuses_mismatched_tensors(cuda_device):
    dev = cuda_device
    wide, cs, pos, slots, kc, vc = (t.to(dev) for t in inputs(7, 4, 4, 2, 128, 128, torch.bfloat16, torch.float32))
    q, k, v = wide[:, :512], wide[:, 512:768], wide[:, 768:]
    ok = (pos, q, k, v, 128, cs, True, kc, vc, slots)
    for i, bad, match in ((0, pos.int(), "positions"), (0, pos[:3], "positions"), (2, k.half(), "same dtype"),
                          (3, v.half(), "dtypes differ"), (4, 64, "head_size"), (5, cs.t(), "cos_sin_cache"),
                          (5, cs.half(), "cos_sin_cache"), (7, kc.half(), "dtypes differ"), (9, slots[:2], "slot_mapping"),
                          (2, wide[:, 512:1024], "width"), (3, v[:3], "differ in length")):
        args = list(ok)
        args[i] = bad
        with pytest.raises(_lib.AiciError, match=match):
            tch_cuda.rotary_embedding_and_cache(*args)


@pytest.mark.parametrize("stride", [1, 128, 1001])
def test_a_single_token_has_no_stride(cuda_device, stride):
    """One token whose first stride is what is left of another layout."""
    dev, H, Hk, D, dtype = cuda_device, 4, 2, 128, torch.bfloat16
    wide, cs, pos, slots, kc, vc = inputs(8, 1, H, Hk, D, 128, dtype, torch.float32)
    x = wide.to(dev)
    odd = lambda lo, n: x.flatten()[lo * D:].as_strided((1, n * D), (stride, 1))  # noqa: E731
    q, k, v = odd(0, H), odd(H, Hk), odd(H + Hk, Hk)
    assert q.is_contiguous() and q.stride(0) == stride
    alone = x.clone()
    kc_d, vc_d = kc.to(dev), vc.to(dev)
    tch_cuda.rotary_embedding_and_cache(pos.to(dev), q, k, v, D, cs.to(dev), True, kc_d, vc_d, slots.to(dev))
    close(x[:, :H * D].reshape(1, H, D), *W.rotate(wide[:, :H * D].view(1, H, D), cs[pos], True), dtype)
    W.write_cache(x[:, H * D:(H + Hk) * D].reshape(1, Hk, D).cpu(), wide[:, (H + Hk) * D:].reshape(1, Hk, D), kc, vc, slots)
    assert torch.equal(kc_d.cpu(), kc) and torch.equal(vc_d.cpu(), vc)
    flat = alone.flatten()
    tch_cuda.rotary_embedding(pos.to(dev), flat.as_strided((1, H, D), (stride, D, 1)),
                              flat[H * D:].as_strided((1, Hk, D), (stride, D, 1)), D, cs.to(dev), True)
    assert torch.equal(alone, x) and _lib.last_status() == 0


def test_yarn_mixes_by_turns(cuda_device):
    """Angles per position from the paper's NTK-by-parts formula worked out in 40 decimal digits: base 500000, trained length
    16384, factor 8.  (A mix linear in the pair's number, as some models are trained with, gives other angles between
    the two ends: pair 30 turns by 1.199e-3 there.)"""
    got = tch_cuda.rotary_cos_sin_cache(2, 128, 5e5, torch.float32, cuda_device, scaling="yarn", factor=8.0,
                                        original_context=16384).cpu().double()
    for j, angle in ((0, 1.0), (20, 1.656044008099e-02), (21, 1.349041989023e-02), (22, 9.952331774935e-03),
                     (25, 3.172472539041e-03), (30, 5.405109533618e-04), (35, 1.170003683811e-04), (38, 5.256482028508e-05),
                     (39, 4.208236768726e-05), (50, 4.411534674558e-06), (63, 3.068925988915e-07)):
        # cosine and sine are off by half a step of f32 each: together by less than 2^-23 of the angle
        assert abs(math.atan2(got[1, 64 + j], got[1, j]) - angle) <= 2.0 ** -23 * angle + 1e-12 * angle, j
        assert abs(got[0, j] - (0.1 * math.log(8.0) + 1)) <= 2.0 ** -24 * 1.3


def prompt_slots(g, T, nblk, start):
    """Slots of one long sequence in shuffled blocks from token `start` of its first block on; a few tokens of it go
    nowhere, and its last ones to single slots of other blocks."""
    blocks = torch.randperm(nblk - 4, generator=g)
    at = torch.arange(T) + start
    slots = blocks[at // 16] * 16 + at % 16
    slots[T - 5:] = (nblk - 4) * 16 + torch.randperm(64, generator=g)[:5]
    slots[torch.randint(0, T, (7,), generator=g)] = -1
    return slots


LARGE = [  # heads, kv heads, head size, rotated part, neox, kv heads of a cache-writing CTA, dtype
    (64, 8, 128, 64, False, 8, torch.float16), (10, 5, 128, 128, True, 4, torch.bfloat16), (7, 7, 256, 256, True, 2, torch.bfloat16),
    (7, 7, 256, 16, False, 4, torch.float16), (6, 3, 256, 240, True, 8, torch.bfloat16), (32, 13, 64, 48, True, 8, torch.float16),
    (40, 40, 96, 96, False, 8, torch.bfloat16), (100, 2, 16, 16, True, 2, torch.float16)]


@pytest.mark.parametrize("H,Hk,D,rot,neox,per,dtype", LARGE)
def test_many_tokens(cuda_device, H, Hk, D, rot, neox, per, dtype):
    """Calls whose CTAs take several kv heads one after the other through their ring of stages, and whose threads
    take four query heads and several runs of tokens."""
    dev, g = cuda_device, torch.Generator().manual_seed(H * D + rot)
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    tiles = -(-4 * per * sms // Hk)  # 8 x (per / 2) x SMs (tile, head) pairs give a CTA `per` heads
    if H >= 32:
        tiles = max(tiles, -(-4 * 4 * 256 * sms * 16 // (H * rot)) // 16 + 2)
    T = tiles * 16 - 7
    assert tiles * Hk >= 4 * per * sms and (per == 8 or tiles * Hk < 8 * per * sms or H >= 32)
    assert H < 32 or T * H * (rot // 16) >= 4 * 4 * 256 * sms
    wide = torch.randn(T, (H + 2 * Hk) * D, device=dev, generator=torch.Generator(dev).manual_seed(T)).to(dtype)
    cs = W.cos_sin(range(700), rot, 1e4, "none", 1.0, 0).to(torch.float32).to(dev)
    pos = torch.randint(0, 700, (T,), generator=g).to(dev)
    nblk = T // 16 + 8
    slots = prompt_slots(g, T, nblk, H % 16)
    kc, vc = torch.full((nblk, Hk, D // 8, 16, 8), 7.0, dtype=dtype), torch.full((nblk, Hk, D, 16), 7.0, dtype=dtype)
    cut = lambda x: (x[:, :H * D], x[:, H * D:(H + Hk) * D], x[:, (H + Hk) * D:])  # noqa: E731
    alone, x, kc_d, vc_d = wide.clone(), wide.clone(), kc.to(dev), vc.to(dev)
    tch_cuda.rotary_embedding_and_cache(pos, *cut(x), D, cs, neox, kc_d, vc_d, slots.to(dev))
    tch_cuda.rotary_embedding(pos, *cut(alone)[:2], D, cs, neox)
    assert torch.equal(x.view(torch.int16), alone.view(torch.int16))
    for a in range(0, T, 1000):  # the definition, some tokens at a time
        rows = slice(a, min(a + 1000, T))
        for got, was, h in ((cut(x)[0], cut(wide)[0], H), (cut(x)[1], cut(wide)[1], Hk)):
            want, mag = W.rotate(was[rows].reshape(-1, h, D), cs[pos[rows]], neox)
            close(got[rows].reshape(-1, h, D), want.cpu(), mag.cpu(), dtype)
    assert torch.equal(cut(x)[2], cut(wide)[2])
    W.write_cache(cut(x)[1].reshape(T, Hk, D).cpu(), cut(wide)[2].reshape(T, Hk, D).cpu(), kc, vc, slots)
    assert torch.equal(kc_d.cpu(), kc) and torch.equal(vc_d.cpu(), vc)
    assert _lib.last_status() == 0


@pytest.mark.parametrize("table", [torch.float32, torch.float16])
@pytest.mark.parametrize("T,H,Hk,D,rot,neox", CASES)
def test_alone_in_f16(cuda_device, T, H, Hk, D, rot, neox, table):
    dev, dtype = cuda_device, torch.float16
    wide, cs, pos, _, _, _ = inputs(T + 5 * D, T, H, Hk, D, rot, dtype, table)
    x = wide.to(dev)
    q, k = x[:, :H * D], x[:, H * D:(H + Hk) * D]
    tch_cuda.rotary_embedding(pos.to(dev), q, k, D, cs.to(dev), neox)
    close(q.reshape(T, H, D), *W.rotate(wide[:, :H * D].view(T, H, D), cs[pos], neox), dtype)
    close(k.reshape(T, Hk, D), *W.rotate(wide[:, H * D:(H + Hk) * D].reshape(T, Hk, D), cs[pos], neox), dtype)
    assert torch.equal(x[:, (H + Hk) * D:].cpu(), wide[:, (H + Hk) * D:]) and _lib.last_status() == 0


def test_rows_past_32_bits(cuda_device):
    """Slices of rows so wide that the last tokens lie more than 2^31 elements behind the first."""
    dev, dtype, H, Hk, D, width, T = cuda_device, torch.float16, 3, 2, 128, 150, 120000
    assert (T - 1000) * width * D > 1 << 31
    wide = torch.zeros(T, width * D, dtype=dtype, device=dev)
    wide[:, -7 * D:] = torch.randn(T, 7 * D, device=dev, generator=torch.Generator(dev).manual_seed(9)).to(dtype)
    was = wide[:, -7 * D:].clone()
    cs = W.cos_sin(range(900), D, 1e4, "none", 1.0, 0).to(torch.float32).to(dev)
    pos = torch.arange(T, device=dev) % 900
    kc = torch.zeros(T // 16, Hk, D // 8, 16, 8, dtype=dtype, device=dev)
    vc = torch.zeros(T // 16, Hk, D, 16, dtype=dtype, device=dev)
    cut = lambda x: (x[:, :H * D], x[:, H * D:(H + Hk) * D], x[:, (H + Hk) * D:])  # noqa: E731
    q, k, v = cut(wide[:, -7 * D:])
    tch_cuda.rotary_embedding_and_cache(pos, q, k, v, D, cs, True, kc, vc, torch.arange(T, device=dev))
    at = torch.tensor([0, 1, 60000, T - 33, T - 17, T - 2, T - 1], device=dev)
    for got, old, h in ((q, cut(was)[0], H), (k, cut(was)[1], Hk)):
        want, mag = W.rotate(old[at].reshape(-1, h, D), cs[pos[at]], True)
        close(got[at].reshape(-1, h, D), want.cpu(), mag.cpu(), dtype)
    assert torch.equal(v, cut(was)[2]) and not wide[:, :-7 * D].any()
    assert torch.equal(kc.permute(0, 3, 1, 2, 4).reshape(T, Hk * D), k) and torch.equal(vc.permute(0, 3, 1, 2).reshape(T, Hk * D), v)
    b = wide.clone()
    tch_cuda.rotary_embedding(pos, *cut(b[:, -7 * D:])[:2], D, cs, True)
    for got, old, h in ((cut(b[:, -7 * D:])[0], q, H), (cut(b[:, -7 * D:])[1], k, Hk)):
        want, mag = W.rotate(old[at].reshape(-1, h, D), cs[pos[at]], True)
        close(got[at].reshape(-1, h, D), want.cpu(), mag.cpu(), dtype)
    assert _lib.last_status() == 0


@pytest.mark.parametrize("T,H,Hk,D,rot,neox", [(5, 80, 1, 256, 256, True), (3, 130, 2, 256, 240, False), (9, 300, 3, 128, 128, True)])
def test_more_heads_than_threads_take_at_once(cuda_device, T, H, Hk, D, rot, neox):
    """Heads beyond four for every slot of a CTA: a thread goes over its token's heads more than once."""
    assert H > 4 * (256 // (rot // 16))
    dev, dtype = cuda_device, torch.bfloat16
    wide, cs, pos, _, _, _ = inputs(T + H, T, H, Hk, D, rot, dtype, torch.float32)
    x = wide.to(dev)
    q, k = x[:, :H * D], x[:, H * D:(H + Hk) * D]
    tch_cuda.rotary_embedding(pos.to(dev), q, k, D, cs.to(dev), neox)
    close(q.reshape(T, H, D), *W.rotate(wide[:, :H * D].view(T, H, D), cs[pos], neox), dtype)
    close(k.reshape(T, Hk, D), *W.rotate(wide[:, H * D:(H + Hk) * D].reshape(T, Hk, D), cs[pos], neox), dtype)
    assert _lib.last_status() == 0
