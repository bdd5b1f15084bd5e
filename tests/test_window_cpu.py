"""Refusals of the operators around windowed attention, and their oracle against hand-worked cases.
Everything here ends before a kernel would be launched."""
import ctypes

import pytest
import torch

from aici_b200 import _lib, batch_info, build, tch_cuda
from aici_b200._lib import AiciError
from oracle import window_ref as W

P = 0x10000  # an aligned address that no refused call touches


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def refused(lib, name, args, match):
    with pytest.raises(AiciError, match=match):
        _lib.check(name, getattr(lib, name)(*args))


STEP = dict(q=P, c=P, bt=P, fb=P, fc=P, n=4, mb=8, bs=8, fcap=10, nb=100, block=16, mt=64, sq=P, pos=P, slot=P, li=P, co=P, fo=P, s=None)


@pytest.mark.parametrize("change,match", [
    (dict(block=32), "block_size must be 16"), (dict(n=0), "num_requests"), (dict(n=16385), "num_requests"),
    (dict(mb=0), "table width"), (dict(mb=9), "table width"), (dict(mt=-1), "max_tokens"), (dict(mt=1 << 30), "max_tokens"),
    (dict(nb=0), "num_blocks"), (dict(nb=(1 << 27) + 1), "num_blocks"), (dict(q=None), "NULL"), (dict(fb=None), "NULL"),
    (dict(pos=None), "NULL"), (dict(pos=P + 8), "16-byte aligned"), (dict(fcap=-1), "negative")])
def test_step_tables_refuses(lib, change, match):
    refused(lib, "aici_step_tables", {**STEP, **change}.values(), match)


ROT = dict(pos=P, q=P, k=P, v=P, cs=P, kc=P, vc=P, slots=P, s64=0, T=4, H=8, Hk=2, D=128, rot=64, neox=1, maxpos=64,
           block=16, nb=8, qs=1024, ks=256, vs=256, tt=2, dt=0, s=None)


@pytest.mark.parametrize("change,match", [
    (dict(dt=2), "only bf16 and f16"), (dict(dt=1, tt=0), "cos_sin_cache"), (dict(D=120), "head_size"), (dict(D=272), "head_size"),
    (dict(rot=0), "rot_dim"), (dict(rot=24), "rot_dim"), (dict(rot=144), "rot_dim"), (dict(block=8), "block_size"),
    (dict(H=0), "bad sizes"), (dict(maxpos=0), "bad sizes"), (dict(qs=1020), "token strides"), (dict(ks=128), "token strides"),
    (dict(vs=252), "token strides"), (dict(q=P + 2), "aligned"), (dict(vc=P + 8), "aligned"), (dict(slots=None), "NULL"),
    (dict(nb=0), "num_blocks")])
def test_rotary_and_cache_refuses(lib, change, match):
    refused(lib, "aici_rotary_embedding_and_cache", {**ROT, **change}.values(), match)


@pytest.mark.parametrize("change,match", [
    (dict(dt=3), "dtype"), (dict(rot=3), "rot_dim"), (dict(rot=258), "rot_dim"), (dict(maxpos=-1), "max_position"),
    (dict(base=1.0), "base"), (dict(base=float("nan")), "base"), (dict(scaling=4), "scaling"), (dict(factor=0.5), "factor"),
    (dict(factor=float("inf")), "factor"), (dict(scaling=3, orig=0), "original_context"), (dict(out=None), "NULL")])
def test_table_refuses(lib, change, match):
    args = {**dict(out=P, maxpos=16, rot=64, base=1e4, scaling=1, factor=2.0, orig=128, dt=2, s=None), **change}
    refused(lib, "aici_rotary_cos_sin_cache", args.values(), match)


DEC = dict(out=P, q=P, kc=P, vc=P, Hk=2, scale=0.1, bt=P, cl=P, block=16, maxctx=64, window=8, sinks=0, n=2, H=8, D=128,
           mb=4, nb=8, qs=1024, bs=4096, hs=2048, dt=0, s=None)
DECODE_REFUSALS = [
    (dict(dt=2), "only bf16 and f16"), (dict(D=64), "head_size"), (dict(block=32), "block_size"), (dict(H=7), "not divisible"),
    (dict(H=34, qs=8192), "at most 16"), (dict(window=0), "window"), (dict(window=-3), "window"), (dict(sinks=-1), "sinks"),
    (dict(scale=0.0), "positive"), (dict(n=-1), "negative"), (dict(maxctx=-1), "negative"), (dict(qs=1023), "q_stride"),
    (dict(qs=512), "q_stride"), (dict(hs=1024), "contiguous head tiles"), (dict(bs=2048), "contiguous head tiles"),
    (dict(out=P + 8), "aligned"), (dict(cl=None), "NULL"), (dict(nb=0), "num_blocks")]


@pytest.mark.parametrize("change,match", DECODE_REFUSALS)
def test_window_decode_refuses(lib, change, match):
    refused(lib, "aici_paged_attention_window", {**DEC, **change}.values(), match)


PRE = dict(out=P, q=P, k=P, v=P, cq=P, ck=P, batch=1, tq=4, tk=4, H=8, Hk=2, D=128, mq=4, mk=4, window=8, sinks=0, s0=1024,
           s1=128, s2=256, s3=128, s4=256, s5=128, s6=1024, s7=128, scale=0.1, dt=1, s=None)
PREFILL_REFUSALS = [
    (dict(dt=2), "only bf16 and f16"), (dict(D=96), "head_size"), (dict(batch=0), "batch"), (dict(batch=65536), "batch"),
    (dict(Hk=3), "not divisible"), (dict(window=0), "window"), (dict(sinks=-2), "sinks"), (dict(scale=-1.0), "positive"),
    (dict(tq=-1), "negative"), (dict(s1=64), "strides"), (dict(s4=260), "strides"), (dict(q=P + 4), "aligned"),
    (dict(cq=None), "NULL"), (dict(k=None), "NULL")]


@pytest.mark.parametrize("change,match", PREFILL_REFUSALS)
def test_window_prefill_refuses(lib, change, match):
    refused(lib, "aici_mha_varlen_window_fwd", {**PRE, **change}.values(), match)


PAGED = dict(out=P, q=P, kc=P, vc=P, cq=P, cl=P, bt=P, batch=1, tq=4, H=8, Hk=2, D=128, block=16, mq=4, mk=4, mb=4, nb=8,
             window=8, sinks=0, s0=1024, s1=128, s2=1024, s3=128, bs=4096, hs=2048, scale=0.1, dt=0, s=None)


@pytest.mark.parametrize("change,match", [
    (dict(dt=2), "only bf16 and f16"), (dict(D=96), "head_size"), (dict(batch=0), "batch"), (dict(window=0), "window"),
    (dict(sinks=-2), "sinks"), (dict(block=8), "block_size"), (dict(hs=64), "contiguous head tiles"), (dict(mb=-1), "negative"),
    (dict(s2=64), "strides"), (dict(bt=None), "NULL"), (dict(nb=0), "num_blocks"), (dict(vc=P + 2), "aligned")])
def test_window_paged_prefill_refuses(lib, change, match):
    refused(lib, "aici_mha_varlen_paged_window_fwd", {**PAGED, **change}.values(), match)


def test_empty_calls_return(lib):
    for name, args in (("aici_paged_attention_window", {**DEC, "n": 0}), ("aici_mha_varlen_window_fwd", {**PRE, "tq": 0}),
                       ("aici_mha_varlen_paged_window_fwd", {**PAGED, "mq": 0}),
                       ("aici_rotary_embedding_and_cache", {**ROT, "T": 0})):
        _lib.check(name, getattr(lib, name)(*args.values()))


def test_python_side_refuses_cpu_tensors_and_wrong_types():
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(AiciError, match="no CPU path"):
        batch_info.step_tables(i, i, i.view(2, 2), i, i[:1], 8, 4)
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    kc, vc = torch.zeros(2, 2, 16, 16, 8, dtype=torch.bfloat16), torch.zeros(2, 2, 128, 16, dtype=torch.bfloat16)
    cs, pos = torch.zeros(8, 128), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(AiciError, match="no CPU path"):
        tch_cuda.rotary_embedding(pos, x, x, 128, cs, True)
    with pytest.raises(AiciError, match="no CPU path"):
        tch_cuda.rotary_embedding_and_cache(pos, x, x, x, 128, cs, True, kc, vc, i)
    with pytest.raises(AiciError, match="no CPU path"):
        tch_cuda.rotary_cos_sin_cache(8, 128, 1e4, torch.float32, "cpu")
    with pytest.raises(AiciError, match="unknown scaling"):
        tch_cuda.rotary_cos_sin_cache(8, 128, 1e4, torch.float32, "cuda", scaling="other")
    with pytest.raises(AiciError, match="no CPU path"):
        tch_cuda.paged_attention_window(x, x, kc, vc, 2, 0.1, i.view(4, 1), i, 16, 16, 4)
    with pytest.raises(AiciError, match="no CPU path"):
        tch_cuda.flash_attn_varlen_window(x, x, x, i[:2], i[:2], 1, 1, 0.1, 4)
    with pytest.raises(AiciError, match="no CPU path"):
        tch_cuda.flash_attn_varlen_paged_window(x, kc, vc, i[:2], i[:1], i.view(1, 4), 1, 1, 0.1, 4)


# ---- the oracle -----------------------------------------------------------------------------------------
def test_oracle_step_by_hand():
    cu, pos, slots, logits, ctx, count, tables, kind = W.step_tables(
        [1, 0, 18], [16, 5, 3], [[7, 0, 0], [4, 0, 0], [9, 0, 0]], [1, 2, 3, 5, 6], 4, 20, 50)
    assert kind is None and cu == [0, 1, 1, 19] and logits == [0, -1, 18] and ctx == [17, 5, 21] and count == 2
    assert tables == [[7, 5, 0], [4, 0, 0], [9, 3, 0]]
    assert pos[:3] == [16, 3, 4] and pos[-2:] == [20, 0] and slots[0] == 80 and slots[1] == 9 * 16 + 3
    assert slots[14] == 48 and slots[-1] == -1
    assert W.step_tables([1], [16], [[7]], [1], 1, 4, 8)[-1] == "bad"
    assert W.step_tables([1], [16], [[7, 0]], [1], 0, 4, 8)[-1] == "blocks"


def test_oracle_window_by_hand():
    assert W.visible(10, 3, 0) == [8, 9, 10] and W.visible(10, 3, 2) == [0, 1, 8, 9, 10]
    assert W.visible(1, 5, 4) == [0, 1] and W.visible(-1, 5, 4) == []
    q, k, v = torch.zeros(2, 4), torch.zeros(5, 1, 4), torch.arange(20.0).view(5, 1, 4)
    o, a, n, _ = W.attention_row(q, k, v, 4, 2, 1, 1.0)  # equal weights of tokens 0, 3, 4
    assert n == 3 and torch.allclose(o[0], v[[0, 3, 4], 0].double().mean(0))


def test_oracle_rotation_keeps_lengths_and_relative_positions():
    cs = W.cos_sin(range(40), 16, 1e4, "none", 1.0, 0)
    x, y = torch.randn(1, 1, 24, dtype=torch.float64), torch.randn(1, 1, 24, dtype=torch.float64)
    for neox in (True, False):
        at = lambda z, p: W.rotate(z, cs[p:p + 1], neox)[0][0, 0]  # noqa: E731
        assert torch.allclose(at(x, 7) @ at(y, 3), at(x, 30) @ at(y, 26))
        assert torch.equal(at(x, 9)[16:], x[0, 0, 16:])
        assert torch.allclose(at(x, 9).norm(), x.norm())
