"""The oracle of a step over a sliding window against hand cases and the host's own bookkeeping, and what the entry points refuse: their
checks come before any GPU work, so descriptors of host memory do."""
import ctypes
import math

import numpy as np
import pytest
import torch

from aici_amd import _lib, attn, kernels, paged
from oracle import steps


def test_seen_by_hand():
    assert steps.seen(0, 0, 0) == [0]
    assert steps.seen(5, 2, 0) == [3, 4, 5]
    assert steps.seen(5, 2, 2) == [0, 1, 3, 4, 5]
    assert steps.seen(5, 100, 3) == [0, 1, 2, 3, 4, 5]
    assert steps.seen(2, 0, 50) == [0, 1, 2]
    assert steps.seen(-1, 3, 2) == []


def test_window_attention_by_hand():
    """One head, one head element, scale 1: keys 0, 1, 2, .. and equal queries; position 4 with a window of 1 and a sink sees 0, 3, 4."""
    kc = torch.zeros((1, 1, 1, 8, 8))
    vc = torch.zeros((1, 1, 8, 8))
    kc[0, 0, 0, :, 0] = torch.arange(8.0)
    vc[0, 0, 0, :] = 10.0 + torch.arange(8.0)
    q = torch.zeros((1, 1, 8))
    q[0, 0, 0] = 1.0
    out, mass, lse = steps.window_attention(q, kc, vc, torch.zeros((1, 1), dtype=torch.int32), [1], [5], 1.0, 1, 1)
    w = [math.exp(x) for x in (0, 3, 4)]
    assert abs(float(out[0, 0, 0]) - (w[0] * 10 + w[1] * 13 + w[2] * 14) / sum(w)) < 1e-12
    assert abs(float(lse[0, 0]) - math.log(sum(w))) < 1e-12 and torch.equal(out, mass)


def test_penalize_by_hand():
    x = torch.tensor([[2.0, -2.0, 3.0, -1.0, 0.5]])
    out = steps.penalize(x, [[0, 1, 2, 2, 1, 7, -3]], [2], [2.0], [0.5], [0.25], torch.tensor([[0.0, 0, 0, 4, 0]]),
                         torch.tensor([[True, True, True, True, False]]))
    # 0 in the prompt alone; 1 in the prompt and once behind it; 2 twice behind it
    assert out.tolist()[0] == [1.0, -4.0 - 0.5 - 0.25, 1.5 - 1.0 - 0.25, 3.0, -math.inf]


def test_step_blocks_hand_case():
    s = steps.StepBlocks(4, 6, 3, 3, window_left=3, sinks=1)
    a = s.step([5, 1, 0], 8)
    assert a["served"] == [5, 1, 0] and s.tables[0][:2] == [0, 1] and s.tables[1][0] == 2
    assert a["positions"] == [0, 1, 2, 3, 4, 0, 0, 0] and a["slot_mapping"] == [0, 1, 2, 3, 4, 8, -1, -1]
    assert a["seqlens_q"] == [0, 5, 6, 6] and a["logit_idxs"] == [4, 5, 0] and a["context_lens"] == [5, 1, 0]
    b = s.step([6, 0, 13], 8)                       # request 2 would need 13 of 12 tokens
    assert b["served"] == [6, 0, -2] and s.tables[0] == [0, 1, 3] and s.kv[0] == 11
    c = s.step([1, -1, 12], 16)                     # column 1 (tokens 4..7) is in front of the window of token 11; request 1 ends
    assert c["ends"][1] == 8 and c["served"] == [1, 0, 12] and s.tables[2] == [4, 5, 1] and s.gone == [2, 0, 0]
    d = s.step([1, 5, 0], 16)                       # request 0 is full; request 1 gets the free block and what request 2's window has passed
    assert d["served"] == [-2, 5, 0] and d["totals"] == [5, 1, 0, 2] and s.tables[1][:2] == [2, 5]
    e = s.step([0, 4, 0], 16)                       # another block for request 1, and there is none
    assert e["served"] == [0, -1, 0] and e["totals"] == [0, 1, 0, 0] and e["slot_mapping"] == [-1] * 16


def test_step_blocks_agrees_with_the_host_bookkeeping():
    """Without a window and with nothing given back, the host's allocator hands out the same blocks, its builder the same index arrays."""
    rng = np.random.default_rng(3)
    bs, R = 16, 6
    s = steps.StepBlocks(bs, 300, R, 40)
    alloc = paged.BlockAllocator(bs, 300)
    lens = [0] * R
    for step in range(12):
        new = [int(rng.integers(2, 40)) for _ in range(R)]
        got = s.step(new, sum(new) + 5)
        builder = paged.BatchInfoBuilder(bs, 640, 0)
        for r in range(R):
            if step == 0:
                alloc.alloc_seq(r, new[r])
            else:
                assert alloc.append_slots(r, lens[r], lens[r] + new[r]) == []
            lens[r] += new[r]
            builder.sched_out(alloc, r, [7] * lens[r], lens[r] - new[r])
        bi = builder.finish()
        n = sum(new)
        assert got["positions"][:n] == bi.positions.tolist() and got["slot_mapping"][:n] == bi.slot_mapping.tolist()
        assert got["seqlens_q"] == bi.seqlens_q.tolist() and got["logit_idxs"] == bi.logit_idxs.tolist()
        assert got["slot_mapping"][n:] == [-1] * 5


def _t(*sizes, dtype=_lib.BF16, data=256):
    t = _lib.Tensor()
    t.data, t.dtype, t.ndim = data, dtype, len(sizes)
    stride = 1
    for i in reversed(range(len(sizes))):
        t.sizes[i], t.strides[i] = sizes[i], stride
        stride *= sizes[i]
    return t


def _call(name, *args):
    _lib.call(name, *(ctypes.pointer(a) if isinstance(a, _lib.Tensor) else a for a in args))


def _decode_args(**over):
    a = dict(out=_t(2, 8, 128), query=_t(2, 8, 128), kc=_t(9, 2, 16, 16, 8), vc=_t(9, 2, 128, 16), hkv=2, scale=1.0,
             tables=_t(2, 4, dtype=_lib.I32), ctx=_t(2, dtype=_lib.I32), bs=16, max_ctx=64, window=31, sinks=4, alibi=None, ws=None)
    a.update(over)
    return [*a.values(), None]


@pytest.mark.parametrize("over,message", [
    (dict(window=-1), "window_size_left must not be negative"), (dict(sinks=-1), "sink_tokens must not be negative"),
    (dict(query=_t(2, 8, 128, dtype=_lib.F32)), "unsupported data type f32"),
    (dict(query=_t(2, 8, 72), out=_t(2, 8, 72), kc=_t(9, 2, 9, 16, 8), vc=_t(9, 2, 72, 16)), "unsupported head size 72"),
    (dict(hkv=3), "not divisible by 3"), (dict(bs=24), "unsupported block size 24"), (dict(max_ctx=65), "block-table columns"),
    (dict(kc=_t(9, 2, 16, 16, 8, dtype=_lib.F16)), "must share a dtype"), (dict(kc=_t(9, 2, 16, 8, 8)), "key_cache shape"),
    (dict(tables=_t(3, 4, dtype=_lib.I32)), "need 2 rows"), (dict(ctx=_t(2, dtype=_lib.I64)), "must be int32"),
    (dict(alibi=_t(7, dtype=_lib.F32)), "alibi_slopes must be f32"), (dict(ws=_t(100, dtype=_lib.F32)), "workspace must be u8"),
    (dict(out=_t(2, 8, 128, data=0)), "out: data pointer is NULL"),
])
def test_paged_attention_window_refuses(over, message):
    with pytest.raises(_lib.HipAttnError, match=message):
        _call("hipattn_paged_attention_window", *_decode_args(**over))


def _chunk_args(**over):
    a = dict(q=_t(20, 8, 128), kc=_t(9, 2, 16, 16, 8), vc=_t(9, 2, 128, 16), tables=_t(2, 4, dtype=_lib.I32), cu=_t(3, dtype=_lib.I32),
             ctx=_t(2, dtype=_lib.I32), max_q=12, max_k=64, scale=1.0, window=31, sinks=4, out=_t(20, 8, 128), lse=None, ws=None)
    a.update(over)
    return [*a.values(), None]


@pytest.mark.parametrize("over,message", [
    (dict(window=-1), "window_size_left must not be negative"), (dict(sinks=-2), "sink_tokens must not be negative"),
    (dict(q=_t(20, 8, 128, dtype=_lib.F32)), "only fp16 and bf16"), (dict(q=_t(20, 7, 128), out=_t(20, 7, 128)), "not divisible"),
    (dict(max_k=65), "mha_varlen_fwd_paged_window: max_seqlen_k 65 needs more"), (dict(scale=0.0), "softmax_scale must be positive"),
    (dict(ctx=_t(3, dtype=_lib.I32)), "need 2 rows"), (dict(out=_t(19, 8, 128)), "out shape differs"),
    (dict(lse=_t(2, 8, 11, dtype=_lib.F32)), "softmax_lse"), (dict(ws=_t(1 << 20, dtype=_lib.F32)), "workspace must be u8"),
    (dict(ws=_t(16 * 20 * 8 * 130 * 4 - 1, dtype=_lib.U8)), "too small"), (dict(ws=_t(1 << 24, dtype=_lib.U8, data=128)), "256-byte aligned"),
])
def test_flash_attn_varlen_paged_window_refuses(over, message):
    with pytest.raises(_lib.HipAttnError, match=message):
        _call("hipattn_mha_varlen_fwd_paged_window", *_chunk_args(**over))


def _penalty_args(**over):
    f = dict(dtype=_lib.F32)
    a = dict(out=_t(3, 100), logits=_t(3, 100), history=_t(50, dtype=_lib.I32), offsets=_t(4, dtype=_lib.I64), prompt=_t(3, dtype=_lib.I32),
             rep=_t(3, **f), freq=_t(3, **f), pres=_t(3, **f), bias=None, mask=None, rows=None)
    a.update(over)
    return [*a.values(), None]


@pytest.mark.parametrize("over,message", [
    (dict(logits=_t(3, 100, dtype=_lib.I32)), "must be f32/f16/bf16"), (dict(out=_t(3, 100, dtype=_lib.F16)), "type of logits or be f32"),
    (dict(out=_t(3, 99)), "shapes differ"), (dict(history=_t(50, dtype=_lib.I64)), "history must be int32"),
    (dict(offsets=_t(3, dtype=_lib.I64)), "must hold 4 entries"), (dict(prompt=_t(2, dtype=_lib.I32)), r"prompt_lens must be int32 \[3\]"),
    (dict(rep=_t(2, dtype=_lib.F32)), r"repetition must be f32 \[3\]"), (dict(pres=_t(3)), "presence must be f32"),
    (dict(bias=_t(3, 99, dtype=_lib.F32)), "bias rows have 99"), (dict(bias=_t(2, 100, dtype=_lib.F32)), "2 bias or mask rows"),
    (dict(mask=_t(3, 16, dtype=_lib.I32)), "mask must be u8"), (dict(mask=_t(1, 16, dtype=_lib.U8), rows=_t(2, dtype=_lib.I32)), "bias_rows"),
    (dict(mask=_t(0, 16, dtype=_lib.U8), rows=_t(3, dtype=_lib.I32)), "0 bias or mask rows"),
    (dict(logits=_t(3, 100, data=65536), out=_t(3, 100, data=65536 + 32)), "must be logits or lie apart"),
    (dict(logits=_t(3, 100, data=65536), out=_t(3, 100, dtype=_lib.F32, data=65536)), "must be logits or lie apart"),
    (dict(logits=_t(3, 100, data=65536), out=_t(3, 100, dtype=_lib.F32, data=1 << 20), bias=_t(3, 100, dtype=_lib.F32, data=1 << 20)),
     "over an input other than logits"),
    (dict(logits=_t(3, 100, data=65536), out=_t(3, 100, data=1 << 20), history=_t(50, dtype=_lib.I32, data=(1 << 20) + 400)),
     "over an input other than logits"),
])
def test_penalize_logits_refuses(over, message):
    with pytest.raises(_lib.HipAttnError, match=message):
        _call("hipattn_penalize_logits", *_penalty_args(**over))


def _step_args(**over):
    i, w = dict(dtype=_lib.I32), dict(dtype=_lib.I64)
    a = dict(new=_t(5, **i), state=_t(5, 2, **i), tables=_t(5, 8, **i), ring=_t(30, **i), ends=_t(2, **w), bs=16, per=0, window=-1, sinks=0,
             state_out=_t(5, 2, **i), ends_out=_t(2, **w), served=_t(5, **i), ctx=_t(5, **i), cu=_t(6, **i), last=_t(5, **i), pos=_t(9, **w),
             slots=_t(9, **i), totals=_t(4, **i), work=_t(24, **i))
    for n, t in enumerate(a.values()):  # each in a KB of its own
        if isinstance(t, _lib.Tensor):
            t.data = 1024 * (n + 1)
    a.update(over)
    return [*a.values(), None]


@pytest.mark.parametrize("over,message", [
    (dict(new=_t(0, dtype=_lib.I32)), "no requests"), (dict(new=_t(5000, dtype=_lib.I32)), "at most 4096"), (dict(bs=12), "unsupported block size"),
    (dict(per=2), "5 requests of 2 rows each do not fit 9 rows"), (dict(per=-1), "must not be negative"), (dict(sinks=-1), "must not be negative"),
    (dict(state=_t(5, 3, dtype=_lib.I32)), "state has the wrong shape"), (dict(tables=_t(4, 8, dtype=_lib.I32)), "block_tables needs 5 rows"),
    (dict(ring=_t(0, dtype=_lib.I32)), "there are none"), (dict(ring=_t(1 << 28, dtype=_lib.I32)), "do not fit 32 bits"),
    (dict(ends=_t(2, dtype=_lib.I32)), "must be int64"), (dict(cu=_t(5, dtype=_lib.I32)), "seqlens_q has the wrong shape"),
    (dict(slots=_t(8, dtype=_lib.I32)), "slot_mapping has the wrong shape"), (dict(pos=_t(0, dtype=_lib.I64)), "0 rows"),
    (dict(work=_t(20, dtype=_lib.I32)), "workspace has the wrong shape"),
    (dict(state_out=_t(5, 2, dtype=_lib.I32, data=2048 + 16)), "must be state and ring_ends or lie apart"),
    (dict(state_out=_t(5, 2, dtype=_lib.I32, data=1024)), "over another input"), (dict(ends_out=_t(2, dtype=_lib.I64, data=2048)), "over another input"),
    (dict(served=_t(5, dtype=_lib.I32, data=1024 + 8)), "an output lies over an input"), (dict(state_out=_t(5, 2, dtype=_lib.I32, data=260)), "8-byte aligned"),
])
def test_step_blocks_refuses(over, message):
    with pytest.raises(_lib.HipAttnError, match=message):
        _call("hipattn_step_blocks", *_step_args(**over))


def test_varlen_attn_refuses_sinks_without_a_window():
    x = torch.zeros((1, 1, 8))
    with pytest.raises(ValueError, match="needs a window"):
        attn.varlen_attn(x, x, x, None, x, x, sink_tokens=4)


def test_varlen_attn_refuses_a_workspace_without_a_window():
    x = torch.zeros((1, 1, 8))
    with pytest.raises(ValueError, match="workspace needs a window"):
        attn.varlen_attn(x, x, x, None, x, x, workspace=x)


@pytest.mark.parametrize("args,message", [
    ((4, 8, 2, 72, 16, 100, 31, 4), "unsupported head size 72"), ((4, 8, 3, 64, 16, 100, 31, 4), "not divisible"),
    ((4, 8, 2, 64, 12, 100, 31, 4), "unsupported block size 12"), ((4, 8, 2, 64, 16, 100, -1, 4), "must not be negative"),
    ((-1, 8, 2, 64, 16, 100, 31, 4), "negative size"),
])
def test_paged_attention_window_workspace_size_refuses(args, message):
    with pytest.raises(_lib.HipAttnError, match=message):
        _lib.call("hipattn_paged_attention_window_workspace_size", *args, _lib.BF16, ctypes.byref(ctypes.c_int64(0)))


def test_chunk_workspace_sizes():
    size = kernels.flash_attn_varlen_paged_window_workspace_size
    assert size(0, 8, 128) == 0 and size(1, 1, 64) == 16 * 66 * 4 and size(2 ** 31 - 1, 2 ** 20, 256) == 64 << 20
    with pytest.raises(_lib.HipAttnError, match="negative or too large"):
        size(-1, 8, 128)
    with pytest.raises(_lib.HipAttnError, match="head size 257"):
        size(4, 8, 257)


@pytest.mark.parametrize("over", [
    dict(q=_t(80000, 8, 128), out=_t(80000, 8, 128)),  # two pieces of 320 MiB
    dict(lse=_t(2, 8, 12, dtype=_lib.F32)), dict(out=_t(20, 8, 128, dtype=_lib.F32)),
    dict(q=_t(20, 8, 160), out=_t(20, 8, 160), kc=_t(9, 2, 20, 16, 8), vc=_t(9, 2, 160, 16)),
])
def test_chunks_ask_for_no_workspace_that_they_cannot_use(over):
    """Without a device the call gets as far as the device."""
    for ws in (_t(0, dtype=_lib.U8, data=0), _t(1000, dtype=_lib.U8)):
        with pytest.raises(_lib.HipAttnError) as e:
            _call("hipattn_mha_varlen_fwd_paged_window", *_chunk_args(ws=ws, **over))
        assert "workspace" not in str(e.value)


def test_chunks_refuse_tables_without_columns():
    """A context on the device that says otherwise would have its blocks read from there."""
    with pytest.raises(_lib.HipAttnError, match="no columns"):
        _call("hipattn_mha_varlen_fwd_paged_window", *_chunk_args(tables=_t(2, 0, dtype=_lib.I32, data=0), max_k=0))


@pytest.mark.parametrize("max_ctx", [2 ** 31 - 1, 2 ** 31 - 15])
def test_paged_attention_refuses_context_bounds_of_31_bits(max_ctx):
    """(rounded up to blocks they leave 32 bits)"""
    with pytest.raises(_lib.HipAttnError, match="block-table columns"):
        _call("hipattn_paged_attention_window", *_decode_args(max_ctx=max_ctx))
    a = _decode_args(max_ctx=max_ctx)
    with pytest.raises(_lib.HipAttnError, match="block-table columns"):
        _call("hipattn_paged_attention_v1", *a[:10], None, None)
