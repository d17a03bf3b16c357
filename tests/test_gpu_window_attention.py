"""Attention with a sliding window and sinks over the paged cache, decode rows and chunks, against a row-by-row restatement in 64 bits over
the keys that are seen and no others.  Everything else in the cache is NaN -- blocks of columns that the window has passed, tokens behind
the context, tokens between the sinks and the window -- and table columns of passed blocks hold numbers that name no block.

Tolerance, per element: the output's own rounding, half a step of |out|; the probabilities, rounded to the cache's type as operands of
the second product, half a step of sum p |v|; and 1e-4 of sum p |v| for scores and sums in fp32 (128 products of up to 6 x 6 x scale, 2^-24 each,
in the exponent; some thousand terms in the sums)."""
import math
import re

import numpy as np
import pytest
import torch

from aici_amd import attn, kernels as K
from aici_amd import workloads as W
from aici_amd._lib import HipAttnError
from aici_amd.kernels import _native
from oracle import steps
from tests.common import make_cache

pytestmark = pytest.mark.gpu
NAN = float("nan")


def bound(out, mass, dtype, rounded=True):
    half = torch.finfo(dtype).eps / 2
    return 1.01 * half * (mass + (out.abs() if rounded else 0)) + 1e-4 * mass + 1e-6


def case(seed, lens_q, ctx, heads, dtype, window, sinks, bs=16):
    """A cache that holds what some new token sees, and NaN in every other place; columns of blocks with nothing to see name no block."""
    hq, hkv, d = heads
    g = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-c // bs) for c in ctx))
    blocks = sum(-(-c // bs) for c in ctx) + 3
    perm = torch.randperm(blocks, generator=g).tolist()
    kc, vc = make_cache(blocks, hkv, d, bs, dtype, fill=NAN)
    tables = torch.zeros((len(ctx), width), dtype=torch.int32)
    junk = [-1, blocks, 2 ** 31 - 1, -(2 ** 31), blocks + 7]
    for b, (lq, lk) in enumerate(zip(lens_q, ctx)):
        first = max(lk - lq, 0) - window  # what the first new token still sees
        used = [j for j in range(lk) if j >= first or j < sinks] if lq else []
        cols = {j // bs for j in used}
        for c in range(-(-lk // bs)):
            tables[b, c] = perm.pop() if c in cols else junk[c % len(junk)]
        for j in used:
            block = int(tables[b, j // bs])
            kc[block, :, :, j % bs, :] = torch.randn((hkv, d // 8, 8), generator=g).to(dtype)
            vc[block, :, :, j % bs] = torch.randn((hkv, d), generator=g).to(dtype)
    q = torch.randn((sum(lens_q), hq, d), generator=g).to(dtype)
    return dict(q=q, kc=kc, vc=vc, tables=tables, lens_q=lens_q, ctx=ctx, scale=1.0 / math.sqrt(d), window=window, sinks=sinks, bs=bs,
                heads=heads, dtype=dtype)


def want(c, alibi=None):
    return steps.window_attention(c["q"], c["kc"], c["vc"], c["tables"], c["lens_q"], c["ctx"], c["scale"], c["window"], c["sinks"], alibi)


def decode(c, device, alibi=None, workspace=None, out=None, q=None):
    q = c["q"].to(device) if q is None else q
    out = torch.full_like(q, NAN) if out is None else out
    K.paged_attention_window(out, q, c["kc"].to(device), c["vc"].to(device), c["heads"][1], c["scale"], c["tables"].to(device),
                             torch.tensor(c["ctx"], dtype=torch.int32, device=device), c["bs"], c["tables"].size(1) * c["bs"], c["window"],
                             c["sinks"], None if alibi is None else alibi.to(device), workspace)
    return out


def chunk(c, device, **kw):
    return K.flash_attn_varlen_paged_window(c["q"].to(device), c["kc"].to(device), c["vc"].to(device), c["tables"].to(device),
                                            W.offsets(c["lens_q"]).to(device), torch.tensor(c["ctx"], dtype=torch.int32, device=device),
                                            max(c["lens_q"]), max(c["ctx"]), c["scale"], c["window"], c["sinks"], **kw)


def check(got, c, expect, rounded=True):
    out, mass, _ = expect
    got = got.cpu().double()
    assert not torch.isnan(got).any()
    over = (got - out).abs() - bound(out, mass, c["dtype"], rounded)
    assert float(over.max()) <= 0, f"largest excess {float(over.max()):.3g}"


CTX = [1, 0, 2, 15, 16, 17, 31, 33, 64, 100, 129, 257, 300, 511]


@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 4, 80), (6, 1, 96), (12, 4, 112), (32, 8, 128), (34, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bs", [8, 16, 32])
def test_decode(device, heads, dtype, bs):
    for n, (window, sinks) in enumerate([(0, 0), (0, 1), (30, 4), (127, 0), (100, 33), (200, 64), (1000, 5), (31, 600)]):
        c = case(100 + n, [1] * len(CTX), CTX, heads, dtype, window, sinks, bs)
        check(decode(c, device), c, want(c))


@pytest.mark.parametrize("launch", ["flat", "partitioned", "partitions of two blocks"])
def test_decode_launches(device, tuning, launch):
    """Long windows in every launch strategy, with many partitions and few."""
    tuning("decode_flat", 1 if launch == "flat" else 0)
    if launch == "partitions of two blocks":
        tuning("decode_part_blocks", 2)
    for dtype, heads, bs in ((torch.bfloat16, (8, 2, 128), 16), (torch.float16, (12, 4, 112), 8), (torch.bfloat16, (4, 2, 64), 32)):
        c = case(7, [1] * 6, [700, 1, 2500, 33, 0, 1999], heads, dtype, 1100, 37, bs)
        check(decode(c, device), c, want(c))


def test_decode_takes_the_same_keys_whatever_the_block_size(device):
    outs = []
    for bs in (8, 16, 32):
        c = case(11, [1] * 3, [900, 64, 333], (8, 2, 128), torch.bfloat16, 250, 20, 16)
        # the same tokens moved into blocks of bs
        kc, vc = make_cache(200, 2, 128, bs, torch.bfloat16, fill=NAN)
        tables = torch.full((3, -(-900 // bs)), -1, dtype=torch.int32)
        nxt = 0
        for b, n in enumerate(c["ctx"]):
            for j in steps.seen(n - 1, 250, 20):
                if tables[b, j // bs] < 0:
                    tables[b, j // bs] = nxt
                    nxt += 1
                kc[tables[b, j // bs], :, :, j % bs] = c["kc"][c["tables"][b, j // 16], :, :, j % 16]
                vc[tables[b, j // bs], :, :, j % bs] = c["vc"][c["tables"][b, j // 16], :, :, j % 16]
        c.update(kc=kc, vc=vc, tables=tables, bs=bs)
        outs.append(decode(c, device))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[1], outs[2])


def test_decode_alibi_and_strides_and_unwritten_rows(device):
    c = case(12, [1] * 4, [40, 300, 17, 129], (8, 2, 128), torch.float16, 60, 5)
    alibi = torch.linspace(-0.3, -0.01, 8)
    wide = torch.full((4, 3 * 8 * 128), NAN, dtype=torch.float16, device=device)
    q = wide[:, 1024:2048].view(4, 8, 128)
    q.copy_(c["q"])
    frame = torch.full((6, 8, 128), 7.0, dtype=torch.float16, device=device)
    out = decode(c, device, alibi=alibi, q=q, out=frame[1:5])
    check(out, c, want(c, alibi))
    assert bool((frame[0] == 7).all()) and bool((frame[5] == 7).all())


def test_a_window_over_everything_is_paged_attention(device):
    d = W.decode_inputs(5, 5, 1, 700, 8, 2, 128, torch.bfloat16, 300).to(device)
    args = (d.q, d.key_cache, d.value_cache, 2, d.scale, d.block_tables, d.context_lens, 16, d.max_ctx)
    a, b = torch.empty_like(d.q), torch.empty_like(d.q)
    K.paged_attention_v1(a, *args)
    K.paged_attention_window(b, *args, 5000, 3)
    assert torch.equal(a, b)


SEQS = [(5, 5), (64, 64), (33, 133), (0, 20), (1, 18), (200, 200), (65, 700), (16, 31), (130, 400), (9, 5)]


@pytest.mark.parametrize("heads", [(4, 2, 8), (4, 4, 32), (4, 2, 40), (8, 2, 64), (4, 4, 80), (6, 1, 96), (12, 4, 112), (16, 2, 128), (4, 2, 160),
                                   (2, 1, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bs", [16, 8, 32])
def test_chunks(device, tuning, heads, dtype, bs):
    for n, (window, sinks) in enumerate([(0, 0), (30, 4), (63, 64), (100, 33), (255, 100), (2000, 5)]):
        c = case(200 + n, [a for a, _ in SEQS], [b for _, b in SEQS], heads, dtype, window, sinks, bs)
        expect = want(c)
        # block images in workgroups of four and eight wavefronts, tiles through registers, and what the library picks: for most of these
        # sizes the kernel of decode rows
        for kernel, images in ((5, -1), (1, -1), (5, 0), (0, -1)) if heads[2] in (32, 64, 80, 96, 112, 128) else ((5, -1), (0, -1)):
            tuning("prefill_kernel", kernel)
            tuning("paged_prefill_dma", images)
            check(chunk(c, device), c, expect)


@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 2, 96), (8, 2, 128)])
def test_long_chunks(device, tuning, heads):
    """Windows of many tiles with sinks of more than one, and the staged route."""
    for window, sinks, lens_q, ctx in ((700, 70, [100, 300], [2100, 1300]), (1023, 4, [40], [1800]), (64, 200, [257], [900])):
        for bs in (16, 8, 32):
            c = case(31, lens_q, ctx, heads, torch.bfloat16, window, sinks, bs)
            expect = want(c)
            for kernel in (0, 5, 1):
                tuning("prefill_kernel", kernel)
                check(chunk(c, device), c, expect)


@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 4, 80), (6, 1, 96), (12, 4, 112), (8, 2, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_chunks_whose_keys_are_dealt_out(device, heads, dtype):
    """Few rows over long windows: several workgroups share a row block's keys, others of the same batch have too few for that."""
    for n, (window, sinks, lens_q, ctx) in enumerate([(2500, 70, [16], [4000]), (1300, 0, [1, 40, 3, 0, 5], [2000, 1700, 40, 9, 3]),
                                                      (900, 130, [150, 2], [1500, 901])]):
        c = case(300 + n, lens_q, ctx, heads, dtype, window, sinks)
        expect = want(c)
        check(chunk(c, device), c, expect)
        check(chunk(c, device, out_dtype=torch.float32), c, expect, rounded=False)


@pytest.mark.parametrize("heads", [(6, 2, 64), (10, 2, 80), (14, 2, 128), (40, 2, 64), (8, 8, 256)])
def test_few_rows_of_odd_groups(device, heads):
    """Columns that no row of heads fills, more heads in a group than columns, batches with empty sequences; in one part and in several."""
    for n, (window, sinks, lens_q, ctx) in enumerate([(2000, 40, [3, 7], [2600, 900]), (50, 3, [0, 1, 12, 0, 2], [7, 1, 300, 0, 2])]):
        for bs in (16, 8, 32):
            c = case(400 + n, lens_q, ctx, heads, torch.float16, window, sinks, bs)
            check(chunk(c, device), c, want(c))


def test_chunk_outputs_in_fp32_lse_and_rows_behind_the_last(device):
    c = case(41, [70, 1, 0, 9], [300, 40, 12, 5], (8, 2, 128), torch.bfloat16, 90, 10)
    expect = want(c)
    out, lse = chunk(c, device, return_lse=True, out_dtype=torch.float32)
    check(out, c, expect, rounded=False)
    row = 0
    for b, n in enumerate(c["lens_q"]):
        got, ref = lse[b, :, :n].cpu().double(), expect[2][row:row + n].T
        assert torch.equal(torch.isinf(got), torch.isinf(ref))
        fin = ~torch.isinf(ref)
        assert n == 0 or float((got - ref)[fin].abs().max()) < 2e-3  # (the top probability's rounding, half a step of bf16, is in the sum)
        row += n
    assert bool((out[row - 9:row - 5] == 0).all())  # positions before the first key see nothing
    # strided q and out with rows that no sequence owns
    T = c["q"].size(0)
    wide = torch.full((T + 5, 10, 128), NAN, dtype=torch.bfloat16, device=device)
    wide[:T, 1:9] = c["q"].to(device)
    frame = torch.full((T + 5, 12, 128), 7.0, dtype=torch.bfloat16, device=device)
    _native.mha_varlen_fwd_paged_window(wide[:, 1:9], c["kc"].to(device), c["vc"].to(device), c["tables"].to(device),
                                        W.offsets(c["lens_q"]).to(device), torch.tensor(c["ctx"], dtype=torch.int32, device=device), 70, 300,
                                        c["scale"], 90, 10, frame[:, 2:10], None, None)
    check(frame[:T, 2:10], c, expect)
    assert bool((frame[T:] == 7).all()) and bool((frame[:, :2] == 7).all()) and bool((frame[:, 10:] == 7).all())


def test_a_window_over_everything_is_causal_attention(device, tuning):
    tuning("prefill_kernel", 5)  # (keys that are not dealt out: the same bits)
    c = case(51, [100, 64], [500, 64], (8, 2, 128), torch.float16, 10000, 0)
    whole = K.flash_attn_varlen_paged(c["q"].to(device), c["kc"].to(device), c["vc"].to(device), c["tables"].to(device),
                                      W.offsets(c["lens_q"]).to(device), torch.tensor(c["ctx"], dtype=torch.int32, device=device), 100, 500,
                                      c["scale"], True)
    assert torch.equal(chunk(c, device), whole)


def test_composition(device):
    """attn.varlen_attn with a window: chunks and decode rows of one batch, their keys written to the cache by the call."""
    dtype, heads, window, sinks, bs = torch.bfloat16, (8, 2, 128), 50, 6, 16
    lens_q, ctx = [40, 3, 1, 1], [90, 3, 200, 1]
    c = case(61, lens_q, ctx, heads, dtype, window, sinks)
    q, kc, vc = c["q"], c["kc"].clone(), c["vc"].clone()
    new_k, new_v, slots = [], [], []
    for b, (n, lk) in enumerate(zip(lens_q, ctx)):
        for j in range(lk - n, lk):
            block = int(c["tables"][b, j // bs])
            new_k.append(c["kc"][block, :, :, j % bs].reshape(2, 128))
            new_v.append(c["vc"][block, :, :, j % bs])
            slots.append(block * bs + j % bs)
            kc[block, :, :, j % bs] = NAN
            vc[block, :, :, j % bs] = NAN

    class Batch:
        q_multi, max_seqlen_q, max_seqlen_k, paged_block_size, paged_max_context_len = 43, 40, 90, bs, 200
        slot_mapping = torch.tensor(slots, dtype=torch.int32, device=device)
        multi_block_tables, multi_context_lens = c["tables"][:2].to(device), torch.tensor(ctx[:2], dtype=torch.int32, device=device)
        seqlens_q = W.offsets(lens_q[:2]).to(device)
        paged_block_tables, paged_context_lens = c["tables"][2:].to(device), torch.tensor(ctx[2:], dtype=torch.int32, device=device)

    y = attn.varlen_attn(q.to(device), torch.stack(new_k).to(device), torch.stack(new_v).to(device), Batch, kc.to(device), vc.to(device),
                         window_size_left=window, sink_tokens=sinks)
    check(y.view(-1, 8, 128), c, want(c))


def test_streams_workspaces_and_replays(device):
    """Decode on a side stream with a workspace of its own, captured and replayed over new inputs beside eager calls."""
    c = case(71, [1] * 3, [2000, 900, 1500], (8, 2, 128), torch.bfloat16, 1200, 20)
    other = case(72, [1] * 3, [2000, 900, 1500], (8, 2, 128), torch.bfloat16, 1200, 20)
    need = K.paged_attention_window_workspace_size(3, 8, 2, 128, 16, c["tables"].size(1) * 16, 1200, 20, torch.bfloat16)
    assert need > 0
    ws = torch.empty((need,), dtype=torch.uint8, device=device)
    with pytest.raises(HipAttnError, match="too small"):
        decode(c, device, workspace=ws[:need - 256])
    eager = [decode(x, device) for x in (c, other)]
    q, kc, vc, tables = (c[k].to(device) for k in ("q", "kc", "vc", "tables"))
    ctx = torch.tensor(c["ctx"], dtype=torch.int32, device=device)
    out, chunk_out = torch.empty_like(q), torch.empty_like(q)
    cu = W.offsets([1, 1, 1]).to(device)

    def step():
        K.paged_attention_window(out, q, kc, vc, 2, c["scale"], tables, ctx, 16, tables.size(1) * 16, 1200, 20, None, ws)
        chunk_out.copy_(K.flash_attn_varlen_paged_window(q, kc, vc, tables, cu, ctx, 1, 2000, c["scale"], 1200, 20))

    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    assert torch.equal(out, eager[0])
    with torch.cuda.graph(graph, stream=side):
        step()
    for k in range(4):
        x = (other, c)[k % 2]
        for t, n in ((q, "q"), (kc, "kc"), (vc, "vc"), (tables, "tables")):
            t.copy_(x[n])
        out.fill_(NAN)
        chunk_out.fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[(k + 1) % 2])
        check(chunk_out, x, want(x))
        assert torch.equal(decode(x, device), out)


def test_far_blocks(device):
    """Blocks beyond 2^31 elements of the cache."""
    hkv, d, bs = 8, 128, 16
    blocks = (1 << 31) // (hkv * d * bs) + 40  # 4.3 GB of keys, as much of values
    c = case(81, [1, 1], [300, 90], (16, 8, 128), torch.bfloat16, 100, 5)
    small = c["kc"].size(0)
    kc = torch.zeros((blocks, hkv, d // 8, bs, 8), dtype=torch.bfloat16, device=device)
    vc = torch.zeros((blocks, hkv, d, bs), dtype=torch.bfloat16, device=device)
    kc[blocks - small:] = c["kc"].to(device)
    vc[blocks - small:] = c["vc"].to(device)
    tables = torch.where((c["tables"] >= 0) & (c["tables"] < small), c["tables"] + (blocks - small), c["tables"]).to(device)
    ctx = torch.tensor(c["ctx"], dtype=torch.int32, device=device)
    out = torch.full_like(c["q"], NAN).to(device)
    K.paged_attention_window(out, c["q"].to(device), kc, vc, 8, c["scale"], tables, ctx, 16, tables.size(1) * 16, 100, 5)
    expect = want(c)
    check(out, c, expect)
    out = K.flash_attn_varlen_paged_window(c["q"].to(device), kc, vc, tables, W.offsets([1, 1]).to(device), ctx, 1, 300, c["scale"], 100, 5)
    check(out, c, expect)


def test_two_streams_at_once(device):
    """Decode and chunks whose keys are dealt out, on two streams without a wait between them: each has scratch memory of its own."""
    cases = [case(90 + k, [16, 20], [1500, 900 + k], (8, 2, 128), torch.bfloat16, 1200, 20) for k in range(2)]
    rows = [case(95 + k, [1] * 3, [2000, 900, 1500 - k], (8, 2, 128), torch.bfloat16, 1200, 20) for k in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    calls = []
    for c, r in zip(cases, rows):
        to = {n: c[n].to(device) for n in ("q", "kc", "vc", "tables")}
        cu, ctx = W.offsets([16, 20]).to(device), torch.tensor(c["ctx"], dtype=torch.int32, device=device)
        rt = {n: r[n].to(device) for n in ("q", "kc", "vc", "tables")}
        rctx, out = torch.tensor(r["ctx"], dtype=torch.int32, device=device), torch.empty_like(rt["q"])

        def call(c=c, to=to, cu=cu, ctx=ctx, r=r, rt=rt, rctx=rctx, out=out):
            chunk = K.flash_attn_varlen_paged_window(to["q"], to["kc"], to["vc"], to["tables"], cu, ctx, 20, 1500, c["scale"], 1200, 20)
            K.paged_attention_window(out, rt["q"], rt["kc"], rt["vc"], 2, r["scale"], rt["tables"], rctx, 16, rt["tables"].size(1) * 16,
                                     1200, 20)
            return chunk, out.clone()

        calls.append(call)
    alone = [call() for call in calls]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for call, stream in zip(calls, streams):
            with torch.cuda.stream(stream):
                got.append(call())
    torch.cuda.synchronize()
    for k, (chunk, out) in enumerate(got):
        assert torch.equal(chunk, alone[k % 2][0]) and torch.equal(out, alone[k % 2][1])
    for (chunk, out), c, r in zip(alone, cases, rows):
        check(chunk, c, want(c))
        check(out, r, want(r))


@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 2, 160), (4, 2, 128), (40, 2, 64)])
def test_one_long_chunk_among_many_short_ones(device, tuning, heads):
    """More sequences than lanes, of none to a few new tokens, and one of many: row blocks lie one sequence behind the other in the launch."""
    for n, (long, window, sinks) in enumerate([(200, 60, 10), (9, 40, 3)]):
        lens_q = [3, 0, 1] * 22 + [0] * 64 + [long] + [2, 1, 0] * 3
        ctx = [a + (7 * k) % 90 for k, a in enumerate(lens_q)]
        c = case(500 + n, lens_q, ctx, heads, torch.bfloat16, window, sinks)
        expect = want(c)
        for kernel, images in ((0, -1), (5, -1), (1, -1), (5, 0)):
            tuning("prefill_kernel", kernel)
            tuning("paged_prefill_dma", images)
            check(chunk(c, device), c, expect)
        tuning("prefill_kernel", 0)
        tuning("paged_prefill_dma", -1)
        bare = [c[k].to(device) for k in ("q", "kc", "vc", "tables")]
        tail = torch.cat([bare[0], torch.full((150, *bare[0].shape[1:]), NAN, dtype=torch.bfloat16, device=device)])
        out = torch.full_like(tail, 5.0)
        # rows behind the last sequence, and a bound that no sequence reaches
        _native.mha_varlen_fwd_paged_window(tail, *bare[1:], W.offsets(lens_q).to(device), torch.tensor(ctx, dtype=torch.int32, device=device),
                                            long + 300, bare[3].size(1) * 16, c["scale"], window, sinks, out, None, None)
        check(out[:-150], c, expect)
        assert bool((out[-150:] == 5).all())


@pytest.mark.parametrize("heads,lens_q,ctx", [((8, 2, 64), [16], [4000]), ((8, 2, 128), [40, 300], [2600, 2900]), ((8, 2, 256), [3, 9], [2600, 2000])])
def test_chunks_with_a_workspace_of_the_callers(device, heads, lens_q, ctx):
    """The same bits as with the library's buffer, eager, captured without a call before, and replayed."""
    c, other = (case(600 + k, lens_q, ctx, heads, torch.bfloat16, 2500, 30) for k in range(2))
    need = K.flash_attn_varlen_paged_window_workspace_size(sum(lens_q), heads[0], heads[2])
    assert need == min(16 * sum(lens_q) * heads[0] * (heads[2] + 2) * 4, 64 << 20)
    store = torch.full((need + 512,), 255, dtype=torch.uint8, device=device)  # (NaN, read as fp32)
    with pytest.raises(HipAttnError, match="too small"):
        chunk(c, device, workspace=store[:need - 1])
    alone = [chunk(x, device) for x in (c, other)]
    check(alone[0], c, want(c))
    q, kc, vc, tables = (c[k].to(device) for k in ("q", "kc", "vc", "tables"))
    cu, lk = W.offsets(lens_q).to(device), torch.tensor(ctx, dtype=torch.int32, device=device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        out = K.flash_attn_varlen_paged_window(q, kc, vc, tables, cu, lk, max(lens_q), max(ctx), c["scale"], 2500, 30, workspace=store[:need])
    for k in range(4):
        x = (other, c)[k % 2]
        for t, n in ((q, "q"), (kc, "kc"), (vc, "vc"), (tables, "tables")):
            t.copy_(x[n])
        out.fill_(NAN)
        store.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, alone[(k + 1) % 2])
        assert torch.equal(chunk(x, device, workspace=store[:need]), out)
        assert bool((store[need:] == 255).all())


@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("kernel", [0, 5])
def test_contexts_beyond_the_bound(device, tuning, heads, kernel):
    """A sequence with more keys than max_seqlen_k: some of them may be left out, and nothing else changes -- not the other sequences, not
    the caller's workspace behind what the call needs.  With a bound that one part holds, and with one that several do."""
    tuning("prefill_kernel", kernel)
    for bound_k, lens_q, ctx in ((64, [3, 5], [2000, 40]), (1500, [2, 7, 1], [2900, 1400, 1500])):
        c = case(700 + bound_k, lens_q, ctx, heads, torch.bfloat16, 3000, 5)
        bare = [c[k].to(device) for k in ("q", "kc", "vc", "tables")]
        need = K.flash_attn_varlen_paged_window_workspace_size(sum(lens_q), heads[0], heads[2])
        for store in (None, torch.full((need + 4096,), 255, dtype=torch.uint8, device=device)):
            out = K.flash_attn_varlen_paged_window(*bare, W.offsets(lens_q).to(device), torch.tensor(ctx, dtype=torch.int32, device=device),
                                                   max(lens_q), bound_k, c["scale"], 3000, 5, workspace=None if store is None else store[:need])
            first = lens_q[0]
            assert bool((out[:first].abs() <= 1.01 * bare[2].nan_to_num(0).abs().max()).all())  # (no NaN: an average of some values)
            expect, mass, _ = want(c)
            check(out[first:], c, (expect[first:], mass[first:], None))
            assert store is None or bool((store[need:] == 255).all())


@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (8, 8, 256)])
def test_rows_beyond_the_bound(device, heads):
    """A sequence with more new tokens than max_seqlen_q: a row beyond is left as it was or right, never made of scratch memory."""
    lens_q, ctx, bound_q = [40, 3, 8], [2600, 900, 2000], 8
    c = case(750, lens_q, ctx, heads, torch.bfloat16, 2500, 30)
    bare = [c[k].to(device) for k in ("q", "kc", "vc", "tables")]
    expect, mass, _ = want(c)
    need = K.flash_attn_varlen_paged_window_workspace_size(sum(lens_q), heads[0], heads[2])
    for store in (None, torch.full((need,), 255, dtype=torch.uint8, device=device)):  # (NaN, read as fp32)
        out = torch.full_like(bare[0], 7.0)
        _native.mha_varlen_fwd_paged_window(*bare, W.offsets(lens_q).to(device), torch.tensor(ctx, dtype=torch.int32, device=device), bound_q,
                                            max(ctx), c["scale"], 2500, 30, out, None, store)
        left = (out == 7).flatten(1).all(1).cpu()
        assert not bool(left[:bound_q].any()) and not bool(left[40:].any())
        check(out[~left], c, (expect[~left], mass[~left], None))


@pytest.mark.parametrize("kernel,images,heads", [(5, -1, (8, 2, 64)), (1, -1, (8, 2, 128)), (5, 0, (8, 2, 128)), (0, -1, (4, 2, 160))])
def test_lse_of_rows_beyond_the_bound(device, tuning, kernel, images, heads):
    """An LSE holds max_seqlen_q rows a head: a sequence with more new tokens writes nothing into the next head's, or behind the last."""
    tuning("prefill_kernel", kernel)
    tuning("paged_prefill_dma", images)
    lens_q, ctx, bound_q = [8, 3, 50], [60, 90, 200], 8
    c = case(760, lens_q, ctx, heads, torch.bfloat16, 100, 3)
    bare = [c[k].to(device) for k in ("q", "kc", "vc", "tables")]
    expect = want(c)
    for dtype in (torch.bfloat16, torch.float32):
        frame = torch.full((3 * heads[0] * bound_q + 256,), 7.0, dtype=torch.float32, device=device)
        lse = frame[:3 * heads[0] * bound_q].view(3, heads[0], bound_q)
        out = torch.full_like(bare[0], 7.0, dtype=dtype)
        _native.mha_varlen_fwd_paged_window(*bare, W.offsets(lens_q).to(device), torch.tensor(ctx, dtype=torch.int32, device=device), bound_q,
                                            max(ctx), c["scale"], 100, 3, out, lse, None)
        assert bool((frame[lse.numel():] == 7).all())
        row = 0
        for b, n in enumerate(lens_q):
            n = min(n, bound_q)
            assert float((lse[b, :, :n].cpu().double() - expect[2][row:row + n].T).abs().max()) < 2e-3
            assert bool((lse[b, :, n:] == 7).all())
            row += lens_q[b]


@pytest.mark.parametrize("heads", [(8, 2, 64), (16, 1, 128), (4, 2, 160)])
def test_bounds_of_31_bits(device, tuning, heads):
    """max_seqlen_q far beyond the rows there are, as the header allows: the launch is one over those there are."""
    lens_q, ctx = [3, 70, 1], [30, 400, 90]
    c = case(770, lens_q, ctx, heads, torch.bfloat16, 150, 3)
    bare = [c[k].to(device) for k in ("q", "kc", "vc", "tables")]
    expect = want(c)
    for kernel in (0, 5, 1):
        tuning("prefill_kernel", kernel)
        for bound in (2 ** 31 - 1, 2 ** 31 - 64):
            out = K.flash_attn_varlen_paged_window(*bare, W.offsets(lens_q).to(device), torch.tensor(ctx, dtype=torch.int32, device=device),
                                                   bound, max(ctx), c["scale"], 150, 3)
            check(out, c, expect)


class Mixed:
    """A batch of chunks and decode rows for attn.varlen_attn, on the device."""

    def __init__(self, seed, heads, chunks, rows, window, sinks, device):
        (self.lens_q, self.ctx), (hq, hkv, d) = zip(*chunks, *[(1, n) for n in rows]), heads
        self.c = case(seed, list(self.lens_q), list(self.ctx), heads, torch.bfloat16, window, sinks)
        m, T = len(chunks), sum(self.lens_q)
        lens = torch.tensor(self.ctx, dtype=torch.int32, device=device)
        self.tokens, self.q_multi = torch.zeros((T,), dtype=torch.int32), T - len(rows)
        self.max_seqlen_q, self.max_seqlen_k = max(self.lens_q), max(self.ctx[:m])
        self.seqlens_q, self.multi_context_lens, self.paged_context_lens = W.offsets(list(self.lens_q[:m])).to(device), lens[:m], lens[m:]
        self.paged_block_size, self.paged_max_context_len = 16, max(rows)
        self.q, self.kc, self.vc, tables = (self.c[k].to(device) for k in ("q", "kc", "vc", "tables"))
        self.multi_block_tables, self.paged_block_tables = tables[:m], tables[m:]
        self.kv = torch.zeros((T, hkv, d), dtype=torch.bfloat16, device=device)
        self.how = dict(window_size_left=window, sink_tokens=sinks)

    def attend(self, workspace=None):
        return attn.varlen_attn(self.q, self.kv, self.kv, self, self.kc, self.vc, cached=True, workspace=workspace, **self.how)

    def workspace(self, device):
        hq, hkv, d = self.c["heads"]
        need = attn.window_workspace_size(self, hq, hkv, d, torch.bfloat16, *self.how.values())
        return torch.full((need,), 255, dtype=torch.uint8, device=device)  # (NaN, read as fp32)

    def check(self, y):
        check(y.view(self.c["q"].shape), self.c, want(self.c))


def test_captured_composition_with_a_workspace(device):
    """Chunks whose keys are dealt out and decode rows in partitions: captured with a workspace the composed call gives the eager call's bits, and
    two graphs captured on one stream, each with its own, run at the same time."""
    made = [Mixed(800 + k, (8, 2, 128), [(16, 3000), (5, 900 + k)], [2000, 1500 - k, 40], 2500, 20, device) for k in range(2)]
    alone = [b.attend() for b in made]
    stores = [b.workspace(device) for b in made]
    assert stores[0].numel() > 0
    for b, y, store in zip(made, alone, stores):
        b.check(y)
        assert torch.equal(b.attend(store), y) and not bool((store == 255).all())  # (made use of)
        store.fill_(255)
    with pytest.raises(HipAttnError, match="too small"):
        made[0].attend(stores[0][:4096])
    side, graphs, outs = torch.cuda.Stream(), [], []
    torch.cuda.synchronize()
    for b, store in zip(made, stores):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(b.attend(store))
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(4):
        for out, store in zip(outs, stores):
            out.fill_(NAN)
            store.fill_(255)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for b, out, y in zip(made, outs, alone):
            assert torch.equal(out, y) and torch.equal(b.attend(), y)


def launched(call):
    """Names of the kernels that a call launches."""
    call()
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        call()
        torch.cuda.synchronize()
    return [e.key for e in prof.key_averages() if "kernel" in e.key]


@pytest.mark.filterwarnings("ignore:Profiler clears events")
@pytest.mark.parametrize("heads,lens_q,past,window,form", [
    ((32, 8, 128), [2000], 4096, 4096, 8), ((32, 32, 80), [1000, 1000], 3000, 2500, 8), ((16, 2, 96), [4000], 4096, 4096, 8),
    ((32, 8, 128), [2000], 0, 4096, 4),         # the first rows of a prompt have short chains
    ((32, 8, 128), [4096, 4096], 4096, 4096, 4), ((64, 8, 128), [4096], 4096, 4096, 4),  # several rounds of workgroups
    ((24, 8, 96), [2600], 4096, 4096, 4), ((16, 2, 64), [4000], 4096, 4096, 4),
    ((32, 8, 128), [2100], 4096, 4096, 4),      # a few more than one to a compute unit
])
def test_the_form_of_the_workgroups(device, heads, lens_q, past, window, form):
    hq, hkv, d = heads
    cols = -(-(max(lens_q) + past) // 16)
    q = torch.zeros((sum(lens_q), hq, d), dtype=torch.bfloat16, device=device)
    kc = torch.zeros((len(lens_q) * cols, hkv, d // 8, 16, 8), dtype=torch.bfloat16, device=device)
    vc = torch.zeros((len(lens_q) * cols, hkv, d, 16), dtype=torch.bfloat16, device=device)
    tables = torch.arange(len(lens_q) * cols, dtype=torch.int32, device=device).view(-1, cols)
    ctx = [n + past for n in lens_q]
    args = (q, kc, vc, tables, W.offsets(lens_q).to(device), torch.tensor(ctx, dtype=torch.int32, device=device), max(lens_q), max(ctx), 0.1)
    names = launched(lambda: K.flash_attn_varlen_paged_window(*args, window, 4))
    assert len(names) == 1 and "prefill_varlen_w8_kernel" in names[0], names
    assert int((re.search(r", (\d+)>\(", names[0]) or re.search(r"Li(\d+)EEEv", names[0])).group(1)) == form


PIECES = [(64, 2), (80, 4), (96, 1), (112, 4), (128, 2)]  # head size, kv heads


@pytest.mark.parametrize("d,hkv", PIECES)
@pytest.mark.parametrize("parts,bs", [(2, 16), (3, 8), (5, 32), (16, 16)])
def test_pieces_of_a_row_blocks_keys(device, tuning, d, hkv, bs, parts):
    """Keys of a row block dealt out to as many workgroups as asked for: pieces that begin in the sinks, in the gap and in the window, blocks with fewer
    tiles than pieces, rows that see nothing of a piece or nothing at all, passed blocks that name no block; whatever the scratch memory held."""
    tuning("window_parts", parts)
    dtype = torch.float16 if parts == 3 else torch.bfloat16
    heads = ((6 if d == 96 else 2 * hkv) if d != 80 else hkv, hkv, d)
    sets = [(SEQS, 255, 100), (SEQS, 63, 64), ([(100, 2100), (300, 1300), (9, 5), (0, 40), (1, 1)], 700, 70), ([(257, 900)], 64, 200),
            ([(3, 1100), (0, 0)] * 40 + [(200, 1500)], 1000, 0)]  # the last: listed row blocks, more sequences than lanes
    for n, (seqs, window, sinks) in enumerate(sets):
        lens_q, ctx = [a for a, _ in seqs], [b for _, b in seqs]
        c = case(900 + n, lens_q, ctx, heads, dtype, window, sinks, bs)
        need = K.flash_attn_varlen_paged_window_workspace_size(sum(lens_q), heads[0], d)
        store = torch.full((need + 4096,), 255, dtype=torch.uint8, device=device)  # (NaN, read as fp32)
        out = chunk(c, device, workspace=store[:need])
        check(out, c, want(c))
        assert bool((store[need:] == 255).all()) and not bool((store[:need] == 255).all())
        assert torch.equal(chunk(c, device), out)


@pytest.mark.filterwarnings("ignore:Profiler clears events")
@pytest.mark.parametrize("heads,rows,bs", [((16, 2, 64), 300, 16), ((32, 32, 80), 300, 8), ((6, 1, 96), 600, 16), ((12, 4, 112), 300, 32),
                                           ((8, 2, 128), 300, 16), ((8, 2, 128), 300, 8)])
def test_pieces_that_the_library_chooses(device, heads, rows, bs):
    """Chunks of some hundred rows over long windows, which the library itself deals out this way."""
    for lens_q, ctx in (([rows], [4000 + rows]), ([rows, 150], [4000 + rows, 4000])):
        c = case(950, lens_q, ctx, heads, torch.bfloat16, 4000, 33, bs)
        to = {n: c[n].to(device) for n in ("q", "kc", "vc", "tables")}
        cu, lk = W.offsets(lens_q).to(device), torch.tensor(ctx, dtype=torch.int32, device=device)
        call = lambda: K.flash_attn_varlen_paged_window(*to.values(), cu, lk, max(lens_q), max(ctx), c["scale"], 4000, 33)
        out = call()
        check(out, c, want(c))
        if len(lens_q) == 1:
            names = launched(call)
            assert len(names) == 2 and any("window_merge_kernel" in n for n in names), names


@pytest.mark.parametrize("heads", [(16, 2, 64), (8, 2, 128)])
def test_pieces_of_bounds_that_do_not_hold(device, tuning, heads):
    """More new tokens than max_seqlen_q, more keys than max_seqlen_k, and two graphs with a workspace each: as without pieces."""
    tuning("window_parts", 4)
    lens_q, ctx = [400, 3, 8], [2600, 900, 2000]
    c = case(960, lens_q, ctx, heads, torch.bfloat16, 2500, 30)
    bare = [c[k].to(device) for k in ("q", "kc", "vc", "tables")]
    expect, mass, _ = want(c)
    cu, lk = W.offsets(lens_q).to(device), torch.tensor(ctx, dtype=torch.int32, device=device)
    store = torch.full((K.flash_attn_varlen_paged_window_workspace_size(sum(lens_q), heads[0], heads[2]),), 255, dtype=torch.uint8, device=device)
    for bound_q, bound_k in ((100, 2600), (400, 700)):
        store.fill_(255)
        out = torch.full_like(bare[0], 7.0)
        _native.mha_varlen_fwd_paged_window(*bare, cu, lk, bound_q, bound_k, c["scale"], 2500, 30, out, None, store)
        left = (out == 7).flatten(1).all(1).cpu()
        assert not bool(left[:bound_q].any()) and not bool(left[400:].any()) and bool(left[:400].any()) == (bound_q < 400)
        check(out[~left], c, (expect[~left], mass[~left], None))  # (this kernel's last piece takes the keys beyond the bound)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        out = K.flash_attn_varlen_paged_window(*bare, cu, lk, 400, 2600, c["scale"], 2500, 30, workspace=store)
    first = chunk(c, device)
    for _ in range(3):
        store.fill_(255)
        out.fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first) and torch.equal(chunk(c, device), first)
