"""The operators of a generation step that stays on the device over a sliding window, as cases that can be timed and compared.

Kinds of case:

  window_decode  one new token per sequence against the last `window` + 1 tokens of its paged context and its first `sinks`
                 tokens (`kernels.paged_attention_window`).
  window_chunk   several new tokens per sequence, causal, with the same window and sinks, over the paged cache
                 (`kernels.flash_attn_varlen_paged_window`).
  step_blocks    the block tables, slots and positions of a step made on the device from how many tokens every request brings:
                 blocks behind the window and of requests that have ended go back to the pool, new ones come from it
                 (`kernels.step_blocks`).
  penalties      repetition, frequency and presence penalties over what a sequence has said, the controller's bias and its
                 packed allow-mask, on a batch's logits (`kernels.penalize_logits`).

`own` picks the framework's calls; otherwise the same is computed in its plain form.  Lengths come from the case alone (spread
evenly over its range); the seed of `prepare` gives their order, the values and the order of the blocks in the pool.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
WIDE, ODD, NARROW, PHI2 = (32, 8, 128), (12, 4, 112), (16, 2, 64), (32, 32, 80)
HEADS = (WIDE, ODD, NARROW, PHI2)
VOCAB = 128256


def _heads(shape):
    return {"query_heads": shape[0], "kv_heads": shape[1], "head_size": shape[2]}


def listed():
    return [
        # A single chat over a short window: where latency counts.
        {"name": "window_decode_1", "kind": "window_decode", "dtype": "bf16", **_heads(WIDE), "block": 16, "rows": 1, "ctx_lo": 1500,
         "ctx_hi": 1500, "window": 1023, "sinks": 4},
        # A small batch of narrower heads, some contexts shorter than the window, one of a single token.
        {"name": "window_decode_48", "kind": "window_decode", "dtype": "fp16", **_heads(ODD), "block": 16, "rows": 48, "ctx_lo": 1,
         "ctx_hi": 2111, "window": 511, "sinks": 17},
        # A full server: long conversations, of which each step reads 4096 tokens and the sinks.
        {"name": "window_decode_128", "kind": "window_decode", "dtype": "bf16", **_heads(WIDE), "block": 16, "rows": 128,
         "ctx_lo": 1024, "ctx_hi": 16384, "window": 4095, "sinks": 4},
        # A follow-up question of one conversation, over a window of a few blocks.
        {"name": "window_chunk_1", "kind": "window_chunk", "dtype": "bf16", **_heads(WIDE), "block": 16, "seqs": 1, "new_lo": 45,
         "new_hi": 45, "prior_lo": 700, "prior_hi": 700, "window": 255, "sinks": 4},
        # Continuous batching: prompt chunks of very different lengths over cached prefixes.
        {"name": "window_chunk_8", "kind": "window_chunk", "dtype": "fp16", **_heads(NARROW), "block": 16, "seqs": 8, "new_lo": 65,
         "new_hi": 1001, "prior_lo": 0, "prior_hi": 4096, "window": 1000, "sinks": 33},
        # Long prompts in large chunks.
        {"name": "window_chunk_2x4096", "kind": "window_chunk", "dtype": "bf16", **_heads(WIDE), "block": 16, "seqs": 2,
         "new_lo": 4096, "new_hi": 4096, "prior_lo": 2048, "prior_hi": 4096, "window": 4095, "sinks": 4},
        # The step of a batch that only generates: a row of its own for every request, idle or not.
        {"name": "step_blocks_64", "kind": "step_blocks", "block": 16, "requests": 64, "rows": 64, "per_request": 1, "kv_lo": 0,
         "kv_hi": 16000, "columns": 1024, "new_hi": 1, "window": -1, "sinks": 0, "spare": 4096},
        # A step that brings prompt chunks beside single tokens, over a window that lets blocks go.
        {"name": "step_blocks_301", "kind": "step_blocks", "block": 16, "requests": 301, "rows": 8192, "per_request": 0, "kv_lo": 0,
         "kv_hi": 8000, "columns": 640, "new_hi": 96, "window": 4095, "sinks": 4, "spare": 65536},
        # Offline generation: many requests, many rows, wide tables.
        {"name": "step_blocks_2048", "kind": "step_blocks", "block": 16, "requests": 2048, "rows": 131072, "per_request": 0,
         "kv_lo": 0, "kv_hi": 16000, "columns": 1024, "new_hi": 120, "window": 8191, "sinks": 64, "spare": 1 << 20},
        # One sequence, a vocabulary that no tile divides.
        {"name": "penalties_1", "kind": "penalties", "dtype": "fp16", "out": "fp16", "rows": 1, "vocab": 50003, "said_lo": 700,
         "said_hi": 700, "allowed": 0.0, "biased": False},
        # A batch under the controller's allow-masks.
        {"name": "penalties_64", "kind": "penalties", "dtype": "bf16", "out": "bf16", "rows": 64, "vocab": VOCAB, "said_lo": 512,
         "said_hi": 4096, "allowed": 0.05, "biased": False},
        # A large batch of long conversations with the controller's bias rows, for a sampler that takes fp32.
        {"name": "penalties_256", "kind": "penalties", "dtype": "bf16", "out": "fp32", "rows": 256, "vocab": VOCAB, "said_lo": 1,
         "said_hi": 16384, "allowed": 0.0, "biased": True},
    ]


# --------------------------------------------------------------------------- drawn cases

def _between(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm uniform where the range spans more than a factor of ten."""
    if hi > 10 * max(lo, 1):
        x = math.exp(rng.uniform(math.log(max(lo, 0.5)), math.log(hi + 0.5)))
        return min(hi, max(lo, int(x + 0.5)))
    return rng.randint(lo, hi)


def draw(rng):
    kind = rng.choice(["window_decode", "window_chunk", "step_blocks", "penalties"])
    if kind == "window_decode":
        hq, hkv, d = rng.choice(HEADS)
        case = {"kind": kind, "dtype": rng.choice(["bf16", "fp16"]), **_heads((hq, hkv, d)), "block": rng.choice([8, 16, 16, 32]),
                "rows": _between(rng, 1, min(128, 131072 // (hkv * d))), "ctx_lo": _between(rng, 1, 1024), "window": _between(rng, 15, 4095),
                "sinks": rng.choice([0, 1, 4, 17, 64])}
        return {**case, "ctx_hi": _between(rng, case["ctx_lo"], 16384)}
    if kind == "window_chunk":
        seqs = _between(rng, 1, 16)
        hi = min(4096, 8192 // seqs)
        case = {"kind": kind, "dtype": rng.choice(["bf16", "fp16"]), **_heads(rng.choice(HEADS)), "block": rng.choice([8, 16, 16, 32]),
                "seqs": seqs, "new_hi": _between(rng, 2, hi), "prior_lo": 0, "window": _between(rng, 15, 4095),
                "sinks": rng.choice([0, 1, 4, 33, 100])}
        return {**case, "new_lo": rng.randint(1, case["new_hi"]), "prior_hi": _between(rng, 1, 4096)}
    if kind == "step_blocks":
        requests = _between(rng, 1, 2048)
        case = {"kind": kind, "block": rng.choice([8, 16, 16, 32]), "requests": requests, "kv_lo": 0, "columns": 1024,
                "window": rng.choice([-1, _between(rng, 15, 8191)]), "sinks": rng.choice([0, 4, 64])}
        generating = rng.random() < 0.5
        new = 1 if generating else _between(rng, 2, max(2, min(1024, 131072 // requests)))
        return {**case, "kv_hi": _between(rng, 1, case["block"] * 1024 - 1024), "new_hi": new,
                "per_request": 1 if generating else 0,
                "rows": requests if generating else max(1, int(requests * new * rng.uniform(0.3, 0.8))),
                # a pool that has room, or one that runs out
                "spare": rng.choice([1 << 17, _between(rng, 1, 8192)])}
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    return {"kind": kind, "dtype": dtype, "out": rng.choice([dtype, "fp32"]), "rows": _between(rng, 1, 192),
            "vocab": rng.choice([VOCAB, 32000, _between(rng, 1000, VOCAB)]), "said_lo": _between(rng, 1, 512),
            "said_hi": _between(rng, 512, 16384), "allowed": rng.choice([0.0, 0.01, 0.5]), "biased": rng.random() < 0.5}


# --------------------------------------------------------------------------- inputs

def _spread(lo, hi, n):
    """n lengths that cover [lo, hi] evenly."""
    return [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _shuffled(lens, gen):
    return torch.tensor(lens, dtype=torch.int64)[torch.randperm(len(lens), generator=gen)]


def _offsets(lens):
    return torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])


def _ceil(x, m):
    return (x + m - 1) // m


def _normal(shape, dtype, dgen, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device=dgen.device).normal_(0.0, std, generator=dgen).to(dtype)


def _caches(case, blocks, dgen):
    dt, hkv, d, bs = DTYPES[case["dtype"]], case["kv_heads"], case["head_size"], case["block"]
    return _normal((blocks, hkv, d // 8, bs, 8), dt, dgen), _normal((blocks, hkv, d, bs), dt, dgen)


def _tables(held, gen):
    """int32 block tables in which the columns `held` [sequences, columns] have blocks of a shuffled pool of their own, the others block 0;
    and the size of that pool."""
    total = int(held.sum())
    tables = torch.zeros(held.shape, dtype=torch.int32)
    tables[held] = torch.randperm(total, generator=gen).to(torch.int32)
    return tables, total


def _chunk_lens(case):
    """(new tokens, tokens cached before them) of every sequence."""
    n = case["seqs"]
    return _spread(case["new_lo"], case["new_hi"], n), _spread(case["prior_lo"], case["prior_hi"], n)[::-1]


def _new_lens(case):
    """What every request of a step_blocks case brings: most of them tokens, some none, some their end."""
    hi = case["new_hi"]
    return [0 if i % 13 == 5 else (-1 if i % 17 == 9 else 1 + (i * 7919) % hi) for i in range(case["requests"])]


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dgen = torch.Generator(device="cuda" if torch.cuda.is_available() else "cpu").manual_seed(seed + 1)
    return {"window_decode": _prepare_decode, "window_chunk": _prepare_chunk, "step_blocks": _prepare_step,
            "penalties": _prepare_penalties}[case["kind"]](case, gen, dgen)


def _prepare_decode(case, gen, dgen):
    bs, W, dev = case["block"], case["window"], dgen.device
    ctx = _shuffled(_spread(case["ctx_lo"], case["ctx_hi"], case["rows"]), gen)
    col = torch.arange(_ceil(case["ctx_hi"], bs))[None, :]
    # blocks between the sinks and the window have gone back to the pool, as they do in a server that runs with a window
    kept = (col < _ceil(case["sinks"], bs)) | ((col + 1) * bs > (ctx - 1 - W)[:, None])
    tables, blocks = _tables((col < _ceil(ctx, bs)[:, None]) & kept, gen)
    kc, vc = _caches(case, blocks, dgen)
    q = _normal((case["rows"], case["query_heads"], case["head_size"]), DTYPES[case["dtype"]], dgen)
    return {"case": case, "q": q, "kc": kc, "vc": vc, "tables": tables.to(dev), "ctx": ctx.to(torch.int32).to(dev),
            "max_ctx": case["ctx_hi"], "scale": 1.0 / math.sqrt(case["head_size"])}


def _prepare_chunk(case, gen, dgen):
    bs, dev = case["block"], dgen.device
    new, prior = (torch.tensor(x) for x in _chunk_lens(case))
    order = torch.randperm(case["seqs"], generator=gen)
    new, ctx = new[order], (new + prior)[order]
    tables, blocks = _tables(torch.arange(_ceil(int(ctx.max()), bs))[None, :] < _ceil(ctx, bs)[:, None], gen)
    kc, vc = _caches(case, blocks, dgen)
    q = _normal((int(new.sum()), case["query_heads"], case["head_size"]), DTYPES[case["dtype"]], dgen)
    return {"case": case, "q": q, "kc": kc, "vc": vc, "tables": tables.to(dev), "ctx": ctx.to(torch.int32).to(dev),
            "cu": _offsets(new).to(torch.int32).to(dev), "max_q": int(new.max()), "max_k": int(ctx.max()),
            "scale": 1.0 / math.sqrt(case["head_size"])}


def _prepare_step(case, gen, dgen):
    bs, R, cols, W, dev = case["block"], case["requests"], case["columns"], case["window"], dgen.device
    new = torch.tensor(_new_lens(case))[torch.randperm(R, generator=gen)]
    kv = torch.tensor(_spread(case["kv_lo"], case["kv_hi"], R))[torch.randperm(R, generator=gen)]
    # what earlier steps have let go of: blocks behind the window of a step that was as long as this one
    gone = torch.zeros_like(kv) if W < 0 else (kv - case["new_hi"] - W).clamp(min=0) // bs
    col = torch.arange(cols)[None, :]
    held = col < _ceil(kv, bs)[:, None]
    if W >= 0:
        held &= (col < _ceil(case["sinks"], bs)) | (col >= gone[:, None])
    used = int(held.sum())
    nb = used + case["spare"]
    perm = torch.randperm(nb, generator=gen).to(torch.int32)
    tables = torch.zeros((R, cols), dtype=torch.int32)
    tables[held] = perm[:used]
    # the pool's free blocks, first to be handed out first, in a ring that has gone round a few times
    head = 3 * nb + int(torch.randint(nb, (1,), generator=gen))
    ring = torch.zeros(nb, dtype=torch.int32)
    ring[(head + torch.arange(nb - used)) % nb] = perm[used:]
    return {"case": case, "new": new.to(torch.int32).to(dev), "state": torch.stack([kv, gone], 1).to(torch.int32).to(dev),
            "tables": tables.to(dev), "ring": ring.to(dev), "ends": torch.tensor([head, head + nb - used], dtype=torch.int64).to(dev)}


def _prepare_penalties(case, gen, dgen):
    S, V, dev = case["rows"], case["vocab"], dgen.device
    said = _shuffled(_spread(case["said_lo"], case["said_hi"], S), gen)
    # what is said repeats itself: half of it comes from few tokens
    n, few = int(said.sum()), min(V, 512)
    u = torch.rand((n,), device=dev, generator=dgen)
    rare = torch.randint(V, (n,), device=dev, generator=dgen)
    s = {"case": case, "logits": _normal((S, V), DTYPES[case["dtype"]], dgen, 4.0), "offsets": _offsets(said).to(dev),
         "history": torch.where(u < 0.5, rare, rare % few * (V // few)).to(torch.int32),
         "prompt": (said * torch.randint(0, 100, (S,), generator=gen) // 100).to(torch.int32).to(dev), "bias": None, "mask": None,
         "repetition": (1.0 + 0.5 * torch.rand((S,), generator=gen)).to(dev), "frequency": (0.5 * torch.rand((S,), generator=gen)).to(dev),
         "presence": torch.rand((S,), generator=gen).to(dev)}
    if case["allowed"]:
        bits = torch.rand((S, _ceil(V, 32) * 32), device=dev, generator=dgen) < case["allowed"]
        s["mask"] = (bits.view(S, -1, 8) * (2 ** torch.arange(8, device=dev))).sum(-1).to(torch.uint8)
    if case["biased"]:
        # the controller's rows: nothing, a push or a bar
        u = torch.rand((S, V), device=dev, generator=dgen)
        s["bias"] = torch.where(u < 0.9, 0.0, torch.where(u < 0.97, 2.0 * u, -math.inf)).to(torch.float32)
    return s


# --------------------------------------------------------------------------- one pass

def run(s):
    return {"window_decode": _decode, "window_chunk": _chunk, "step_blocks": _step, "penalties": _penalties}[s["case"]["kind"]](s)


def _softmax_product(scores, seen, v):
    """softmax(scores where seen) @ v; zeros where a row sees nothing."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return torch.matmul(e, v) / torch.where(total == 0, torch.ones_like(total), total)


def _cached(s, pos):
    """fp32 keys and values [rows, n, kv heads, head size] at positions pos [rows, n] of the sequences."""
    bs = s["case"]["block"]
    block, at = s["tables"].long().gather(1, pos // bs), pos % bs
    return s["kc"][block, :, :, at, :].flatten(3).float(), s["vc"][block, :, :, at].float()


def _decode(s):
    case = s["case"]
    S, hq, d = s["q"].shape
    hkv, bs, W, sinks = case["kv_heads"], case["block"], case["window"], case["sinks"]
    if own:
        from aici_amd import kernels
        out = torch.empty_like(s["q"])
        kernels.paged_attention_window(out, s["q"], s["kc"], s["vc"], hkv, s["scale"], s["tables"], s["ctx"], bs, s["max_ctx"], W, sinks)
        return out
    ctx = s["ctx"].long()[:, None]
    n = min(W + 1, s["max_ctx"])
    first = torch.arange(min(sinks, s["max_ctx"]), device=ctx.device)[None, :].expand(S, -1)
    last = ctx - n + torch.arange(n, device=ctx.device)[None, :]
    pos = torch.cat([first, last], 1)
    seen = torch.cat([first < ctx - n, last >= 0], 1)
    k, v = _cached(s, torch.where(seen, pos, torch.zeros_like(pos)))
    q = s["q"].float().view(S, hkv, hq // hkv, d)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * s["scale"]
    out = _softmax_product(scores, seen[:, None, None, :], v.permute(0, 2, 1, 3).contiguous())
    return out.reshape(S, hq, d).to(s["q"].dtype)


def _owners(starts, n):
    """For each of n rows, the last of the requests that begin at or before it (starts ascending)."""
    return torch.zeros(n + 1, dtype=torch.int64, device=starts.device).index_add_(0, starts.clamp(max=n), torch.ones_like(starts))[:n].cumsum(0) - 1


def _chunk(s):
    case = s["case"]
    T, hq, d = s["q"].shape
    hkv, W, sinks = case["kv_heads"], case["window"], case["sinks"]
    if own:
        from aici_amd import kernels
        return kernels.flash_attn_varlen_paged_window(s["q"], s["kc"], s["vc"], s["tables"], s["cu"], s["ctx"], s["max_q"], s["max_k"],
                                                      s["scale"], W, sinks)
    cu, ctx = s["cu"].long(), s["ctx"].long()
    b, lq, lk, g = ctx.numel(), s["max_q"], s["max_k"], hq // hkv
    i = torch.arange(lq, device=cu.device)
    q = s["q"].float()[(cu[:-1, None] + i).clamp(max=T - 1)].view(b, lq, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * lq, d)
    j = torch.arange(lk, device=cu.device)
    k, v = _cached(s, torch.minimum(j[None, :], ctx[:, None] - 1))
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(b, hkv, g, lq, lk) * s["scale"]
    at = (ctx - (cu[1:] - cu[:-1]))[:, None, None] + i[:, None]
    seen = (j <= at) & ((j >= at - W) | (j < sinks)) & (j < ctx[:, None, None])
    out = _softmax_product(scores, seen[:, None, None], v.permute(0, 2, 1, 3).unsqueeze(2).expand(b, hkv, g, lk, d))
    row = torch.arange(T, device=cu.device)
    owner = _owners(cu[:-1], T)
    return out.permute(0, 3, 1, 2, 4)[owner, row - cu[owner]].reshape(T, hq, d).to(s["q"].dtype)


def _step(s):
    case = s["case"]
    bs, T, q, W, sinks = case["block"], case["rows"], case["per_request"], case["window"], case["sinks"]
    if own:
        from aici_amd import kernels
        step = kernels.step_blocks(s["new"], s["state"], s["tables"], s["ring"], s["ends"], bs, T, rows_per_request=q, window_size_left=W,
                                   sink_tokens=sinks)
        return {**step._asdict(), "block_tables": s["tables"], "ring": s["ring"]}
    new, kv, gone = s["new"].long(), s["state"][:, 0].long(), s["state"][:, 1].long()
    R, cols = s["tables"].shape
    nb, dev = s["ring"].numel(), new.device
    head, tail = s["ends"][0], s["ends"][1]
    col = torch.arange(cols, device=dev)[None, :]
    held = _ceil(kv, bs)
    ended = new < 0
    # what goes back to the pool, in the order of requests and columns: behind the sinks and the window, or everything
    sunk = _ceil(sinks, bs) if W >= 0 else 0
    dead = torch.maximum(gone, (kv - W).clamp(min=0) // bs) if W >= 0 else gone
    live = (col < held[:, None]) & ((col < sunk) | (col >= gone[:, None]))
    back = live & (ended[:, None] | ((col >= sunk) & (col < dead[:, None])))
    rank = back.flatten().cumsum(0) - 1
    ring = torch.cat([s["ring"], s["ring"][:1]])
    ring.scatter_(0, torch.where(back.flatten(), (tail + rank) % nb, nb), s["tables"].flatten())
    ring = ring[:nb]
    freed = back.sum()
    # who is served: what fits its own row of the table, as long as rows and blocks last, in the order of requests
    fits = (kv + new <= cols * bs) & ((new <= q) if q else (new <= T))
    want = torch.where((new > 0) & fits, new, 0)
    need = torch.where(want > 0, _ceil(kv + new, bs) - held, 0)
    lasts = need.cumsum(0) <= tail - head + freed
    if not q:
        lasts &= want.cumsum(0) <= T
    given = torch.where(lasts, want, 0)
    served = torch.where((new > 0) & ~fits, -2, torch.where((want > 0) & ~lasts, -1, given))
    take = (col >= held[:, None]) & (col < _ceil(kv + given, bs)[:, None]) & (given > 0)[:, None]
    rank = take.flatten().cumsum(0) - 1
    tables = torch.where(take.flatten(), ring[(head + rank) % nb], s["tables"].flatten()).view(R, cols)
    s["tables"].copy_(tables)
    length = torch.where(ended, 0, kv + given)
    state = torch.stack([length, torch.where(ended, 0, dead)], 1)
    context = torch.where(given > 0, length, 0)
    # the rows: one request behind the other, or `q` for each
    cu = torch.cat([given.new_zeros(1), given.cumsum(0)])
    row = torch.arange(T, device=dev)
    if q:
        begin = q * torch.arange(R, device=dev)
        owner = (row // q).clamp(max=R - 1)
    else:
        begin = cu[:-1]
        owner = _owners(begin, T)
    at = row - begin[owner]
    used = at < given[owner]
    pos = torch.where(used, kv[owner] + at, 0)
    slot = torch.where(used, tables[owner, (pos // bs).clamp(max=cols - 1)].long() * bs + pos % bs, -1)
    last = torch.where(given > 0, begin + given - 1, 0)
    ends = torch.stack([head + take.sum(), tail + freed])
    totals = torch.stack([given.sum(), (served < 0).sum(), ends[1] - ends[0], take.sum()])
    i32 = torch.int32
    s["ring"].copy_(ring)
    return {"state": state.to(i32), "ends": ends, "served": served.to(i32), "context_lens": context.to(i32), "seqlens_q": cu.to(i32),
            "logit_idxs": last.to(i32), "positions": pos, "slot_mapping": slot.to(i32), "totals": totals.to(i32), "block_tables": s["tables"],
            "ring": s["ring"]}


def _penalties(s):
    case = s["case"]
    S, V = s["logits"].shape
    out = DTYPES[case["out"]]
    if own:
        from aici_amd import kernels
        return kernels.penalize_logits(s["logits"], s["history"], s["offsets"], s["prompt"], s["repetition"], s["frequency"], s["presence"],
                                       bias=s["bias"], mask=s["mask"], out_dtype=out)
    n = s["history"].numel()
    owner = _owners(s["offsets"][:-1], n)
    flat = owner * V + s["history"].long()
    answered = torch.arange(n, device=flat.device) - s["offsets"][owner] >= s["prompt"].long()[owner]
    seen = torch.zeros(S * V, dtype=torch.int32, device=flat.device).index_add_(0, flat, torch.ones_like(s["history"])).view(S, V) > 0
    count = torch.zeros(S * V, dtype=torch.int32, device=flat.device).index_add_(0, flat, answered.to(torch.int32)).view(S, V).float()
    x = s["logits"].float()
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        x = x + s["bias"][:, :V]
    if s["mask"] is not None:
        token = torch.arange(V, device=x.device)
        x = torch.where((s["mask"][:, token >> 3] >> (token & 7).to(torch.uint8)) & 1 > 0, x, -math.inf)
    return x.to(out)


# --------------------------------------------------------------------------- work and exact values

def work(case):
    if case["kind"] == "window_decode":
        hq, hkv, d = case["query_heads"], case["kv_heads"], case["head_size"]
        n = [min(c, case["window"] + 1) + min(case["sinks"], max(0, c - case["window"] - 1)) for c in _spread(case["ctx_lo"], case["ctx_hi"], case["rows"])]
        return {"bytes": 4 * hkv * d * sum(n) + 4 * case["rows"] * hq * d + 4 * sum(_ceil(c, case["block"]) for c in n) + 4 * case["rows"],
                "flops": 4 * hq * d * sum(n)}
    if case["kind"] == "window_chunk":
        hq, hkv, d, W, sinks = case["query_heads"], case["kv_heads"], case["head_size"], case["window"], case["sinks"]
        new, prior = _chunk_lens(case)
        keys = pairs = 0
        for n, p in zip(new, prior):
            first = max(0, p - W)
            keys += n + p - first + min(sinks, first)
            pairs += sum(min(i + 1, W + 1) + min(sinks, max(0, i - W)) for i in range(p, p + n))
        return {"bytes": 4 * hkv * d * keys + 4 * hq * d * sum(new) + 4 * _ceil(keys, case["block"]), "flops": 4 * hq * d * pairs}
    if case["kind"] == "step_blocks":
        R, T, bs = case["requests"], case["rows"], case["block"]
        new = _new_lens(case)
        moved = sum(_ceil(n, bs) for n in new if n > 0) + sum(_ceil(case["kv_hi"] // 2, bs) for n in new if n < 0)
        # lengths and states in and out, what is said of each request, every row's position and slot, blocks taken and given back
        return {"bytes": R * (4 + 8 + 8 + 16) + T * 12 + 8 * moved, "flops": 10 * R + 5 * T}
    S, V = case["rows"], case["vocab"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    return {"bytes": S * V * (size[case["dtype"]] + size[case["out"]] + (4 if case["biased"] else 0)) + (S * V // 8 if case["allowed"] else 0)
            + 4 * sum(_spread(case["said_lo"], case["said_hi"], S)) + 28 * S, "flops": 6 * S * V}


def exact(case, seed):
    s = prepare(case, seed)
    return {"window_decode": _exact_attention, "window_chunk": _exact_attention, "step_blocks": _exact_step,
            "penalties": _exact_penalties}[case["kind"]](s)


def _exact_attention(s):
    """Each sequence by itself in 64 bits, over all keys, head by head."""
    case = s["case"]
    hq, hkv, d, bs, W, sinks = (case[k] for k in ("query_heads", "kv_heads", "head_size", "block", "window", "sinks"))
    ctx = s["ctx"].tolist()
    cu = s["cu"].tolist() if "cu" in s else list(range(len(ctx) + 1))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(ctx):
        blocks = s["tables"][b, :(n + bs - 1) // bs].long()
        k = s["kc"][blocks].permute(1, 0, 3, 2, 4).reshape(hkv, -1, d)[:, :n].double()
        v = s["vc"][blocks].permute(1, 0, 3, 2).reshape(hkv, -1, d)[:, :n].double()
        q = s["q"][cu[b]:cu[b + 1]].double()
        rows = torch.arange(n - q.size(0), n, device=q.device)[:, None]
        keys = torch.arange(n, device=q.device)[None, :]
        hidden = (keys > rows) | ((keys < rows - W) & (keys >= sinks))
        for h in range(hq):
            scores = (q[:, h] @ k[h // (hq // hkv)].t().contiguous()) * s["scale"]
            scores[hidden] = -math.inf
            weights = torch.exp(scores - scores.max(1, keepdim=True).values)
            out[cu[b]:cu[b + 1], h] = (weights @ v[h // (hq // hkv)]) / weights.sum(1, keepdim=True)
    return out


def _exact_step(s):
    """Request after request, block after block, as a list of free blocks would go."""
    case = s["case"]
    bs, T, q, W, sinks = (case[k] for k in ("block", "rows", "per_request", "window", "sinks"))
    new, state, tables, ring = s["new"].tolist(), s["state"].tolist(), s["tables"].tolist(), s["ring"].tolist()
    head, tail = s["ends"].tolist()
    nb, cols, R = len(ring), len(tables[0]), len(new)
    sunk = _ceil(sinks, bs) if W >= 0 else 0
    lens, goner = [], []
    for r in range(R):
        kv, gone = state[r]
        dead = max(gone, max(0, kv - W) // bs) if W >= 0 else gone
        for c in range(_ceil(kv, bs)):
            if (c < sunk or c >= gone) and (new[r] < 0 or sunk <= c < dead):
                ring[tail % nb] = tables[r][c]
                tail += 1
        lens.append(0 if new[r] < 0 else kv)
        goner.append(0 if new[r] < 0 else dead)
    avail, asked, rows, taken = tail - head, 0, 0, 0
    served, begin = [], []
    pos, slot = [0] * T, [-1] * T
    for r in range(R):
        n, kv = new[r], state[r][0]
        begin.append(q * r if q else (begin[-1] + max(0, served[-1]) if r else 0))
        if n <= 0:
            served.append(0)
            continue
        if kv + n > cols * bs or n > (q or T):
            served.append(-2)
            continue
        asked += _ceil(kv + n, bs) - _ceil(kv, bs)
        rows += n
        if asked > avail or (not q and rows > T):
            served.append(-1)
            continue
        served.append(n)
        for c in range(_ceil(kv, bs), _ceil(kv + n, bs)):
            tables[r][c] = ring[head % nb]
            head += 1
            taken += 1
        for i in range(n):
            pos[begin[r] + i] = kv + i
            slot[begin[r] + i] = tables[r][(kv + i) // bs] * bs + (kv + i) % bs
        lens[r] = kv + n
    given = [max(0, x) for x in served]
    dev, i32 = s["new"].device, torch.int32
    cu = [0]
    for x in given:
        cu.append(cu[-1] + x)

    def t(x, dt=i32):
        return torch.tensor(x, dtype=dt, device=dev)

    return {"state": t([list(x) for x in zip(lens, goner)]), "ends": t([head, tail], torch.int64), "served": t(served),
            "context_lens": t([l if x else 0 for l, x in zip(lens, given)]), "seqlens_q": t(cu),
            "logit_idxs": t([b + x - 1 if x else 0 for b, x in zip(begin, given)]), "positions": t(pos, torch.int64), "slot_mapping": t(slot),
            "totals": t([sum(given), sum(x < 0 for x in served), tail - head, taken]), "block_tables": t(tables), "ring": t(ring)}


def _exact_penalties(s):
    """Row after row in 64 bits."""
    V = s["logits"].size(1)
    offsets, prompt = s["offsets"].tolist(), s["prompt"].tolist()
    out = s["logits"].double()
    for r in range(out.size(0)):
        said = s["history"][offsets[r]:offsets[r + 1]].long()
        times = torch.bincount(said[prompt[r]:], minlength=V).double()
        ever = torch.bincount(said, minlength=V) > 0
        rep = s["repetition"][r].double()
        x = out[r]
        x[ever] = torch.where(x[ever] > 0, x[ever] / rep, x[ever] * rep)
        x -= s["frequency"][r].double() * times
        x[times > 0] -= s["presence"][r].double()
        if s["bias"] is not None:
            x += s["bias"][r, :V].double()
        if s["mask"] is not None:
            bits = (s["mask"][r][:, None].long() >> torch.arange(8, device=x.device)) & 1
            x[bits.flatten()[:V] == 0] = -math.inf
    return out
