"""The operators of a generation step that verifies trees of drafted tokens on weights of 8 bits, as cases that can be timed and compared.

Kinds of case:

  tree_attention  the rows of drafted trees against their sequences' paged contexts: a row sees the context in front of the tree and the
                  rows of the tree that its mask names (`kernels.paged_attention_tree`).
  linear_fp8      x @ weight.T with the weight in e4m3 and a scale for each 128 x 128 of it, the rows of x rounded to e4m3 with a scale
                  for each 128 columns (`kernels.linear_fp8`).
  tree_rows       positions and masks of a step's trees from the parents of their rows (`kernels.tree_rows`).
  tree_accept     the drafted tokens that the model's choices confirm, and their keys and values moved to where the next step looks for
                  them, in every layer's cache (`kernels.tree_accept`).

`own` picks the framework's calls; otherwise the same is computed in its plain form.  Lengths and the shape of the trees come from the
case alone; the seed of `prepare` gives the order, the values and the order of the blocks in the pool.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
WIDE, ODD, NARROW, PHI2 = (32, 8, 128), (12, 4, 112), (16, 2, 64), (32, 32, 80)
HEADS = (WIDE, ODD, NARROW, PHI2)
# (rows, columns) of weights: 32 / 8 heads of 128 over 4096 with 14336 in between, 32 heads of 80 over 2560, 12 / 4 heads of 112 over 1344
WEIGHTS = ((6144, 4096), (4096, 4096), (28672, 4096), (4096, 14336), (7680, 2560), (2560, 10240), (2240, 1344), (1344, 1344))
VOCAB = 128256
MOST_KEYS = 64 * 8192 * 8 * 128  # of a drawn tree_attention case, x kv heads x head size
MOST_SCORES = 64 * 32 * 32 * 16384
MOST_PRODUCTS = 4096 * 28672 * 4096


def _heads(shape):
    return {"query_heads": shape[0], "kv_heads": shape[1], "head_size": shape[2]}


def listed():
    return [
        # A single chat and a tree of its next few tokens: where latency counts.
        {"name": "tree_attention_1", "kind": "tree_attention", "dtype": "bf16", **_heads(WIDE), "block": 16, "seqs": 1, "nodes_lo": 24,
         "nodes_hi": 24, "prior_lo": 1500, "prior_hi": 1500},
        # A small batch of narrower heads, some trees of one row, some contexts that are only a tree.
        {"name": "tree_attention_12", "kind": "tree_attention", "dtype": "fp16", **_heads(ODD), "block": 16, "seqs": 12, "nodes_lo": 1,
         "nodes_hi": 45, "prior_lo": 0, "prior_hi": 4011},
        # Every head with keys of its own, large trees.
        {"name": "tree_attention_8", "kind": "tree_attention", "dtype": "fp16", **_heads(PHI2), "block": 16, "seqs": 8, "nodes_lo": 64,
         "nodes_hi": 64, "prior_lo": 500, "prior_hi": 8000},
        # A full server: long conversations.
        {"name": "tree_attention_64", "kind": "tree_attention", "dtype": "bf16", **_heads(WIDE), "block": 16, "seqs": 64, "nodes_lo": 16,
         "nodes_hi": 32, "prior_lo": 1024, "prior_hi": 15000},
        # The projection of q, k and v of a single token.
        {"name": "linear_fp8_1", "kind": "linear_fp8", "dtype": "bf16", "rows": 1, "out": 6144, "in": 4096, "residual": False},
        # A step of a few trees through the widest projection.
        {"name": "linear_fp8_37", "kind": "linear_fp8", "dtype": "bf16", "rows": 37, "out": 28672, "in": 4096, "residual": False},
        # A batch of trees through the projection that closes a layer.
        {"name": "linear_fp8_301", "kind": "linear_fp8", "dtype": "fp16", "rows": 301, "out": 4096, "in": 14336, "residual": True},
        # A long prompt.
        {"name": "linear_fp8_4096", "kind": "linear_fp8", "dtype": "bf16", "rows": 4096, "out": 28672, "in": 4096, "residual": False},
        # One tree; the step of a full server, with large trees.
        {"name": "tree_rows_1", "kind": "tree_rows", "seqs": 1, "nodes_lo": 24, "nodes_hi": 24, "prior_lo": 1024, "prior_hi": 2048},
        {"name": "tree_rows_256", "kind": "tree_rows", "seqs": 256, "nodes_lo": 1, "nodes_hi": 200, "prior_lo": 0, "prior_hi": 16000},
        # One tree over few layers; a full server's over all.
        {"name": "tree_accept_1", "kind": "tree_accept", "dtype": "bf16", **_heads(WIDE), "block": 16, "layers": 8, "seqs": 1,
         "nodes_lo": 24, "nodes_hi": 24},
        {"name": "tree_accept_64", "kind": "tree_accept", "dtype": "bf16", **_heads(WIDE), "block": 16, "layers": 32, "seqs": 64,
         "nodes_lo": 16, "nodes_hi": 61},
    ]


# --------------------------------------------------------------------------- drawn cases

def _between(rng, lo, hi):
    """A whole number in [lo, hi], its logarithm uniform where the range spans more than a factor of ten."""
    if hi > 10 * max(lo, 1):
        x = math.exp(rng.uniform(math.log(max(lo, 0.5)), math.log(hi + 0.5)))
        return min(hi, max(lo, int(x + 0.5)))
    return rng.randint(lo, hi)


def draw(rng):
    kind = rng.choice(["tree_attention", "tree_attention", "linear_fp8", "linear_fp8", "tree_rows", "tree_accept"])
    if kind == "tree_attention":
        hq, hkv, d = rng.choice(HEADS)
        nodes = _between(rng, 1, 130)
        prior = _between(rng, 1, 15000)
        seqs = _between(rng, 1, max(1, min(64, MOST_KEYS // (hkv * d * (prior + nodes)), MOST_SCORES // (hq * nodes * (prior + nodes)))))
        return {"kind": kind, "dtype": rng.choice(["bf16", "fp16"]), **_heads((hq, hkv, d)), "block": rng.choice([8, 16, 16, 32]), "seqs": seqs,
                "nodes_lo": rng.randint(1, nodes), "nodes_hi": nodes, "prior_lo": _between(rng, 0, prior), "prior_hi": prior}
    if kind == "linear_fp8":
        n, k = rng.choice(WEIGHTS + ((16 * _between(rng, 1, 1792), 16 * _between(rng, 1, 896)),) * 4)
        return {"kind": kind, "dtype": rng.choice(["bf16", "fp16"]), "rows": _between(rng, 1, min(4096, MOST_PRODUCTS // (n * k))), "out": n,
                "in": k, "residual": rng.random() < 0.3}
    if kind == "tree_rows":
        nodes = _between(rng, 1, 300)
        return {"kind": kind, "seqs": _between(rng, 1, 256), "nodes_lo": rng.randint(1, nodes), "nodes_hi": nodes, "prior_lo": 0,
                "prior_hi": _between(rng, 1, 16000)}
    hq, hkv, d = rng.choice(HEADS)
    layers, nodes = _between(rng, 1, 32), _between(rng, 1, 130)
    most = 32 * 64 * 64 * 8 * 128 // (layers * nodes * hkv * d)
    return {"kind": kind, "dtype": rng.choice(["bf16", "fp16"]), **_heads((hq, hkv, d)), "block": rng.choice([8, 16, 16, 32]), "layers": layers,
            "seqs": _between(rng, 1, max(1, min(128, most))), "nodes_lo": rng.randint(1, nodes), "nodes_hi": nodes}


# --------------------------------------------------------------------------- inputs

def _spread(lo, hi, n):
    """n lengths that cover [lo, hi] evenly."""
    return [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _offsets(lens):
    return torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])


def _ceil(x, m):
    return (x + m - 1) // m


def _normal(shape, dtype, dgen, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device=dgen.device).normal_(0.0, std, generator=dgen).to(dtype)


def _tree(n):
    """The parents of a tree of n rows, row 0 its root: the later of the rows in front more often, so that some paths are long."""
    rng = random.Random(n)
    return [-1] + [int(i * math.sqrt(rng.random())) for i in range(1, n)]


def _path(n):
    """The rows of that tree from its root down to the row that is deepest (the first of them)."""
    parents = _tree(n)
    depth = [0] * n
    for i in range(1, n):
        depth[i] = depth[parents[i]] + 1
    at, path = depth.index(max(depth)), []
    while at >= 0:
        path.append(at)
        at = parents[at]
    return path[::-1]


def _confirmed(n, i):
    """The rows of the i-th sequence's tree that the model's choices confirm: some of the way to its deepest row."""
    path = _path(n)
    return path[:1 + (len(path) * (1 + i % 4)) // 4]


def _nodes(case):
    return _spread(case["nodes_lo"], case["nodes_hi"], case["seqs"])


def _priors(case):
    return _spread(case["prior_lo"], case["prior_hi"], case["seqs"])[::-1]


def _tables(lens, bs, gen):
    """int32 block tables of sequences of that many tokens over a shuffled pool, and its size."""
    held = torch.arange(max(1, _ceil(int(lens.max()), bs)))[None, :] < _ceil(lens, bs)[:, None]
    total = int(held.sum())
    tables = torch.zeros(held.shape, dtype=torch.int32)
    tables[held] = torch.randperm(total, generator=gen).to(torch.int32)
    return tables, max(1, total)


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dgen = torch.Generator(device="cuda" if torch.cuda.is_available() else "cpu").manual_seed(seed + 1)
    return {"tree_attention": _prepare_attention, "linear_fp8": _prepare_linear, "tree_rows": _prepare_rows,
            "tree_accept": _prepare_accept}[case["kind"]](case, gen, dgen)


def _prepare_rows(case, gen, dgen):
    dev = dgen.device
    nodes = torch.tensor(_nodes(case))[torch.randperm(case["seqs"], generator=gen)]
    priors = torch.randint(case["prior_lo"], case["prior_hi"] + 1, nodes.shape, generator=gen)
    cu = _offsets(nodes)
    # a drafter that goes on from what it trusts: the later rows in front are parents more often
    at = torch.arange(int(cu[-1])) - cu[:-1].repeat_interleave(nodes)
    parents = torch.where(at == 0, -1, (at * torch.rand(at.shape, generator=gen).sqrt()).long())
    return {"case": case, "parents": parents.to(torch.int32).to(dev), "cu": cu.to(torch.int32).to(dev), "ctx": (nodes + priors).to(torch.int32).to(dev),
            "max_q": int(nodes.max())}


def _prepare_attention(case, gen, dgen):
    dt, hkv, d, bs, dev = DTYPES[case["dtype"]], case["kv_heads"], case["head_size"], case["block"], dgen.device
    order = torch.randperm(case["seqs"], generator=gen)
    nodes, priors = torch.tensor(_nodes(case))[order], torch.tensor(_priors(case))[order]
    s = {"case": case, "parents": torch.tensor([x for n in nodes.tolist() for x in _tree(n)], dtype=torch.int32).to(dev),
         "cu": _offsets(nodes).to(torch.int32).to(dev), "ctx": (nodes + priors).to(torch.int32).to(dev), "max_q": int(nodes.max())}
    s["mask"] = _packed(_ancestors(s["parents"].long(), s["cu"].long(), s["max_q"])[0])
    tables, blocks = _tables(s["ctx"].cpu().long(), bs, gen)
    return {**s, "tables": tables.to(dev), "kc": _normal((blocks, hkv, d // 8, bs, 8), dt, dgen), "vc": _normal((blocks, hkv, d, bs), dt, dgen),
            "q": _normal((sum(_nodes(case)), case["query_heads"], d), dt, dgen), "max_k": int(s["ctx"].max()), "scale": 1.0 / math.sqrt(d)}


def _prepare_linear(case, gen, dgen):
    dt, m, n, k = DTYPES[case["dtype"]], case["rows"], case["out"], case["in"]
    nb, kb = _ceil(n, 128), _ceil(k, 128)
    w = torch.zeros((nb * 128, kb * 128), device=dgen.device)
    w[:n, :k] = _normal((n, k), torch.float32, dgen, 0.02)
    w = w.view(nb, 128, kb, 128)
    scale = w.abs().amax((1, 3)) / 448.0  # the blocks' largest values have the largest number of 8 bits
    w = (w / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(nb * 128, kb * 128)[:n, :k].contiguous()
    # activations behind a norm: a few columns are much larger than the others
    loud = torch.where(torch.rand((k,), device=dgen.device, generator=dgen) < 0.01, 20.0, 1.0)
    x = (_normal((m, k), torch.float32, dgen) * loud).to(dt)
    return {"case": case, "x": x, "w": w, "scale": scale, "residual": _normal((m, n), dt, dgen) if case["residual"] else None}


def _prepare_accept(case, gen, dgen):
    dt, hkv, d, bs, dev = DTYPES[case["dtype"]], case["kv_heads"], case["head_size"], case["block"], dgen.device
    order = torch.randperm(case["seqs"], generator=gen).tolist()
    nodes = [_nodes(case)[i] for i in order]
    # the trees begin anywhere in a block
    first = torch.randint(bs, (case["seqs"],), generator=gen)
    columns = _ceil(max(nodes) + bs - 1, bs)
    blocks = case["seqs"] * columns
    tables = torch.randperm(blocks, generator=gen).view(-1, columns)
    tokens, parents, chosen, slots = [], [], [], []
    for r, (i, n) in enumerate(zip(order, nodes)):
        # siblings' tokens differ; what the model has chosen is a child's token on the confirmed way and no child's behind it
        said = torch.randperm(VOCAB, generator=gen)[:2 * n].tolist()
        want = said[n:]
        path = _confirmed(n, i)
        for a, b in zip(path, path[1:]):
            want[a] = said[b]
        at = int(first[r]) + torch.arange(n)
        tokens += said[:n]
        chosen += want
        parents += _tree(n)
        slots += (tables[r][at // bs] * bs + at % bs).tolist()
    i32 = {k: torch.tensor(v, dtype=torch.int32).to(dev) for k, v in (("tokens", tokens), ("parents", parents), ("chosen", chosen), ("slots", slots))}
    kcs, vcs = _normal((case["layers"], blocks, hkv, d // 8, bs, 8), dt, dgen), _normal((case["layers"], blocks, hkv, d, bs), dt, dgen)
    s = {"case": case, **i32, "cu": _offsets(torch.tensor(nodes)).to(torch.int32).to(dev), "max_q": max(nodes), "kcs": kcs, "vcs": vcs}
    if own:
        from aici_amd import kernels
        s["caches"] = kernels.CacheList(list(kcs), list(vcs))
    return s


# --------------------------------------------------------------------------- one pass

def run(s):
    return {"tree_attention": _attention, "linear_fp8": _linear, "tree_rows": _rows, "tree_accept": _accept}[s["case"]["kind"]](s)


def _owners(starts, n):
    """For each of n rows, the last of the sequences that begin at or before it (starts ascending)."""
    return torch.zeros(n + 1, dtype=torch.int64, device=starts.device).index_add_(0, starts.clamp(max=n), torch.ones_like(starts))[:n].cumsum(0) - 1


def _ancestors(parents, cu, most):
    """Which rows of its tree a row sees, itself and its ancestors, bool [rows, most]; and how many ancestors it has."""
    T = parents.numel()
    start = cu[_owners(cu[:-1], T)]
    at = torch.arange(T, device=parents.device) - start
    seen = torch.zeros((T, most), dtype=torch.bool, device=parents.device)
    depth = torch.full((T,), -1, dtype=torch.int64, device=parents.device)
    while bool((at >= 0).any()):
        up = at >= 0
        depth += up
        seen |= (torch.arange(most, device=parents.device)[None, :] == at[:, None]) & up[:, None]
        at = torch.where(up, parents[start + at.clamp(min=0)], at)
    return seen, depth


def _packed(seen):
    """Bits of 64-bit words, bit j of word i for column 64 i + j."""
    T, n = seen.shape
    words = torch.zeros((T, _ceil(n, 64) * 64), dtype=torch.int64, device=seen.device)
    words[:, :n] = seen
    return (words.view(T, -1, 64) << torch.arange(64, device=seen.device)).sum(-1)


def _rows(s):
    if own:
        from aici_amd import kernels
        positions, mask = kernels.tree_rows(s["parents"], s["cu"], s["ctx"], s["max_q"])
        return {"positions": positions, "mask": mask}
    cu = s["cu"].long()
    seen, depth = _ancestors(s["parents"].long(), cu, s["max_q"])
    first = s["ctx"].long() - (cu[1:] - cu[:-1])
    return {"positions": first[_owners(cu[:-1], depth.numel())] + depth, "mask": _packed(seen)}


def _attention(s):
    case = s["case"]
    T, hq, d = s["q"].shape
    hkv, bs = case["kv_heads"], case["block"]
    if own:
        from aici_amd import kernels
        return kernels.paged_attention_tree(s["q"], s["kc"], s["vc"], s["tables"], s["cu"], s["ctx"], s["max_q"], s["max_k"], s["scale"], s["mask"])
    cu, ctx = s["cu"].long(), s["ctx"].long()
    b, lq, lk, g = ctx.numel(), s["max_q"], s["max_k"], hq // hkv
    i, j = torch.arange(lq, device=cu.device), torch.arange(lk, device=cu.device)
    row = (cu[:-1, None] + i).clamp(max=T - 1)
    q = s["q"].float()[row].view(b, lq, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * lq, d)
    pos = torch.minimum(j[None, :], ctx[:, None] - 1)
    block = s["tables"].long().gather(1, pos // bs)
    k = s["kc"][block, :, :, pos % bs, :].flatten(3).float()
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(b, hkv, g, lq, lk) * s["scale"]
    del k
    node = j[None, :] - (ctx - (cu[1:] - cu[:-1]))[:, None]  # [b, lk]: the row of the tree that a key belongs to
    at = node.clamp(min=0, max=lq - 1)
    bit = (s["mask"][row].gather(2, (at >> 6)[:, None, :].expand(b, lq, lk)) >> (at & 63)[:, None, :]) & 1
    seen = ((node < 0)[:, None, :] | (bit > 0)) & (j[None, :] < ctx[:, None])[:, None, :]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    del scores
    total = e.sum(-1, keepdim=True)
    v = s["vc"][block, :, :, pos % bs].float().permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(e.view(b, hkv, g * lq, lk), v).view(b, hkv, g, lq, d) / torch.where(total == 0, torch.ones_like(total), total)
    row = torch.arange(T, device=cu.device)
    owner = _owners(cu[:-1], T)
    return out.permute(0, 3, 1, 2, 4)[owner, row - cu[owner]].reshape(T, hq, d).to(s["q"].dtype)


def _linear(s):
    if own:
        from aici_amd import kernels
        return kernels.linear_fp8(s["x"], s["w"], s["scale"], residual=s["residual"])
    x, w = s["x"], s["w"]
    (m, k), n, kb = x.shape, w.size(0), s["scale"].size(1)
    blocks = torch.zeros((m, kb * 128), device=x.device)
    blocks[:, :k] = x
    blocks = blocks.view(m, kb, 128)
    part, power = torch.frexp(blocks.abs().amax(-1))
    power = (power - 9 + (part > 0.875)).clamp(min=-126)[..., None]  # the least with max <= 448 * 2 ** power
    # (powers of two by their bits: 2 ** power need not be exact on the device, and half of what is between two numbers of 8 bits hangs on it)
    up, down = ((127 - power) << 23).view(torch.float32), ((127 + power) << 23).view(torch.float32)
    rounded = (blocks * up).to(torch.float8_e4m3fn).float() * down
    weight = w.float() * s["scale"].repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    y = torch.matmul(rounded.view(m, kb * 128)[:, :k], weight.t()).to(x.dtype)
    return y if s["residual"] is None else (y.float() + s["residual"].float()).to(x.dtype)


def _accept(s):
    if own:
        from aici_amd import kernels
        lens, path, following = kernels.tree_accept(s["tokens"], s["parents"], s["chosen"], s["cu"], s["max_q"], s["slots"], s["caches"])
        return {"lens": lens, "path": path, "next": following, "kcs": s["kcs"], "vcs": s["vcs"]}
    cu, bs = s["cu"].long(), s["case"]["block"]
    R, T, most = cu.numel() - 1, s["tokens"].numel(), s["max_q"]
    dev = cu.device
    begin, n = cu[:-1], cu[1:] - cu[:-1]
    i = torch.arange(most, device=dev)
    row = (begin[:, None] + i).clamp(max=T - 1)
    inside = i[None, :] < n[:, None]
    parents, tokens = s["parents"].long()[row], s["tokens"][row]
    path = torch.full((R, most), -1, dtype=torch.int64, device=dev)
    at = torch.where(n > 0, 0, -1)
    last = at
    for k in range(most):
        path[:, k] = at
        last = torch.where(at >= 0, at, last)
        fits = inside & (parents == at[:, None]) & (tokens == s["chosen"][(begin + at.clamp(min=0)).clamp(max=T - 1)][:, None]) & (at >= 0)[:, None]
        at = torch.where(fits.any(1), fits.to(torch.int32).argmax(1), -1)
    lens = (path >= 0).sum(1)
    following = torch.where(n > 0, s["chosen"][(begin + last.clamp(min=0)).clamp(max=T - 1)], -1)
    moved = (path >= 0) & (path != i[None, :])
    src = s["slots"].long()[(begin[:, None] + path.clamp(min=0)).clamp(max=T - 1)][moved]
    dst = s["slots"].long()[row][moved]
    for kc, vc in zip(s["kcs"], s["vcs"]):
        kc[dst // bs, :, :, dst % bs, :] = kc[src // bs, :, :, src % bs, :]
        vc[dst // bs, :, :, dst % bs] = vc[src // bs, :, :, src % bs]
    i32 = torch.int32
    return {"lens": lens.to(i32), "path": path.to(i32), "next": following.to(i32), "kcs": s["kcs"], "vcs": s["vcs"]}


# --------------------------------------------------------------------------- work and exact values

def work(case):
    if case["kind"] == "linear_fp8":
        m, n, k = case["rows"], case["out"], case["in"]
        return {"bytes": n * k + 4 * _ceil(n, 128) * _ceil(k, 128) + 2 * m * k + 2 * m * n * (2 if case["residual"] else 1), "flops": 2 * m * n * k}
    nodes = _nodes(case)
    words = _ceil(max(nodes), 64)
    if case["kind"] == "tree_rows":
        return {"bytes": sum(nodes) * (4 + 8 + 8 * words) + 8 * case["seqs"], "flops": 0}
    hq, hkv, d = case["query_heads"], case["kv_heads"], case["head_size"]
    if case["kind"] == "tree_accept":
        moved = sum(sum(a != b for a, b in enumerate(_confirmed(n, i))) for i, n in enumerate(nodes))
        return {"bytes": 8 * hkv * d * case["layers"] * moved + 16 * sum(nodes) + 4 * case["seqs"] * (3 + max(nodes)), "flops": 0}
    seen = {}
    for n in set(nodes):
        parents, depth = _tree(n), [1] * n
        for i in range(1, n):
            depth[i] = depth[parents[i]] + 1
        seen[n] = sum(depth)
    priors = _priors(case)
    keys = sum(nodes) + sum(priors)
    pairs = sum(n * p + seen[n] for n, p in zip(nodes, priors))
    return {"bytes": 4 * hkv * d * keys + 4 * hq * d * sum(nodes) + 8 * words * sum(nodes) + 4 * sum(_ceil(n + p, case["block"]) for n, p in zip(nodes, priors)),
            "flops": 4 * hq * d * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree_attention": _exact_attention, "linear_fp8": _exact_linear, "tree_rows": _exact_rows, "tree_accept": _exact_accept}[case["kind"]](s)


def _trees(s):
    """(first row, rows, parents as a list) of every sequence."""
    cu, parents = s["cu"].tolist(), s["parents"].tolist()
    return [(a, b - a, parents[a:b]) for a, b in zip(cu, cu[1:])]


def _family(parents, i):
    """Row i and its ancestors."""
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out


def _exact_rows(s):
    positions, mask, words = [], [], _ceil(s["max_q"], 64)
    for (a, n, parents), ctx in zip(_trees(s), s["ctx"].tolist()):
        for i in range(n):
            family = _family(parents, i)
            positions.append(ctx - n + len(family) - 1)
            bits = sum(1 << j for j in family)
            part = [(bits >> (64 * w)) & (2 ** 64 - 1) for w in range(words)]
            mask.append([p - 2 ** 64 if p >= 2 ** 63 else p for p in part])
    dev = s["cu"].device
    return {"positions": torch.tensor(positions, device=dev), "mask": torch.tensor(mask, dtype=torch.int64, device=dev)}


def _exact_attention(s):
    """Each sequence by itself in 64 bits, head by head."""
    case = s["case"]
    hq, hkv, d, bs = (case[k] for k in ("query_heads", "kv_heads", "head_size", "block"))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for r, ((a, n, parents), ctx) in enumerate(zip(_trees(s), s["ctx"].tolist())):
        blocks = s["tables"][r, :(ctx + bs - 1) // bs].long()
        k = s["kc"][blocks].permute(1, 0, 3, 2, 4).reshape(hkv, -1, d)[:, :ctx].double()
        v = s["vc"][blocks].permute(1, 0, 3, 2).reshape(hkv, -1, d)[:, :ctx].double()
        q = s["q"][a:a + n].double()
        hidden = torch.ones((n, ctx), dtype=torch.bool)
        hidden[:, :ctx - n] = False
        for i in range(n):
            hidden[i, [ctx - n + f for f in _family(parents, i)]] = False
        hidden = hidden.to(q.device)
        for h in range(hq):
            scores = (q[:, h] @ k[h // (hq // hkv)].t().contiguous()) * s["scale"]
            scores[hidden] = -math.inf
            weights = torch.exp(scores - scores.max(1, keepdim=True).values)
            out[a:a + n, h] = (weights @ v[h // (hq // hkv)]) / weights.sum(1, keepdim=True)
    return out


def _exact_linear(s):
    """The nearest of the numbers of 8 bits found among all of them, the products in 64 bits."""
    x, w = s["x"].double(), s["w"].double()
    dev, (n, k) = x.device, w.shape
    table = torch.tensor([(m / 8 if e == 0 else 1 + m / 8) * 2.0 ** (max(e, 1) - 7) for e in range(16) for m in range(8)][:127], dtype=torch.float64,
                         device=dev)
    middle = (table[1:] + table[:-1]) / 2
    y = torch.zeros((x.size(0), n), dtype=torch.float64, device=dev)
    for b in range(s["scale"].size(1)):
        part = x[:, 128 * b:128 * b + 128]
        most = part.abs().amax(1, keepdim=True)
        # the least power of two that holds the largest: from one that may be below it, and the exponent of a double
        unit = ((torch.floor(torch.log2(most.clamp(min=2.0 ** -110))).long() - 10 + 1023) << 52).view(torch.float64)
        for _ in range(3):
            unit = torch.where(most > 448.0 * unit, 2 * unit, unit)
        v = part / unit
        low, high = torch.bucketize(v.abs(), middle), torch.bucketize(v.abs(), middle, right=True)
        code = torch.where(low % 2 == 0, low, high)  # between two of them: the even one
        rows = s["scale"][:, b].double().repeat_interleave(128)[:n, None]
        y += (torch.sign(v) * table[code] * unit) @ (w[:, 128 * b:128 * b + 128] * rows).t().contiguous()
    if s["residual"] is not None:
        y = y.to(s["x"].dtype).double() + s["residual"].double()
    return y


def _exact_accept(s):
    """Sequence after sequence, row after row."""
    tokens, chosen, slots, bs = s["tokens"].tolist(), s["chosen"].tolist(), s["slots"].tolist(), s["case"]["block"]
    lens, paths, following = [], [], []
    src, dst = [], []
    for a, n, parents in _trees(s):
        path = [0] if n else []
        while path:
            child = [c for c in range(n) if parents[c] == path[-1] and tokens[a + c] == chosen[a + path[-1]]]
            if not child:
                break
            path.append(child[0])
        lens.append(len(path))
        paths.append(path + [-1] * (s["max_q"] - len(path)))
        following.append(chosen[a + path[-1]] if path else -1)
        src += [slots[a + p] for p in path]
        dst += [slots[a + i] for i in range(len(path))]
    dev = s["cu"].device
    src, dst = torch.tensor(src, device=dev), torch.tensor(dst, device=dev)
    k, v = s["kcs"].transpose(3, 4).flatten(4), s["vcs"].transpose(3, 4)  # [layers, blocks, heads, tokens, head size]
    out = []
    for t in (k, v):
        t = t.clone()
        t[:, dst // bs, :, dst % bs] = t[:, src // bs, :, src % bs].clone()
        out.append(t)
    i32 = torch.int32
    return {"lens": torch.tensor(lens, dtype=i32, device=dev), "path": torch.tensor(paths, dtype=i32, device=dev),
            "next": torch.tensor(following, dtype=i32, device=dev), "kcs": out[0].unflatten(4, (-1, 8)).transpose(3, 4), "vcs": out[1].transpose(3, 4)}
