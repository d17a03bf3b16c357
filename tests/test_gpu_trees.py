"""Trees of drafted tokens: kernels.tree_rows, kernels.tree_accept and kernels.paged_attention_tree against the 64-bit restatement in
oracle/trees.py, and their refusals.

Tolerance of the attention: the probabilities are rounded to the cache's type (half a step, u = eps / 2, of each: u times the outputs with the
values' magnitudes, A) and so is the output (u of it); a score of d products summed in fp32 is off by at most d 2^-23 of the sum S of their
magnitudes, which moves a probability and the normaliser by that much each, as do exp2 and the additions of up to 2^14 of them in runs of at
most 2^9 (2^-14 together): u (A + |out|) (1 + 2^-6) + 2 (d 2^-23 S + 2^-14) A."""
import math
import random

import pytest
import torch

from aici_amd import kernels as K
from aici_amd._lib import HipAttnError
from oracle import trees

from common import make_cache

gpu = pytest.mark.gpu


def tree(n, seed):
    """Parents of a random tree (now and then a second root, or a row that names one behind it)."""
    rng = random.Random(seed)
    out = [-1] + [int(i * math.sqrt(rng.random())) for i in range(1, n)]
    if n > 6 and seed % 3 == 0:
        out[n // 2], out[n - 2] = -1, n + 5
    return out[:n]


class Case:
    """Sequences of `nodes` rows behind `priors` keys over a shuffled pool whose other blocks hold NaN."""

    def __init__(self, seed, nodes, priors, heads, bs, dtype, device, masks=None, behind=0):
        g = torch.Generator().manual_seed(seed)
        self.hq, self.hkv, self.d = heads
        self.nodes, self.ctx, self.bs, self.dtype = nodes, [n + p for n, p in zip(nodes, priors)], bs, dtype
        cols = [(c + bs - 1) // bs for c in self.ctx]
        pool = sum(cols) + 3
        perm = torch.randperm(pool, generator=g).tolist()
        self.kc, self.vc = make_cache(pool, self.hkv, self.d, bs, dtype, fill=float("nan"))
        width = max(cols + [1]) + 1
        self.tables = torch.full((len(nodes), width), 1 << 30, dtype=torch.int32)
        self.keys, self.values = [], []
        for s, c in enumerate(self.ctx):
            blocks = [perm.pop() for _ in range(cols[s])]
            self.tables[s, :cols[s]] = torch.tensor(blocks, dtype=torch.int32)
            k, v = (torch.randn((c, self.hkv, self.d), generator=g).to(dtype) for _ in range(2))
            self.keys.append(k)
            self.values.append(v)
        self.cu = [0]
        for n in nodes:
            self.cu.append(self.cu[-1] + n)
        self.T = self.cu[-1] + behind
        self.most, self.max_k = max(nodes + [0]), max(self.ctx + [0])
        self.parents = [x for i, n in enumerate(nodes) for x in tree(n, seed + i)]
        _, self.seen = trees.rows(self.parents, self.cu, self.ctx, self.most)
        if masks is not None:
            self.seen = masks(self.seen, g)
        self.q = torch.randn((self.T, self.hq, self.d), generator=g).to(dtype)
        self.device = device
        self.fill()

    def fill(self):
        """The keys and values into the cache."""
        for s, c in enumerate(self.ctx):
            for t in range(c):
                b, o = int(self.tables[s, t // self.bs]), t % self.bs
                self.kc[b, :, :, o, :] = self.keys[s][t].view(self.hkv, self.d // 8, 8)
                self.vc[b, :, :, o] = self.values[s][t]

    def mask(self):
        packed = trees.pack(self.seen)
        return torch.cat([packed, torch.full((self.T - packed.size(0), packed.size(1)), -1, dtype=torch.int64)]).to(self.device)

    def args(self):
        dev = self.device
        cu, ctx = torch.tensor(self.cu, dtype=torch.int32, device=dev), torch.tensor(self.ctx, dtype=torch.int32, device=dev)
        return [self.q.to(dev), self.kc.to(dev), self.vc.to(dev), self.tables.to(dev), cu, ctx, self.most, self.max_k, 1.0 / math.sqrt(self.d),
                self.mask()]

    def check(self, out):
        u = torch.finfo(self.dtype).eps / 2
        for s, n in enumerate(self.nodes):
            if n == 0:
                continue
            a, b = self.cu[s], self.cu[s + 1]
            want, size, most = trees.attention(self.q[a:b].to(self.device), self.keys[s].to(self.device), self.values[s].to(self.device),
                                               self.seen[a:b, :n].to(self.device), 1.0 / math.sqrt(self.d))
            got = out[a:b].double()
            tol = u * (size + want.abs()) * (1 + 2.0 ** -6) + 2 * (self.d * 2.0 ** -23 * most + 2.0 ** -14) * size
            bad = ~((got - want).abs() <= tol)
            same = (got == want) | (torch.isnan(got) & torch.isnan(want))
            bad &= ~same
            assert not bool(bad.any()), (s, n, self.ctx[s], float((got - want).abs().max()), int(bad.sum()))


HEADS = [(32, 8, 128), (12, 4, 112), (16, 2, 64), (8, 8, 80), (6, 2, 96), (8, 2, 256), (20, 1, 128), (3, 3, 64)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("bs", [8, 16, 32])
def test_attention_of_trees(device, heads, bs, dtype):
    """Trees of one row to more than a word of the mask holds, contexts that are only the tree, whole blocks, ends inside a block."""
    c = Case(3, [1, 24, 64, 7, 70, 0, 33], [45, 700, 0, 1, 333, 17, 64], heads, bs, dtype, device)
    c.check(K.paged_attention_tree(*c.args()))


@gpu
@pytest.mark.parametrize("nodes,priors", [([1], [0]), ([1], [1]), ([1], [5000]), ([5], [4091]), ([64], [2048]), ([200, 3], [100, 9000]), ([16] * 40, list(range(40)))])
def test_attention_of_trees_lengths(device, nodes, priors):
    c = Case(5, nodes, priors, (32, 8, 128), 16, torch.bfloat16, device)
    c.check(K.paged_attention_tree(*c.args()))


@gpu
def test_attention_of_any_mask(device):
    """Masks that are no trees': random ones, rows that see nothing of the tree, and with no keys in front of it nothing at all."""
    def masks(seen, g):
        out = torch.rand(seen.shape, generator=g) < 0.3
        out[::5] = False
        return out

    c = Case(7, [40, 12, 65, 9], [0, 50, 0, 0], (16, 2, 64), 16, torch.float16, device, masks)
    out = K.paged_attention_tree(*c.args())
    c.check(out)
    assert bool((out[0] == 0).all()) and bool((out[55] == 0).all())


@gpu
@pytest.mark.parametrize("bs", [8, 16, 32])
@pytest.mark.parametrize("odd", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite(device, odd, bs):
    """A row of the tree with such keys or values counts for the rows that see it and for no others."""
    c = Case(11, [21, 33], [40, 3], (12, 4, 112), bs, torch.bfloat16, device)
    for s, t in ((0, 44), (0, 60), (1, 20)):
        c.values[s][t, :, 5:70] = odd
        c.values[s][t, 0, 100] = 2.0
    c.fill()
    c.check(K.paged_attention_tree(*c.args()))
    for s, t in ((0, 50), (1, 3)):
        c.keys[s][t] = float("nan")
    c.fill()
    c.check(K.paged_attention_tree(*c.args()))


@gpu
def test_causal_mask_is_that_of_the_prefill(device):
    """A chain of drafts is a chunk of a prompt."""
    c = Case(13, [30, 64, 5], [300, 20, 1000], (32, 8, 128), 16, torch.bfloat16, device, lambda seen, g: torch.cat(
        [torch.ones((n, seen.size(1)), dtype=torch.bool).tril() for n in (30, 64, 5)]))
    args = c.args()
    out = K.paged_attention_tree(*args)
    c.check(out)
    c.check(K.flash_attn_varlen_paged(*args[:-1]))


@gpu
def test_strides_rows_behind_and_dead_sequences(device):
    """q a slice of a wider product, mask rows apart, a table wider than the contexts, rows behind the last sequence left as they were, bits behind
    the tree set."""
    c = Case(17, [9, 0, 30], [100, 40, 7], (12, 4, 112), 16, torch.float16, device, behind=6)
    args = c.args()
    wide = torch.zeros((c.T, 12 * 112 + 2 * 4 * 112), dtype=c.dtype, device=device)
    q = wide[:, :12 * 112].view(c.T, 12, 112)
    q.copy_(args[0])
    mask = torch.full((c.T, 3), -1, dtype=torch.int64, device=device)
    keep = torch.zeros((c.T, 64), dtype=torch.bool)
    for s, n in enumerate(c.nodes):  # (bits from n on are not looked at)
        keep[c.cu[s]:c.cu[s + 1], n:] = True
    mask[:, 1] = args[9][:, 0] | trees.pack(keep)[:, 0].to(device)
    out = torch.full((c.T, 16, 112), 3.0, dtype=c.dtype, device=device)
    got = K.paged_attention_tree(q, *args[1:9], mask[:, 1:2], out=out[:, 2:14])
    assert got.data_ptr() == out[:, 2:14].data_ptr()
    c.check(got)
    assert bool((out[39:] == 3.0).all()) and bool((out[:, :2] == 3.0).all()) and bool((out[:, 14:] == 3.0).all())


@gpu
def test_offsets_beyond_32_bits(device):
    """Blocks at the far end of a cache of more than 2^32 elements."""
    c = Case(19, [20], [70], (8, 8, 128), 16, torch.bfloat16, device)
    far = (1 << 32) // (8 * 128 * 16) + 100
    args = c.args()
    small_k, small_v = args[1], args[2]
    args[1] = torch.empty((far,) + small_k.shape[1:], dtype=c.dtype, device=device)
    args[2] = torch.empty((far,) + small_v.shape[1:], dtype=c.dtype, device=device)
    blocks = small_k.size(0)
    args[1][far - blocks:] = small_k
    args[2][far - blocks:] = small_v
    args[3] = torch.where(args[3] < blocks, args[3] + (far - blocks), args[3])
    c.check(K.paged_attention_tree(*args))


@gpu
def test_workspace_capture_and_streams(device):
    """A caller's workspace, eager and captured, has the bits of the library's; without one a captured call is right too; two streams at once."""
    c = Case(23, [24, 5], [3000, 1200], (32, 8, 128), 16, torch.bfloat16, device)
    args = c.args()
    eager = K.paged_attention_tree(*args)
    c.check(eager)
    need = K.paged_attention_tree_workspace_size(c.T, 32, 128)
    store = torch.full((need,), 255, dtype=torch.uint8, device=device)
    assert torch.equal(K.paged_attention_tree(*args, workspace=store), eager)
    assert not bool((store == 255).all())
    out, bare = torch.empty_like(eager), torch.empty_like(eager)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        K.paged_attention_tree(*args, out=out, workspace=store)
        K.paged_attention_tree(*args, out=bare)
    for _ in range(3):
        out.fill_(float("nan"))
        bare.fill_(float("nan"))
        store.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        c.check(bare)
        assert torch.equal(K.paged_attention_tree(*args), eager)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(K.paged_attention_tree(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(o, eager) for o in outs)


def crowd(heads, nodes, priors):
    """The trees and others beside them, so many that a compute unit has more than one workgroup whatever the columns of one."""
    hq, hkv, _ = heads
    nodes, priors = list(nodes), list(priors)
    while (sum(nodes) * hq // hkv // 16 + len(nodes)) * hkv <= 300 or (max(nodes) * hq // hkv + 15) // 16 * len(nodes) * hkv <= 300:
        nodes.append(20 + 13 * len(nodes) % 41)
        priors.append(7 * len(nodes) % 90)
    return nodes, priors


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("bs", [8, 16, 32])
def test_attention_of_a_crowd(device, heads, bs, dtype):
    """More trees than compute units take at once: columns of a context share its keys."""
    c = Case(29, *crowd(heads, [1, 24, 64, 7, 70, 0, 33], [45, 700, 0, 1, 333, 17, 64]), heads, bs, dtype, device)
    out = K.paged_attention_tree(*c.args())
    c.check(out)
    assert torch.equal(out, K.paged_attention_tree(*c.args()))


@gpu
@pytest.mark.parametrize("heads", [(32, 8, 128), (16, 2, 64)])
@pytest.mark.parametrize("nodes,priors", [([3] * 300, list(range(300))), ([1, 2] * 200, [0, 5] * 200), ([70, 1] + [5] * 320, [900, 0] + [40] * 320),
                                          ([40] * 9, [600] * 9), ([33], [20000])])
def test_bounds_beyond_what_there_is(device, heads, nodes, priors):
    """Many sequences, and bounds of rows and keys that a captured step would have: larger than any."""
    c = Case(31, nodes, priors, heads, 16, torch.bfloat16, device)
    c.check(K.paged_attention_tree(*c.args()))
    args = c.args()
    args[9] = torch.cat([args[9], torch.full((c.T, 3), -1, dtype=torch.int64, device=device)], 1)
    args[6], args[7] = 200, c.max_k + 30000
    args[3] = torch.cat([args[3], torch.full((len(nodes), 30000 // 16 + 1), 1 << 30, dtype=torch.int32, device=device)], 1)
    c.check(K.paged_attention_tree(*args))


@gpu
@pytest.mark.parametrize("heads", [(32, 8, 128), (12, 4, 112), (8, 2, 256)])
def test_bounds_below_what_there_is(device, heads):
    """Rows beyond the bound are left out or computed; those of sequences that it allows for are whole."""
    nodes, priors = crowd(heads, [9, 30, 16], [100, 40, 333])
    for some in (3, len(nodes)):
        c = Case(37, nodes[:some], priors[:some], heads, 16, torch.float16, device)
        args = c.args()
        args[6] = 25
        out = torch.full_like(args[0], 3.0)
        K.paged_attention_tree(*args, out=out)
        whole = K.paged_attention_tree(*c.args())
        for s, n in enumerate(c.nodes):
            rows = slice(c.cu[s], c.cu[s + 1])
            left = (out[rows] == 3.0).flatten(1).all(1)
            assert n > 25 or not bool(left.any())
            err = (out[rows][~left].double() - whole[rows][~left].double()).abs()
            # (both within u (A + |out|) and little more, and A and |out| are at most the values' 5: 2 x 10 eps / 2, twice that allowed)
            assert not bool((err > 20 * torch.finfo(c.dtype).eps).any())


@gpu
@pytest.mark.parametrize("bs", [8, 16])
@pytest.mark.parametrize("odd", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_in_a_crowd(device, odd, bs):
    heads = (16, 8, 64)
    c = Case(41, *crowd(heads, [20, 64], [33, 129]), heads, bs, torch.float16, device)
    rng = random.Random(3)
    for s, n in enumerate(c.nodes):
        for j in rng.sample(range(n), n // 4):  # of the tree's keys and values: rows that do not see them are as they were
            c.values[s][c.ctx[s] - n + j] = odd
            if j % 2:
                c.keys[s][c.ctx[s] - n + j] = odd
    c.fill()
    c.check(K.paged_attention_tree(*c.args()))


@gpu
def test_offsets_beyond_32_bits_in_a_crowd(device):
    heads = (8, 8, 128)
    c = Case(43, *crowd(heads, [70, 20], [70, 5]), heads, 16, torch.bfloat16, device)
    args = c.args()
    small_k, small_v = args[1], args[2]
    blocks = small_k.size(0)
    far = (1 << 32) // (8 * 128 * 16) + 100 + blocks
    args[1] = torch.empty((far,) + small_k.shape[1:], dtype=c.dtype, device=device)
    args[2] = torch.empty((far,) + small_v.shape[1:], dtype=c.dtype, device=device)
    args[1][far - blocks:] = small_k
    args[2][far - blocks:] = small_v
    args[3] = torch.where(args[3] < blocks, args[3] + (far - blocks), args[3])
    c.check(K.paged_attention_tree(*args))


@gpu
@pytest.mark.parametrize("nodes", [[1], [24], [64], [65, 1, 0, 200], [1024], [3] * 100])
def test_tree_rows(device, nodes):
    ctx = [n + (i * 37) % 90 for i, n in enumerate(nodes)]
    cu = [2]
    for n in nodes:
        cu.append(cu[-1] + n)
    T = cu[-1] + 3
    for seed in (1, 3):
        parents = [0, 5] + [x for i, n in enumerate(nodes) for x in tree(n, seed + i)] + [-1, 0, 1]
        if max(nodes) == 1024 and seed == 3:  # a chain
            parents[2:1026] = range(-1, 1023)
        i32 = [torch.tensor(x, dtype=torch.int32, device=device) for x in (parents, cu, ctx)]
        positions, mask = K.tree_rows(*i32, max(nodes))
        want, seen = trees.rows(parents, cu, ctx, max(nodes))
        assert mask.shape == (T, (max(nodes) + 63) // 64)
        assert torch.equal(positions.cpu(), want) and torch.equal(mask.cpu(), trees.pack(seen))


@gpu
def test_tree_rows_beyond_the_bound(device):
    """Rows beyond max_seqlen_q, rounded up to a word, have no mask; the rows' count still says where the tree begins."""
    parents, cu, ctx = list(range(-1, 99)), [0, 100], [130]
    i32 = [torch.tensor(x, dtype=torch.int32, device=device) for x in (parents, cu, ctx)]
    positions, mask = K.tree_rows(*i32, 40)
    want, seen = trees.rows(parents, cu, ctx, 40)
    assert torch.equal(positions.cpu(), want) and torch.equal(mask.cpu(), trees.pack(seen))
    assert positions.tolist()[63:65] == [93, 0]


def _accept_case(nodes, seed, vocab):
    g = random.Random(seed)
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    parents = [x for i, n in enumerate(nodes) for x in tree(n, seed + i)]
    tokens = [g.randrange(vocab) for _ in parents]
    chosen = [g.randrange(vocab) for _ in parents]
    # now and then the model chooses what one of a row's children says
    for a, b in zip(cu, cu[1:]):
        for i in range(a, b):
            up = parents[i]
            if 0 <= up < i - a and g.random() < 0.4:
                chosen[a + up] = tokens[i]
    return cu, parents, tokens, chosen


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("nodes,bs", [([1], 16), ([24], 16), ([30, 0, 64, 1, 5], 8), ([65, 200, 16], 32), ([1024], 16), ([9] * 30, 16)])
def test_tree_accept(device, nodes, bs, dtype):
    """The way, the token behind it and every byte of the caches, for trees that begin anywhere in a block."""
    for seed in (1, 2, 3):
        cu, parents, tokens, chosen = _accept_case(nodes, seed, 3 if seed == 2 else 50)
        g = torch.Generator().manual_seed(seed)
        layers, hkv, d, R = 3, 3, 80, len(nodes)
        cols = (max(nodes) + 2 * bs) // bs
        tables = torch.randperm(R * cols, generator=g).view(R, cols)
        slots = []
        for r, n in enumerate(nodes):
            at = int(torch.randint(bs, (1,), generator=g)) + torch.arange(n)
            slots += (tables[r][at // bs] * bs + at % bs).tolist()
        if seed == 3 and len(slots) > 4:
            slots[3] = -1  # a row that has not been cached moves nowhere and nothing moves there
            slots[2] = R * cols * bs + 7
        caches = [make_cache(R * cols, hkv, d, bs, dtype, gen=g) for _ in range(layers)]
        kcs, vcs = [k.to(device) for k, _ in caches], [v.to(device) for _, v in caches]
        want = trees.accept(tokens, parents, chosen, cu, max(nodes))
        i32 = {k: torch.tensor(v, dtype=torch.int32, device=device) for k, v in (("tokens", tokens), ("parents", parents), ("chosen", chosen), ("cu", cu))}
        slot_t = torch.tensor(slots, dtype=torch.int64 if seed == 2 else torch.int32, device=device)
        kept = K.tree_accept(i32["tokens"], i32["parents"], i32["chosen"], i32["cu"], max(nodes), slot_t, K.CacheList(kcs, vcs))
        bare = K.tree_accept(i32["tokens"], i32["parents"], i32["chosen"], i32["cu"], max(nodes))
        for a, b in zip(kept, bare):
            assert torch.equal(a, b)
        assert kept.lens.tolist() == [len(p) for p, _ in want] and kept.next_tokens.tolist() == [t for _, t in want]
        assert kept.path.tolist() == [p + [-1] * (max(nodes) - len(p)) for p, _ in want]
        limit = R * cols * bs
        for (k, v), kd, vd in zip(caches, kcs, vcs):
            old_k, old_v = k.clone(), v.clone()
            for r, (path, _) in enumerate(want):
                for to, row in enumerate(path):
                    src, dst = slots[cu[r] + row], slots[cu[r] + to]
                    if 0 <= src < limit and 0 <= dst < limit:
                        k[dst // bs, :, :, dst % bs, :] = old_k[src // bs, :, :, src % bs, :]
                        v[dst // bs, :, :, dst % bs] = old_v[src // bs, :, :, src % bs]
            assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)


@gpu
def test_rows_and_accept_captured(device):
    cu, parents, tokens, chosen = _accept_case([24, 60], 4, 4)
    i32 = [torch.tensor(x, dtype=torch.int32, device=device) for x in (tokens, parents, chosen, cu, [100, 200])]
    eager = K.tree_accept(*i32[:4], 60)
    rows = K.tree_rows(i32[1], i32[3], i32[4], 60)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        kept = K.tree_accept(*i32[:4], 60)
        got = K.tree_rows(i32[1], i32[3], i32[4], 60)
    for _ in range(3):
        for t in (*kept, *got):
            t.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*kept, *got), (*eager, *rows)))


@gpu
def test_nothing_to_do(device):
    """No rows, no sequences."""
    none = torch.zeros((0,), dtype=torch.int32, device=device)
    cu = torch.zeros((3,), dtype=torch.int32, device=device)
    ctx = torch.zeros((2,), dtype=torch.int32, device=device)
    positions, mask = K.tree_rows(none, cu, ctx, 0)
    assert positions.shape == (0,) and mask.shape == (0, 0)
    kept = K.tree_accept(none, none, none, cu, 8)
    assert kept.lens.tolist() == [0, 0] and kept.next_tokens.tolist() == [-1, -1] and bool((kept.path == -1).all())
    c = Case(29, [4], [9], (8, 8, 64), 16, torch.float16, device)
    args = c.args()
    args[0], args[9] = args[0][:0], args[9][:0]
    args[6] = 0
    assert K.paged_attention_tree(*args).shape == (0, 8, 64)


@gpu
def test_refusals(device):
    c = Case(31, [10, 80], [50, 60], (12, 4, 112), 16, torch.float16, device)
    good = c.args()

    def refuse(match, **changes):
        names = ["q", "kc", "vc", "tables", "cu", "ctx", "max_q", "max_k", "scale", "mask"]
        args = [changes.pop(n, a) for n, a in zip(names, good)]
        with pytest.raises(HipAttnError, match=match):
            K.paged_attention_tree(*args, **changes)

    refuse("tree_mask must be int64", mask=good[9].to(torch.int32))
    refuse("does not hold 80 rows", mask=good[9][:, :1])
    refuse("tree_mask has 89 rows", mask=good[9][:89])
    refuse("caches must have q's dtype", q=good[0].bfloat16())
    refuse("only fp16 and bf16", q=good[0].float(), kc=good[1].float(), vc=good[2].float())
    refuse("out is", out=torch.empty(good[0].shape, dtype=torch.float32, device=device))
    refuse("head size 72 not supported", q=good[0][:, :, :72])
    refuse("block-table columns", max_k=10000)
    refuse("workspace must be u8", workspace=torch.empty((1 << 20,), dtype=torch.int32, device=device))
    refuse("is too small", workspace=torch.empty((1 << 10,), dtype=torch.uint8, device=device))
    refuse("need 2 rows", tables=good[3][:1])
    refuse("int32", ctx=good[5].long())
    i32 = [torch.tensor(x, dtype=torch.int32, device=device) for x in ([-1, 0, 1], [0, 3], [9])]
    with pytest.raises(HipAttnError, match="at most 1024 rows"):
        K.tree_rows(*i32, 1025)
    with pytest.raises(HipAttnError, match="at most 1024 rows"):
        K.tree_accept(i32[0], i32[0], i32[0], i32[1], 1025)
    with pytest.raises(HipAttnError, match="parents must be int32"):
        K.tree_rows(i32[0].long(), i32[1], i32[2], 3)
    with pytest.raises(HipAttnError, match="chosen has 2 elements"):
        K.tree_accept(i32[0], i32[0], i32[0][:2], i32[1], 3)
    with pytest.raises(HipAttnError, match="or not at all"):
        K.tree_accept(i32[0], i32[0], i32[0], i32[1], 3, slot_mapping=i32[0])
    kc, vc = (t.to(device) for t in make_cache(4, 2, 64, 16, torch.float16, fill=0.0))
    with pytest.raises(HipAttnError, match="or not at all"):
        K.tree_accept(i32[0], i32[0], i32[0], i32[1], 3, caches=K.CacheList([kc], [vc]))
    with pytest.raises(HipAttnError, match="one type, one shape"):
        K.CacheList([kc, kc[:2]], [vc, vc])
    with pytest.raises(HipAttnError, match="2 key caches and 1 value caches"):
        K.CacheList([kc, kc], [vc])


def test_cpu_tensors_are_refused():
    c = Case(37, [4], [9], (8, 8, 64), 16, torch.float16, "cpu")
    with pytest.raises(HipAttnError, match="expected a GPU tensor"):
        K.paged_attention_tree(*c.args())
    i32 = [torch.tensor(x, dtype=torch.int32) for x in ([-1, 0, 1], [0, 3], [9])]
    with pytest.raises(HipAttnError, match="expected a GPU tensor"):
        K.tree_rows(*i32, 3)
    with pytest.raises(HipAttnError, match="expected a GPU tensor"):
        K.tree_accept(i32[0], i32[0], i32[0], i32[1], 3)
    kc, vc = make_cache(4, 2, 64, 16, torch.float16, fill=0.0)
    with pytest.raises(HipAttnError, match="expected GPU tensors"):
        K.CacheList([kc], [vc])


def test_oracle_of_trees():
    """The restatement on a tree that is checked by hand."""
    parents, cu = [-1, 0, 0, 1, 2, 3], [0, 6]
    positions, seen = trees.rows(parents, cu, [16], 6)
    assert positions.tolist() == [10, 11, 11, 12, 12, 13]
    assert [[j for j in range(6) if seen[i, j]] for i in range(6)] == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 2, 4], [0, 1, 3, 5]]
    assert trees.pack(seen).tolist() == [[1], [3], [5], [11], [21], [43]]
    assert trees.accept([9, 5, 6, 7, 8, 4], parents, [6, 0, 8, 0, 3, 0], cu, 6) == [([0, 2, 4], 3)]
    assert trees.accept([9, 5, 6], [-1, 0, 0], [7, 0, 0], [0, 3, 3], 3) == [([0], 7), ([], -1)]
