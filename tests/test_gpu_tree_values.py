"""Tree attention over keys and values that are not finite, checked to the value: where the 64-bit restatement of oracle/trees.py is infinite or NaN the
kernel's output is the same, of the same sign, and where it is finite the tolerance is that of test_gpu_trees.py.

A probability of zero times an infinity is NaN, in 64 bits as here, so none may be rounded to zero here alone: scores of d products of normal
numbers over sqrt(d) stay within some +-6, probabilities above e^-12 = 6e-6 of the largest, where fp16 has numbers down to 6e-8."""
import math
import random

import pytest
import torch

from aici_amd import kernels as K
from oracle import trees

from test_gpu_trees import Case, crowd

pytestmark = pytest.mark.gpu


def check(c, out):
    """As Case.check, and the same infinities and NaN; how many outputs should be +inf, -inf and NaN."""
    u, counts = torch.finfo(c.dtype).eps / 2, [0, 0, 0]
    for s, n in enumerate(c.nodes):
        if n == 0:
            continue
        a, b = c.cu[s], c.cu[s + 1]
        want, size, most = trees.attention(c.q[a:b].to(c.device), c.keys[s].to(c.device), c.values[s].to(c.device), c.seen[a:b, :n].to(c.device),
                                           1.0 / math.sqrt(c.d))
        got, finite = out[a:b].double(), torch.isfinite(want)
        tol = u * (size + want.abs()) * (1 + 2.0 ** -6) + 2 * (c.d * 2.0 ** -23 * most + 2.0 ** -14) * size
        assert bool(torch.isfinite(tol[finite]).all())
        good = torch.where(finite, (got - want).abs() <= tol, (got == want) | (torch.isnan(got) & torch.isnan(want)))
        assert bool(good.all()), (s, n, c.ctx[s], int((~good).sum()), want[~good][:4].tolist(), got[~good][:4].tolist())
        for i, kind in enumerate((want == math.inf, want == -math.inf, torch.isnan(want))):
            counts[i] += int(kind.sum())
    return counts


def spoil(c, odd, seed):
    """Values that are not finite: of a third of the trees' rows, of some keys in front of a tree (the last ones, whose pair reaches into it, among them),
    all elements of some heads or a few."""
    rng = random.Random(seed)
    for s, (n, ctx) in enumerate(zip(c.nodes, c.ctx)):
        for j in rng.sample(range(n), n // 3):
            c.values[s][ctx - n + j, rng.randrange(c.hkv), rng.randrange(c.d // 2):] = odd
        front = ctx - n
        for t in rng.sample(range(front), min(front, 2)) + ([front - 1] if front > 0 else []):
            c.values[s][t, rng.randrange(c.hkv), rng.randrange(c.d)] = odd
    c.fill()


@pytest.mark.parametrize("odd", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("bs,dtype", [(8, torch.float16), (16, torch.bfloat16), (16, torch.float16), (32, torch.bfloat16)])
@pytest.mark.parametrize("heads", [(12, 4, 112), (16, 8, 64), (8, 2, 256)])
@pytest.mark.parametrize("many", [False, True])
def test_values(device, many, heads, bs, odd, dtype):
    nodes, priors = [21, 33, 64], [40, 3, 129]
    c = Case(61, *(crowd(heads, nodes, priors) if many else (nodes, priors)), heads, bs, dtype, device)
    spoil(c, odd, 5)
    plus, minus, nan = check(c, K.paged_attention_tree(*c.args()))
    assert (plus > 100) == (odd == math.inf) and (minus > 100) == (odd == -math.inf) and (nan > 100) == (odd != odd)


@pytest.mark.parametrize("many", [False, True])
def test_infinities_of_both_signs(device, many):
    """A row that sees both is NaN, one that sees one of them has it."""
    heads = (12, 4, 112)
    nodes, priors = [50, 20], [70, 9]
    c = Case(67, *(crowd(heads, nodes, priors) if many else (nodes, priors)), heads, 16, torch.bfloat16, device)
    rng = random.Random(7)
    for s, (n, ctx) in enumerate(zip(c.nodes, c.ctx)):
        for j in rng.sample(range(n), n // 2):
            c.values[s][ctx - n + j] = rng.choice([math.inf, -math.inf])
    c.fill()
    plus, minus, nan = check(c, K.paged_attention_tree(*c.args()))
    assert nan > 100 and plus + minus > 100


@pytest.mark.parametrize("odd", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_of_long_contexts(device, odd, dtype):
    """Parts of a context whose results a merge adds up, in trees of one and of several words of the mask."""
    c = Case(71, [24, 200, 1], [1500, 3000, 4000], (32, 8, 128), 16, dtype, device)
    spoil(c, odd, 9)
    counts = check(c, K.paged_attention_tree(*c.args()))
    assert max(counts) > 1000


@pytest.mark.parametrize("many", [False, True])
def test_keys(device, many):
    """One element of some keys is infinite: a row's score of such a key is infinite, of either sign, and the row NaN or without that key."""
    heads = (16, 8, 64)
    nodes, priors = [20, 64], [33, 129]
    c = Case(73, *(crowd(heads, nodes, priors) if many else (nodes, priors)), heads, 16, torch.float16, device)
    rng = random.Random(11)
    for s, (n, ctx) in enumerate(zip(c.nodes, c.ctx)):
        for j in rng.sample(range(n), n // 4):
            c.keys[s][ctx - n + j, :, rng.randrange(64)] = rng.choice([math.inf, -math.inf])
    c.fill()
    _, _, nan = check(c, K.paged_attention_tree(*c.args()))
    assert nan > 100
