"""Tree attention over caches whose blocks and heads lie apart: everything that its checks of strides let through, against the 64-bit restatement of
oracle/trees.py.  Values need no more than 8-byte boundaries, where the kernel that copies them in pieces of 16 bytes is not the one that runs."""
import pytest
import torch

from aici_amd import kernels as K

from test_gpu_trees import HEADS, Case, crowd

pytestmark = pytest.mark.gpu


def apart(t, head_pad, block_pad, first=0):
    """The cache with that many elements behind every head and every block, and in front of the first; NaN in all of them."""
    blocks, heads = t.shape[:2]
    inner = t[0, 0].numel()
    head = inner + head_pad
    block = heads * head + block_pad
    store = torch.full((first + blocks * block,), float("nan"), dtype=t.dtype, device=t.device)
    out = store[first:].as_strided(t.shape, (block, head, *t.stride()[2:]))
    out.copy_(t)
    return out


PADS = [(4, 0), (0, 4), (4, 4), (8, 16), (12, 20)]


@pytest.mark.parametrize("pads", PADS)
@pytest.mark.parametrize("heads", [(32, 8, 128), (12, 4, 112), (20, 1, 128), (8, 2, 256), (3, 3, 64)])
@pytest.mark.parametrize("bs", [8, 16, 32])
def test_values_apart_in_a_crowd(device, heads, bs, pads):
    """As many trees as have their columns share keys in LDS, where the values' boundaries allow for it."""
    assert heads in HEADS
    c = Case(47, *crowd(heads, [1, 40, 64, 0, 33], [45, 300, 0, 17, 64]), heads, bs, torch.bfloat16, device)
    args = c.args()
    args[2] = apart(args[2], *pads)
    args[1] = apart(args[1], 8 * (pads[0] // 8), 8 * (pads[1] // 8))
    out = K.paged_attention_tree(*args)
    c.check(out)
    assert not bool(torch.isnan(out).any())


@pytest.mark.parametrize("pads", PADS)
@pytest.mark.parametrize("nodes,priors", [([5], [4091]), ([64], [2048]), ([200, 3], [100, 20000]), ([8] * 40, list(range(100, 2100, 50)))])
def test_values_apart_lengths(device, nodes, priors, pads):
    """Few trees, parts of long contexts, and 32 columns to a kv head."""
    c = Case(53, nodes, priors, (32, 8, 128), 16, torch.float16, device)
    args = c.args()
    args[2] = apart(args[2], *pads, first=8)
    c.check(K.paged_attention_tree(*args))


@pytest.mark.parametrize("nodes,priors", [([24], [1500]), ([200, 3], [100, 9000]), ([40] * 9, [600] * 9), ([1, 24, 64, 7, 70, 0, 33], [45, 700, 0, 1, 333, 17, 64])])
@pytest.mark.parametrize("many", [False, True])
def test_out_over_q(device, nodes, priors, many):
    """out is q itself, and lies beside q in rows of one wider matrix: the bits of a place of its own."""
    heads = (32, 8, 128)
    c = Case(59, *(crowd(heads, nodes, priors) if many else (nodes, priors)), heads, 16, torch.bfloat16, device)
    args = c.args()
    want = K.paged_attention_tree(*args)
    c.check(want)
    wide = torch.zeros((c.T, 2, 32, 128), dtype=c.dtype, device=device)
    wide[:, 0] = args[0]
    beside = K.paged_attention_tree(wide[:, 0], *args[1:], out=wide[:, 1])
    assert torch.equal(beside, want) and torch.equal(wide[:, 0], args[0])
    assert torch.equal(K.paged_attention_tree(*args, out=args[0]), want)
