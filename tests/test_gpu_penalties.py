"""Penalties, bias and allow-mask on logits (kernels.penalize_logits) against a token-by-token restatement in 64 bits.

Tolerance, per element: half a step of the output's type, and six fp32 operations, 2^-24 each of at most the largest intermediate value."""
import math

import numpy as np
import pytest
import torch

from aici_amd import kernels as K
from aici_amd import llama
from oracle import steps

pytestmark = pytest.mark.gpu


def make(seed, S, V, dtype, lens, bias=False, mask=False):
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    hot = rng.integers(0, V, 20)
    said = [[int(hot[rng.integers(20)]) if rng.random() < 0.5 else int(rng.integers(-2, V + 3)) for _ in range(n)] for n in lens]
    c = dict(logits=(4 * torch.randn((S, V), generator=g)).to(dtype), said=said, prompt=[int(rng.integers(0, n + 2)) for n in lens],
             repetition=0.7 + torch.rand(S, generator=g), frequency=torch.rand(S, generator=g) - 0.2, presence=torch.rand(S, generator=g),
             bias=None, allowed=None)
    if bias:
        c["bias"] = torch.where(torch.rand((S, V + 3), generator=g) < 0.1, -math.inf, torch.randn((S, V + 3), generator=g))
    if mask:
        c["allowed"] = torch.rand((S, V), generator=g) < 0.3
    return c


def want(c):
    return steps.penalize(c["logits"], c["said"], c["prompt"], c["repetition"], c["frequency"], c["presence"], c["bias"], c["allowed"])


def args(c, device, offsets=torch.int64):
    flat = [t for s in c["said"] for t in s]
    at = np.cumsum([0] + [len(s) for s in c["said"]]).tolist()
    return dict(history=torch.tensor(flat, dtype=torch.int32, device=device), history_offsets=torch.tensor(at, dtype=offsets, device=device),
                prompt_lens=torch.tensor(c["prompt"], dtype=torch.int32, device=device), repetition=c["repetition"].to(device),
                frequency=c["frequency"].to(device), presence=c["presence"].to(device),
                bias=None if c["bias"] is None else c["bias"].to(device),
                mask=None if c["allowed"] is None else steps.allow_bits(c["allowed"]).to(device))


def check(got, c, expect):
    got = got.cpu()
    half = torch.finfo(got.dtype).eps / 2
    expect = expect.to(torch.float64)
    fin = torch.isfinite(expect)
    assert torch.equal(got.double()[~fin], expect[~fin])
    counts = max([len(s) for s in c["said"]] + [1])
    largest = 2 * c["logits"].double().abs() + counts + 8
    over = (got.double() - expect).abs() - (1.01 * half * expect.abs() + 6 * 2.0 ** -24 * largest)
    assert bool((over[fin] <= 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("S,V,lens", [(1, 1, [3]), (2, 7, [0, 5]), (3, 1000, [1, 700, 33]), (5, 8192, [64, 0, 63, 5000, 1]), (2, 8193, [513, 2000]),
                                      (4, 50003, [30, 3000, 1, 0]), (2, 128256, [100, 4000])])
def test_penalties(device, dtype, S, V, lens):
    for n, (bias, mask) in enumerate([(False, False), (True, False), (False, True), (True, True)]):
        c = make(10 * n + S, S, V, dtype, lens, bias, mask)
        a, expect = args(c, device, torch.int64 if n % 2 else torch.int32), want(c)
        check(K.penalize_logits(c["logits"].to(device), **a), c, expect)
        check(K.penalize_logits(c["logits"].to(device), out_dtype=torch.float32, **a), c, expect)
        x = c["logits"].to(device)
        assert K.penalize_logits(x, out=x, **a) is x
        check(x, c, expect)


def test_a_short_mask_bars_what_lies_behind_it(device):
    c = make(8, 2, 3000, torch.bfloat16, [40, 300], False, True)
    a, short = args(c, device), 1000
    a["mask"] = a["mask"][:, :short // 8].contiguous()
    c["allowed"][:, short:] = False
    check(K.penalize_logits(c["logits"].to(device), **a), c, want(c))


def test_untouched_logits_keep_their_bits(device):
    """No penalty, nothing said, nothing barred: the logits as they are, infinities and NaN among them."""
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = torch.randn((2, 5000), device=device).to(dtype)
        x[0, 3], x[1, 4], x[0, 7] = math.inf, -math.inf, math.nan
        none = torch.zeros((3,), dtype=torch.int32, device=device)
        y = K.penalize_logits(x, torch.zeros((0,), dtype=torch.int32, device=device), none)
        assert torch.equal(y.nan_to_num(123.0), x.nan_to_num(123.0)) and bool(torch.isnan(y[0, 7]))


def test_one_token_said_over_and_over(device):
    V = 40000
    c = dict(logits=torch.zeros((1, V), dtype=torch.float32), said=[[777] * 20000], prompt=[5], repetition=[1.5], frequency=[0.25], presence=[1.0])
    c["logits"][0, 777] = 3.0
    out = K.penalize_logits(c["logits"].to(device), torch.full((20000,), 777, dtype=torch.int32, device=device),
                            torch.tensor([0, 20000], device=device), torch.tensor([5], dtype=torch.int32, device=device),
                            torch.tensor([1.5], device=device), torch.tensor([0.25], device=device), torch.tensor([1.0], device=device))
    assert float(out[0, 777]) == 2.0 - 0.25 * 19995 - 1.0 and int((out != 0).sum()) == 1


def test_strides_rows_and_frames(device):
    """Logits as columns of a wider array, rows of bias and mask picked by bias_rows, an output in a frame."""
    c = make(5, 4, 999, torch.bfloat16, [10, 50, 3, 8], True, True)
    pick = [2, 0, 3, 1]
    order = torch.tensor(pick)
    a = args({**c, "bias": c["bias"][torch.argsort(order)], "allowed": c["allowed"][torch.argsort(order)]}, device)
    wide = torch.full((4, 1200), 9.0, dtype=torch.bfloat16, device=device)
    wide[:, 101:1100] = c["logits"].to(device)
    frame = torch.full((4, 1100), 7.0, dtype=torch.float32, device=device)
    K.penalize_logits(wide[:, 101:1100], out=frame[:, 51:1050], bias_rows=torch.tensor(pick, dtype=torch.int32, device=device), **a)
    check(frame[:, 51:1050], c, want(c))
    assert bool((frame[:, :51] == 7).all()) and bool((frame[:, 1050:] == 7).all())


def test_sampling_behind_penalties(device):
    """The greedy end of a step: the token that the restated logits hold highest."""
    c = make(6, 3, 2000, torch.float32, [300, 20, 1], False, True)
    a = args(c, device)
    masks = a.pop("mask")
    a.pop("bias")
    pen = llama.Penalties(**a)
    tokens = llama.aici_greedy(c["logits"].to(device), masks, pen)
    assert tokens.tolist() == want(c).argmax(1).tolist()
    drawn = llama.aici_sample(c["logits"].to(device), masks, torch.zeros(3, device=device), torch.ones(3, device=device),
                              torch.zeros(3, device=device), penalties=pen)
    assert torch.equal(drawn, tokens)


def test_replays(device):
    c = make(7, 2, 3001, torch.float16, [100, 60], True)
    a, x = args(c, device), c["logits"].to(device)
    out = torch.empty_like(x)
    K.penalize_logits(x, out=out, **a)
    eager = out.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        K.penalize_logits(x, out=out, **a)
    for k in range(3):
        out.zero_()
        x.copy_(c["logits"].to(device) + k)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, K.penalize_logits(x, **a)) and (k > 0 or torch.equal(out, eager))


def test_rows_beyond_32_bits(device):
    """Rows of logits and of the output that lie more than 2^31 elements apart."""
    V, apart = 1003, (1 << 31) + 24
    store, out_store = (torch.empty((apart + V,), dtype=torch.bfloat16, device=device) for _ in range(2))
    logits, out = (s.as_strided((2, V), (apart, 1)) for s in (store, out_store))
    g = torch.Generator().manual_seed(5)
    x = torch.randn((2, V), generator=g).to(torch.bfloat16)
    logits.copy_(x)
    said = torch.randint(0, V, (90,), generator=g, dtype=torch.int32)
    offsets = torch.tensor([0, 40, 90], device=device)
    knobs = dict(repetition=torch.tensor([1.3, 0.8], device=device), presence=torch.tensor([0.5, -0.25], device=device))
    K.penalize_logits(logits, said.to(device), offsets, out=out, **knobs)
    small = K.penalize_logits(x.to(device), said.to(device), offsets, **knobs)
    assert torch.equal(out, small) and not torch.equal(small, x.to(device))
