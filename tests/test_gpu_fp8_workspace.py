"""Steps of a model on weights of 8 bits that are captured on one stream and replayed on two at once: with workspaces of their own they hand one another
no rounded rows.  Every projection, the last one too, has weights of 8 bits here, and attention its own workspace, so that nothing else of a step lies in
memory that belongs to the capture's stream."""
import random

import pytest
import torch

from aici_amd import kernels as K
from aici_amd import llama, paged
from aici_amd._lib import HipAttnError

pytestmark = pytest.mark.gpu
CFG = llama.LlamaConfig(1024, 1536, 1024, 2, 8, 2, 1e-5, 4096, 10000.0, torch.bfloat16)
BS = 16


def model_of(device, fp8=True):
    weights = llama.random_weights(CFG, 9, std=0.05)
    if fp8:
        weights["lm_head"] = llama.Fp8Weight(*K.quantize_weight_fp8(weights["lm_head"]))
    return llama.Llama(CFG, weights, device, fp8=fp8)


class Step:
    """A prompt in the caches, and the tree that follows it."""

    def __init__(self, model, seed, prompt, drafts, device):
        rng, alloc = random.Random(seed), paged.BlockAllocator(BS, 40)
        self.model = model
        self.caches = [paged.alloc_gpu_cache_layer(40, CFG.num_key_value_heads, CFG.head_dim, BS, CFG.dtype, device) for _ in range(2)]
        for kc, vc in self.caches:
            kc.zero_()
            vc.zero_()
        tokens = [rng.randrange(1000) for _ in range(prompt + 1 + drafts)]
        alloc.alloc_seq(1, prompt)
        first = paged.BatchInfoBuilder(BS, 4096, 1)
        first.sched_out(alloc, 1, tokens[:prompt], 0)
        self.prompt = first.finish().to(device)
        model.forward(self.prompt, self.caches, paged_prefill=True, fused=True)
        assert not alloc.append_slots(1, prompt, len(tokens))
        then = paged.BatchInfoBuilder(BS, 4096, 1)
        then.sched_out(alloc, 1, tokens, prompt)
        parents = [-1] + [rng.randrange(i + 1) for i in range(drafts)]
        self.batch = then.finish().to(device).with_trees(torch.tensor(parents, dtype=torch.int32, device=device))
        self.store = torch.empty((model.workspace_size(self.batch),), dtype=torch.uint8, device=device)
        self.fp8 = torch.empty((model.fp8_workspace_size(self.batch),), dtype=torch.uint8, device=device)

    def run(self, **kw):
        return self.model.forward(self.batch, self.caches, fused=True, workspace=self.store, **kw)


def test_captured_on_one_stream_replayed_on_two(device):
    model = model_of(device)
    steps = [Step(model, seed, prompt, drafts, device) for seed, prompt, drafts in ((1, 200, 40), (2, 77, 150), (3, 30, 8))]
    beside = Step(model, 5, 120, 60, device)
    want, want_beside = [s.run() for s in steps], beside.run()
    assert all(torch.equal(s.run(fp8_workspace=s.fp8), w) for s, w in zip(steps, want))
    side, graphs, got = torch.cuda.Stream(), [], []
    torch.cuda.synchronize()
    for s in steps:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            got.append(s.run(fp8_workspace=s.fp8))
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(10):
        for s, g in zip(steps, got):
            s.fp8.fill_(255)
            g.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        with torch.cuda.stream(side):
            eager = beside.run()  # (its rounded rows lie in the library's memory of the capture's stream)
        torch.cuda.synchronize()
        assert torch.equal(eager, want_beside) and all(torch.equal(g, w) for g, w in zip(got, want))
        assert not any(bool((s.fp8[:256] == 255).all()) for s in steps)


def test_sizes(device):
    model = model_of(device)
    step = Step(model, 4, 50, 60, device)
    rows = step.batch.tokens.numel()
    x = {k: torch.zeros((rows, k), dtype=CFG.dtype, device=device) for k in (1024, 1536)}
    weights = [w.data for layer in model.layers for w in layer.values() if isinstance(w, llama.Fp8Weight)] + [model.lm_head.data]
    need = max(K.linear_fp8_workspace_size(x[w.size(1)], w) for w in weights)
    assert model.fp8_workspace_size(step.batch) == need > 0
    with pytest.raises(HipAttnError, match="workspace has"):
        step.run(fp8_workspace=step.fp8[:need // 2 // 256 * 256])
    plain = model_of(device, fp8=False)
    assert plain.fp8_workspace_size(step.batch) == 0
    want = plain.forward(step.prompt, step.caches, paged_prefill=True, fused=True)
    assert torch.equal(plain.forward(step.prompt, step.caches, paged_prefill=True, fused=True, fp8_workspace=step.fp8), want)
