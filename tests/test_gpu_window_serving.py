"""A small model served over a sliding window with everything on the device: chunks and decode rows by `paged.DeviceBlocks`, attention with
window and sinks, penalties, allow-masks and the greedy token; the generation step is captured once and replayed, while blocks that the
window passes go from one request to another.  Every step's logits against a 64-bit restatement of the model over the whole sequence.

Tolerance: 2 layers of 10 tensors that are rounded to fp16 and 3 more, half a step each (2^-11 of their norm), no map between them taken to stretch
a relative error more than twofold: 23 x 2 x 2^-11 = 0.0225 of the logits' norm."""
import math
from dataclasses import replace

import pytest
import torch

from aici_amd import llama, paged
from oracle import steps

pytestmark = pytest.mark.gpu
CFG = llama.LlamaConfig(512, 768, 1000, 2, 8, 2, 1e-5, 512, 10000.0, torch.float16)
TOLERANCE = 23 * 2 * 2.0 ** -11


def reference(weights, table, tokens, device, window, sinks):
    """Logits of the last token of a sequence, 64 bits."""
    w = {k: v.to(device).double() for k, v in weights.items()}
    n, d, hq, hkv = len(tokens), CFG.head_dim, CFG.num_attention_heads, CFG.num_key_value_heads
    pos = torch.arange(n, device=device)
    cos, sin = (t[:, None, :] for t in table[:n].double().chunk(2, 1))
    seen = pos[None, :] <= pos[:, None]
    if window is not None:
        seen &= (pos[None, :] > pos[:, None] - window) | (pos[None, :] < sinks)

    def norm(x, scale):
        return x * torch.rsqrt((x * x).mean(1, keepdim=True) + CFG.rms_norm_eps) * scale

    def rotate(x):
        a, b = x.chunk(2, 2)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], 2)

    x = w["model.embed_tokens"][torch.tensor(tokens, device=device)]
    for i in range(CFG.num_hidden_layers):
        p = f"model.layers.{i}."
        h = norm(x, w[p + "input_layernorm"])
        q, k, v = (h @ w[p + f"self_attn.{c}_proj"].t().contiguous() for c in "qkv")
        q, k, v = rotate(q.view(n, hq, d)), rotate(k.view(n, hkv, d)), v.view(n, hkv, d)
        y = torch.empty_like(q)
        for head in range(hq):
            s = q[:, head] @ k[:, head // (hq // hkv)].t().contiguous() / math.sqrt(d)
            y[:, head] = torch.softmax(s.masked_fill(~seen, -math.inf), 1) @ v[:, head // (hq // hkv)].contiguous()
        x = x + y.reshape(n, hq * d) @ w[p + "self_attn.o_proj"].t().contiguous()
        h = norm(x, w[p + "post_attention_layernorm"])
        gate = h @ w[p + "mlp.gate_proj"].t().contiguous()
        x = x + (gate * torch.sigmoid(gate) * (h @ w[p + "mlp.up_proj"].t().contiguous())) @ w[p + "mlp.down_proj"].t().contiguous()
    return norm(x[-1:], w["model.norm"])[0] @ w["lm_head"].t().contiguous()


@pytest.mark.parametrize("window,sinks,blocks", [(41, 5, 21), (None, 0, 40)])
def test_generation(device, window, sinks, blocks):
    """With a window and sinks in a small pool, and over whole contexts."""
    R, L, V = 4, 256, CFG.vocab_size
    weights = llama.random_weights(CFG, 3, std=0.05)
    model = llama.Llama(replace(CFG, sliding_window=window, attention_sinks=sinks), weights, device)
    # 21 blocks: four windows and their sinks hold five each; without letting go the sequences would need more
    pool = paged.DeviceBlocks(16, blocks, R, L, device, -1 if window is None else window - 1, sinks)
    caches = [paged.alloc_gpu_cache_layer(blocks, CFG.num_key_value_heads, CFG.head_dim, 16, CFG.dtype, device) for _ in range(2)]
    for kc, vc in caches:
        kc.fill_(float("nan"))
        vc.fill_(float("nan"))
    g = torch.Generator().manual_seed(9)
    allowed = torch.rand((R, V), generator=g) < 0.4
    masks = steps.allow_bits(allowed).to(device)
    history = torch.full((R, L), -1, dtype=torch.int32, device=device)
    knobs = {k: torch.full((R,), v, device=device) for k, v in (("repetition", 1.2), ("frequency", 0.02), ("presence", 0.05))}
    prompt = torch.zeros((R,), dtype=torch.int32, device=device)
    penalties = llama.Penalties(history.view(-1), torch.arange(R + 1, device=device) * L, prompt, **knobs)
    tokens = torch.zeros((R,), dtype=torch.int32, device=device)
    said = [[] for _ in range(R)]

    def finish(logits, context_lens):
        """The step's end: the token, and the history it goes into."""
        picked = llama.aici_greedy(logits, masks, penalties)
        running = context_lens > 0
        tokens.copy_(torch.where(running, picked, tokens))
        at = context_lens.long()[:, None]
        history.scatter_(1, at, torch.where(running[:, None], tokens[:, None], history.gather(1, at)))

    def check(logits, before, rows):
        for r in rows:
            ref = reference(weights, model.rotary.cos_sin, said[r], device, window, sinks)
            err = float((logits[r].double() - ref).norm() / ref.norm())
            assert err <= TOLERANCE, (r, len(said[r]), err)
            knob = [float(knobs[k][0]) for k in ("repetition", "frequency", "presence")]
            pen = steps.penalize(logits[r:r + 1].cpu(), [said[r]], [int(prompt[r])], *([k] for k in knob), None, allowed[r:r + 1])[0]
            token = int(tokens[r])
            # (the highest of them, up to the rounding of the penalised logits to fp16)
            assert float(pen[token]) >= float(pen.max()) - 2 * 2.0 ** -11 * float(pen.max().abs()) - 1e-4
            said[r].append(token)

    def prompts(lens):
        """Prompt chunks for the requests that have a length; the others idle, or end where it is negative."""
        new = torch.tensor(lens, dtype=torch.int32, device=device)
        step = pool.step(new, 150)
        for r, n in enumerate(lens):
            if n:
                said[r] = torch.randint(0, V, (max(n, 0),), generator=g).tolist()
                history[r] = -1
                history[r, :max(n, 0)] = torch.tensor(said[r], dtype=torch.int32)
                prompt[r] = max(n, 0)
        flat = [t for r, n in enumerate(lens) if n > 0 for t in said[r]]
        ids = torch.zeros((150,), dtype=torch.int32, device=device)
        ids[:len(flat)] = torch.tensor(flat, dtype=torch.int32)
        logits = model.forward(pool.batch_info(step, ids, max_new=max(lens)), caches, fused=True)
        assert torch.equal(logits, model.forward(pool.batch_info(step, ids, max_new=max(lens)), caches))
        assert step.served.tolist() == [max(n, 0) for n in lens]
        finish(logits, step.context_lens)
        check(logits, None, [r for r, n in enumerate(lens) if n > 0])

    prompts([37, 5, 64, 20])
    new = torch.ones((R,), dtype=torch.int32, device=device)

    def generate():
        step = pool.step(new, R, rows_per_request=1)
        logits = model.forward(pool.batch_info(step, tokens), caches, fused=True)
        finish(logits, step.context_lens)
        return step, logits

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step, logits = generate()
    torch.cuda.synchronize()
    check(logits, None, range(R))
    with torch.cuda.graph(graph, stream=side):
        step, logits = generate()
    for k in range(70):
        if k == 30:  # request 2 ends, another takes its row; the others wait
            new.copy_(torch.tensor([0, 0, -1, 0], dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            prompts([0, 0, 45, 0])
            new.fill_(1)
        if k == 50:  # request 1 idles for a step
            new.copy_(torch.tensor([1, 0, 1, 1], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        rows = [r for r in range(R) if int(step.served[r]) == 1]
        assert rows == ([0, 2, 3] if k == 50 else [0, 1, 2, 3])
        if k % 9 == 0 or k > 66:
            check(logits, None, rows)
        else:
            for r in rows:
                said[r].append(int(tokens[r]))
        new.fill_(1)
    assert window is None or int(pool.ring_ends[0]) > blocks  # blocks have been handed out more than once
    assert [len(s) for s in said] == [37 + 72, 5 + 71, 45 + 41, 20 + 72]


def test_captured_chunks_with_a_workspace(device):
    """A captured prompt step of the model, its attention in a workspace of the caller's, has the eager step's bits."""
    R, T = 2, 20
    cfg = replace(CFG, max_position_embeddings=3200)
    model = llama.Llama(replace(cfg, sliding_window=2500, attention_sinks=4), llama.random_weights(cfg, 5, "cpu"), device)
    pool = paged.DeviceBlocks(16, 200, R, 3200, device, 2499, 4)
    caches = [paged.alloc_gpu_cache_layer(200, CFG.num_key_value_heads, CFG.head_dim, 16, CFG.dtype, device) for _ in range(2)]
    for kc, vc in caches:
        kc.zero_()
        vc.zero_()
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, CFG.vocab_size, (3000,), generator=g).to(torch.int32).to(device)
    for n in (3000, T):
        step = pool.step(torch.tensor([n, 0], dtype=torch.int32, device=device), n)
        batch = pool.batch_info(step, ids[:n], max_new=n)
        eager = model.forward(batch, caches, fused=True)
    need = model.workspace_size(batch)
    assert need == 16 * T * CFG.num_attention_heads * (CFG.head_dim + 2) * 4
    assert llama.Llama(cfg, llama.random_weights(cfg, 5, "cpu"), device).workspace_size(batch) == 0
    store = torch.full((need,), 255, dtype=torch.uint8, device=device)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        assert torch.equal(model.forward(batch, caches, fused=True, workspace=store), eager)
    torch.cuda.synchronize()
    assert not bool((store == 255).all())  # (made use of)
    with torch.cuda.graph(graph, stream=side):
        logits = model.forward(batch, caches, fused=True, workspace=store)
    for _ in range(3):
        logits.fill_(float("nan"))
        store.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, eager)
        assert torch.equal(model.forward(batch, caches, fused=True), eager)
