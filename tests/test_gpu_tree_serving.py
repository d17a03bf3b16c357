"""A small model that generates by verifying trees of drafted tokens: prompts as chunks, then steps whose trees are made of the model's own
continuation and of guesses, in blocks of the host's allocator; logits, the kept rows and the caches against restatements.  And the same steps on
weights of 8 bits.

Tolerance of the logits against the 64-bit model: 2 layers of 10 tensors that are rounded to fp16 and 3 more, half a step each (2^-11 of their norm),
no map between them taken to stretch a relative error more than twofold: 23 x 2 x 2^-11 = 0.0225 of the logits' norm."""
import random

import pytest
import torch

from aici_amd import kernels as K
from aici_amd import llama, paged
from oracle import trees

from test_gpu_window_serving import CFG, TOLERANCE, reference

pytestmark = pytest.mark.gpu
BS = 16


class Server:
    """Requests, their tokens and blocks; row 0 of a step's tree is the newest token, which the cache does not hold yet."""

    def __init__(self, model, device, blocks=60):
        self.model, self.device, self.alloc = model, device, paged.BlockAllocator(BS, blocks)
        self.caches = [paged.alloc_gpu_cache_layer(blocks, CFG.num_key_value_heads, CFG.head_dim, BS, CFG.dtype, device) for _ in range(2)]
        for kc, vc in self.caches:
            kc.fill_(float("nan"))
            vc.fill_(float("nan"))
        self.list = K.CacheList([k for k, _ in self.caches], [v for _, v in self.caches])
        self.said = {}

    def batch(self, parts):
        """parts: (request, all its tokens with the new ones, tokens in the cache)."""
        builder = paged.BatchInfoBuilder(BS, 4096, 1)
        for sid, tokens, computed in parts:
            if computed == 0:
                self.alloc.alloc_seq(sid, len(tokens))
            else:
                assert not self.alloc.append_slots(sid, computed, len(tokens))
            builder.sched_out(self.alloc, sid, tokens, computed)
        return builder.finish().to(self.device)

    def prompts(self, prompts):
        batch = self.batch([(sid, tokens, 0) for sid, tokens in prompts.items()])
        logits = self.model.forward(batch, self.caches, paged_prefill=True, fused=True)
        for sid, row in zip(batch.seq_ids, range(len(prompts))):
            self.said[sid] = prompts[sid] + [int(logits[row].argmax())]
        return logits

    def step(self, drafts, **forward):
        """drafts: request -> (drafted tokens, parents counted from the newest token).  Trees of one row come last, as the batch's decode rows."""
        order = sorted(drafts, key=lambda sid: len(drafts[sid][0]) == 0)
        batch = self.batch([(sid, self.said[sid] + drafts[sid][0], len(self.said[sid]) - 1) for sid in order])
        parents = [p for sid in order if drafts[sid][0] for p in [-1] + drafts[sid][1]]
        rows = {sid: 1 + len(drafts[sid][0]) for sid in order}
        batch = batch.with_trees(torch.tensor(parents, dtype=torch.int32, device=self.device))
        logits = self.model.forward(batch, self.caches, **forward)
        chosen = greedy(logits)
        multi = batch.q_multi
        kept = K.tree_accept(batch.tokens[:multi], torch.tensor(parents, dtype=torch.int32, device=self.device), chosen[:multi], batch.seqlens_q,
                             batch.max_seqlen_q, batch.slot_mapping[:multi], self.list)
        at, out = 0, {}
        for i, sid in enumerate(order):
            n = rows[sid]
            if drafts[sid][0]:
                path = [r for r in kept.path[i].tolist() if r >= 0]
                following = int(kept.next_tokens[i])
                assert len(path) == int(kept.lens[i])
            else:
                path, following = [0], int(chosen[at])
            tree = [self.said[sid][-1]] + drafts[sid][0]
            before = self.said[sid][:-1]
            out[sid] = (before, tree, [-1] + drafts[sid][1], logits[at:at + n], chosen[at:at + n].tolist(), path, following)
            self.said[sid] = before + [tree[r] for r in path] + [following]
            self.alloc.trim(sid, len(before) + len(path))
            at += n
        return batch, out


def greedy(logits):
    """Every row's token, with nothing barred."""
    return llama.aici_greedy(logits, torch.full((logits.size(0), 4 * -(-CFG.vocab_size // 32)), 255, dtype=torch.uint8, device=logits.device))


def guesses(rng, n, truth):
    """A tree of n drafts: `truth` as far as it goes along one branch, and guesses around it."""
    tokens, parents, tip = [], [], 0
    for i in range(n):
        if truth and rng.random() < 0.5:
            tokens.append(truth.pop(0))
            parents.append(tip)
            tip = i + 1
        else:
            tokens.append(rng.randrange(CFG.vocab_size))
            parents.append(rng.randrange(i + 1))
    return tokens, parents


@pytest.mark.parametrize("fused", [False, True])
def test_generation_by_trees(device, fused):
    weights = llama.random_weights(CFG, 3, std=0.05)
    server = Server(llama.Llama(CFG, weights, device), device)
    table, rng = server.model.rotary.cos_sin, random.Random(5)
    server.prompts({7: [rng.randrange(1000) for _ in range(37)], 8: [rng.randrange(1000) for _ in range(5)], 9: [rng.randrange(1000) for _ in range(64)]})

    def truth(sid, n):
        """The next tokens by the 64-bit model."""
        tokens = list(server.said[sid])
        for _ in range(n):
            tokens.append(int(reference(weights, table, tokens, device, None, 0).argmax()))
        return tokens[len(server.said[sid]):]

    free = server.alloc.get_num_free_blocks()
    kept = 0
    for k in range(6):
        drafts = {sid: guesses(rng, 0 if (sid + k) % 5 == 0 else rng.randint(1, 30), truth(sid, 5)) for sid in (7, 8, 9)}
        _, out = server.step(drafts, fused=fused)
        for sid, (before, tree, parents, logits, chosen, path, following) in out.items():
            for row in range(len(tree)):
                family = trees.family(parents, row)[::-1]
                ref = reference(weights, table, before + [tree[r] for r in family], device, None, 0)
                err = float((logits[row].double() - ref).norm() / ref.norm())
                assert err <= TOLERANCE, (k, sid, row, err)
                assert chosen[row] == int(logits[row].argmax())
            assert [(path, following)] == trees.accept(tree, parents, chosen, [0, len(tree)], len(tree))
            kept += len(path) - 1
    assert kept >= 10  # (drafts along the model's own continuation have been kept)
    # what was not kept has gone back: blocks for the tokens in the cache alone
    held = sum(-(-(len(t) - 1) // BS) for t in server.said.values())
    assert server.alloc.get_num_free_blocks() == 60 - held and free > 0


def test_generation_by_trees_on_8_bit_weights(device):
    """The same with weights of 8 bits: the forward pass is the composition of its calls, bit for bit, and the moved caches give the bits of caches
    that hold the kept tokens from the start."""
    cfg = CFG
    weights = llama.random_weights(cfg, 4, std=0.05)
    model = llama.Llama(cfg, weights, device, fp8=True)
    assert all(isinstance(layer[n], llama.Fp8Weight) for layer in model.layers for n in ("qkv", "o", "gate_up", "down"))
    server, rng = Server(model, device), random.Random(6)
    server.prompts({1: [rng.randrange(1000) for _ in range(33)], 2: [rng.randrange(1000) for _ in range(70)]})
    kept = 0
    for k in range(6):
        drafts = {}
        for sid in (1, 2):
            # the model's own continuation, from a step of one row each on a copy of the cache
            drafts[sid] = guesses(rng, rng.randint(2, 20), continuation(server, sid, 4))
        image = [(kc.clone(), vc.clone()) for kc, vc in server.caches]
        batch, out = server.step(drafts, fused=k % 2 == 0)
        for (kc, vc), (ik, iv) in zip(server.caches, image):
            assert not torch.equal(torch.nan_to_num(kc), torch.nan_to_num(ik))
        logits = composed(model, batch, image)
        got = torch.cat([out[sid][3] for sid in sorted(out, key=lambda s: batch.seq_ids.index(s))])
        assert torch.equal(logits, got)
        # the kept rows' keys and values, moved by hand
        cu, slots = batch.seqlens_q.tolist(), batch.slot_mapping.tolist()
        for i, sid in enumerate(batch.seq_ids):
            path = out[sid][5]
            kept += len(path) - 1
            for kc, vc in image:
                src = torch.tensor([slots[cu[i] + r] for r in path], device=device)
                dst = torch.tensor([slots[cu[i] + j] for j in range(len(path))], device=device)
                k_rows, v_rows = kc[src // BS, :, :, src % BS].clone(), vc[src // BS, :, :, src % BS].clone()
                kc[dst // BS, :, :, dst % BS] = k_rows
                vc[dst // BS, :, :, dst % BS] = v_rows
        for (kc, vc), (ik, iv) in zip(server.caches, image):
            assert torch.equal(torch.nan_to_num(kc), torch.nan_to_num(ik)) and torch.equal(torch.nan_to_num(vc), torch.nan_to_num(iv))
    assert kept >= 4


def continuation(server, sid, n):
    """The model's next n tokens after what a request has said, on copies of the caches and with blocks that go back."""
    image = [(kc.clone(), vc.clone()) for kc, vc in server.caches]
    tokens = list(server.said[sid])
    first = len(tokens)
    for _ in range(n):
        batch = server.batch([(sid, tokens, len(tokens) - 1)])
        tokens.append(int(server.model.forward(batch, image, fused=True)[0].argmax()))
    server.alloc.trim(sid, first - 1)
    return tokens[first:]


def composed(model, batch, caches):
    """The forward pass of a batch of trees by calls of its own."""
    cfg = model.cfg
    hq, hkv, d = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
    x = model.wte[batch.tokens.long()]
    n = x.size(0)

    def norm(x, w):
        out = torch.empty_like(x)
        K.rms_norm(out, x, w, cfg.rms_norm_eps)
        return out

    for layer, (kc, vc) in zip(model.layers, caches):
        q, k, v = K.linear_fp8(norm(x, layer["rms_1"]), *layer["qkv"]).split([hq * d, hkv * d, hkv * d], 1)
        q, k, v = q.contiguous(), k.contiguous(), v.reshape(n, hkv, d)
        K.rotary_embedding(batch.positions, q, k, d, model.rotary.cos_sin, True)
        K.reshape_and_cache(k.view(n, hkv, d), v, kc, vc, batch.slot_mapping)
        y = K.paged_attention_tree(q.view(n, hq, d), kc, vc, batch.multi_block_tables, batch.seqlens_q, batch.multi_context_lens, batch.max_seqlen_q,
                                   batch.max_seqlen_k, d ** -0.5, batch.tree_mask)
        x = K.linear_fp8(y.view(n, hq * d), *layer["o"], residual=x)
        gate_up = K.linear_fp8(norm(x, layer["rms_2"]), *layer["gate_up"])
        act = torch.empty((n, gate_up.size(1) // 2), dtype=x.dtype, device=x.device)
        K.silu_and_mul(act, gate_up)
        x = K.linear_fp8(act, *layer["down"], residual=x)
    x = norm(x, model.ln_f)[batch.logit_idxs.long()]
    return K.linear(x, model.lm_head) if K.linear_takes(x, model.lm_head) else x @ model.lm_head.t()


def test_captured_tree_step(device):
    """A step of trees captured with a workspace and replayed has the eager step's bits, the acceptance and the move of the caches with it."""
    model = llama.Llama(CFG, llama.random_weights(CFG, 5, std=0.05), device, fp8=True)
    server, rng = Server(model, device), random.Random(7)
    server.prompts({1: [rng.randrange(1000) for _ in range(50)], 2: [rng.randrange(1000) for _ in range(20)]})
    batch = server.batch([(sid, server.said[sid] + [rng.randrange(1000) for _ in range(9)], len(server.said[sid]) - 1) for sid in (1, 2)])
    parents = torch.tensor([-1, 0, 0, 1, 1, 2, 3, 3, 6, 8] * 2, dtype=torch.int32, device=device)
    plain = model.workspace_size(batch)
    batch = batch.with_trees(parents)
    need = model.workspace_size(batch)
    assert plain == 0 and need > 0
    store = torch.empty((need,), dtype=torch.uint8, device=device)
    image = [(kc.clone(), vc.clone()) for kc, vc in server.caches]

    def step():
        rows = batch.with_trees(parents)
        logits = model.forward(rows, server.caches, fused=True, workspace=store)
        chosen = greedy(logits)
        return logits, K.tree_accept(rows.tokens, parents, chosen, rows.seqlens_q, rows.max_seqlen_q, rows.slot_mapping, server.list)

    def restore():
        for (kc, vc), (ik, iv) in zip(server.caches, image):
            kc.copy_(ik)
            vc.copy_(iv)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        want = step()
        after = [(kc.clone(), vc.clone()) for kc, vc in server.caches]
    torch.cuda.synchronize()
    restore()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for _ in range(3):
        restore()
        got[0].fill_(float("nan"))
        for t in got[1]:
            t.fill_(-9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
        for (kc, vc), (ak, av) in zip(server.caches, after):
            assert torch.equal(torch.nan_to_num(kc), torch.nan_to_num(ak)) and torch.equal(torch.nan_to_num(vc), torch.nan_to_num(av))


def test_weights_of_8_bits_are_joined(device):
    """Weights that come in 8 bits already, where their rows fill blocks of scales; else a refusal.  A window and trees do not go together."""
    cfg = llama.LlamaConfig(1024, 512, 1000, 1, 8, 2, 1e-5, 512, 10000.0, torch.bfloat16)
    weights = llama.random_weights(cfg, 8, std=0.05)
    eights = {k: llama.Fp8Weight(*K.quantize_weight_fp8(v)) if "_proj" in k else v for k, v in weights.items()}
    model, same = llama.Llama(cfg, eights, device), llama.Llama(cfg, weights, device, fp8=True)
    for n in ("qkv", "o", "gate_up", "down"):
        a, b = model.layers[0][n], same.layers[0][n]
        assert torch.equal(a.data.view(torch.uint8), b.data.view(torch.uint8)) and torch.equal(a.scale, b.scale)
    mixed = dict(eights)
    mixed["model.layers.0.self_attn.k_proj"] = weights["model.layers.0.self_attn.k_proj"]
    with pytest.raises(ValueError, match="weights of 8 bits are joined"):
        llama.Llama(cfg, mixed, device)
    server = Server(llama.Llama(CFG, llama.random_weights(CFG, 5), device), device)
    batch = server.batch([(1, [1, 2, 3], 0)])
    batch = batch.with_trees(torch.tensor([-1, 0, 0], dtype=torch.int32, device=device))
    from aici_amd.attn import varlen_attn
    q = torch.zeros((3, 8, 64), dtype=torch.float16, device=device)
    with pytest.raises(ValueError, match="no window"):
        varlen_attn(q, q[:, :2], q[:, :2], batch, *server.caches[0], window_size_left=5)
    none = paged.BatchInfoBuilder(BS, 4096, 1)
    none.sched_out(server.alloc, 1, [1, 2, 3], 2)
    with pytest.raises(ValueError, match="the batch has none"):
        none.finish().to(device).with_trees(torch.zeros((0,), dtype=torch.int32, device=device))
