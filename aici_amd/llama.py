"""A Llama-shaped engine step on top of the HIP kernels: the block order of
rllm/rllm-cuda/src/llm/llama.rs (attention :75-101, MLP :133-145, block :163-176,
model :201-213) followed by the AICI logit-mask + greedy step
(rllm-cuda/src/llm/tmodel.rs:277-283, 234-236).

The embedding is a library gather.  The projections of a step of at most 128 rows, and
the head of any step with at most that many sequences, go through the C ABI's linear
kernels: the weight is read once at the rate of the memory, silu_and_mul happens where the
gate and up products are finished, and so do the residual addition and, from 17 rows on, the
RMS norm that follow o_proj and down_proj; up to 4 rows are normalised by the projections
behind the norm.  Projections of more rows are library GEMMs
(torch on ROCm).
Projections with weights of 8 bits (`Fp8Weight`) go through the C ABI's linear_fp8, whatever
the rows.
Everything else -- rms_norm, rotary, the paged-KV attention composition,
silu_and_mul, bias + argmax -- goes through the C ABI as well.  Weights are random
(there are no checkpoints here): the harness measures and checks the step's
data path, not a language model.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import kernels
from .attn import RotaryEmbedding, varlen_attn, window_workspace_size
from .paged import BatchInfo


@dataclass
class LlamaConfig:
    """The fields of llama.rs:19-31 `LlamaConfig` that the forward pass reads."""
    hidden_size: int
    intermediate_size: int
    vocab_size: int
    num_hidden_layers: int
    num_attention_heads: int
    num_key_value_heads: int
    rms_norm_eps: float = 1e-5
    max_position_embeddings: int = 8192
    rope_theta: float = 10000.0
    dtype: torch.dtype = torch.bfloat16
    sliding_window: Optional[int] = None  # tokens a token sees, with itself (None: all), in every layer; no field of the reference's
    # The first tokens of a sequence, whose keys stay visible beside the window at the rotary positions they have in the sequence: neither counted
    # anew inside the cache nor a learned term of the softmax, which other models mean by sinks.
    attention_sinks: int = 0

    @property
    def head_dim(self) -> int:
        return self.hidden_size // self.num_attention_heads

    @staticmethod
    def llama3_8b(max_position_embeddings: int = 16640) -> "LlamaConfig":
        return LlamaConfig(4096, 14336, 128256, 32, 32, 8, 1e-5, max_position_embeddings, 500000.0, torch.bfloat16)


def random_weights(cfg: LlamaConfig, seed: int, device=None, std: float = 0.02) -> Dict[str, torch.Tensor]:
    """N(0, std^2) matrices and 1 + N(0, std^2) norm scales, rounded to cfg.dtype.  Names
    follow the checkpoint paths llama.rs loads (:103-118, :147-158, :178-192, :216-240).
    Without `device` everything is drawn on the CPU from one seeded generator (so a CPU
    check sees the same bits); with it, on the device."""
    g = torch.Generator(device=device if device is not None else "cpu").manual_seed(seed)
    H, I, V = cfg.hidden_size, cfg.intermediate_size, cfg.vocab_size
    qd = cfg.head_dim * cfg.num_attention_heads
    kvd = cfg.head_dim * cfg.num_key_value_heads

    def mat(rows: int, cols: int) -> torch.Tensor:
        w = torch.empty((rows, cols), dtype=cfg.dtype if device is not None else torch.float32, device=device)
        w.normal_(0.0, std, generator=g)
        return w.to(cfg.dtype)

    def scale(n: int) -> torch.Tensor:
        w = torch.empty((n,), dtype=torch.float32, device=device)
        w.normal_(0.0, std, generator=g)
        return (w + 1.0).to(cfg.dtype)

    ws = {"model.embed_tokens": mat(V, H), "model.norm": scale(H), "lm_head": mat(V, H)}
    for i in range(cfg.num_hidden_layers):
        p = f"model.layers.{i}."
        ws[p + "input_layernorm"] = scale(H)
        ws[p + "self_attn.q_proj"] = mat(qd, H)
        ws[p + "self_attn.k_proj"] = mat(kvd, H)
        ws[p + "self_attn.v_proj"] = mat(kvd, H)
        ws[p + "self_attn.o_proj"] = mat(H, qd)
        ws[p + "post_attention_layernorm"] = scale(H)
        ws[p + "mlp.gate_proj"] = mat(I, H)
        ws[p + "mlp.up_proj"] = mat(I, H)
        ws[p + "mlp.down_proj"] = mat(H, I)
    return ws


class Fp8Weight(NamedTuple):
    """A weight [N, K] in float8_e4m3fn with its f32 scales [ceil(N / 128), ceil(K / 128)], as `kernels.linear_fp8` takes it."""
    data: torch.Tensor
    scale: torch.Tensor


def _cat_rows(weights: Sequence[Union[torch.Tensor, Fp8Weight]]) -> Union[torch.Tensor, Fp8Weight]:
    """One weight of the rows of several."""
    if not any(isinstance(w, Fp8Weight) for w in weights):
        return torch.cat(list(weights))
    if not all(isinstance(w, Fp8Weight) for w in weights) or any(w.data.size(0) % 128 for w in weights[:-1]):
        raise ValueError("weights of 8 bits are joined with one another, and behind rows that are multiples of 128")
    return Fp8Weight(torch.cat([w.data for w in weights]), torch.cat([w.scale for w in weights]))


def _rows(t: torch.Tensor, idx: torch.Tensor) -> torch.Tensor:
    """t[idx]: index_select takes 32- and 64-bit indices as they are, others are converted."""
    return t.index_select(0, idx if idx.dtype in (torch.int32, torch.int64) else idx.long())


class Llama:
    """llama.rs:194-213.  `forward` returns the logits of every sequence's last token, of a batch of trees (`BatchInfo.with_trees`) those of every row.
    The projections' weights may be `Fp8Weight`s; with fp8 those that are not become such.  Embedding, norms and lm_head stay as they are."""

    def __init__(self, cfg: LlamaConfig, weights: Dict[str, Union[torch.Tensor, Fp8Weight]], device, fp8: bool = False):
        self.cfg = cfg
        self.device = device
        self.skinny_linear = True  # False: every projection is a library GEMM
        self.fused_norm = True     # False: the norm behind those projections is a launch of its own
        w = {k: Fp8Weight(v.data.to(device), v.scale.to(device)) if isinstance(v, Fp8Weight) else v.to(device) for k, v in weights.items()}
        self.wte = w["model.embed_tokens"]
        self.ln_f = w["model.norm"]
        self.lm_head = w["lm_head"]
        self.layers: List[Dict[str, torch.Tensor]] = []
        for i in range(cfg.num_hidden_layers):
            p = f"model.layers.{i}."
            self.layers.append({
                "rms_1": w[p + "input_layernorm"],
                # one GEMM for q, k, v and one for gate, up: rows concatenated
                "qkv": _cat_rows([w[p + "self_attn.q_proj"], w[p + "self_attn.k_proj"], w[p + "self_attn.v_proj"]]),
                "o": w[p + "self_attn.o_proj"],
                "rms_2": w[p + "post_attention_layernorm"],
                "gate_up": _cat_rows([w[p + "mlp.gate_proj"], w[p + "mlp.up_proj"]]),
                "down": w[p + "mlp.down_proj"],
            })
            if fp8:
                layer = self.layers[-1]
                for name in ("qkv", "o", "gate_up", "down"):
                    if not isinstance(layer[name], Fp8Weight):
                        layer[name] = Fp8Weight(*kernels.quantize_weight_fp8(layer[name]))
        self.rotary = RotaryEmbedding(cfg.head_dim, cfg.rope_theta, cfg.max_position_embeddings,
                                      cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim, cfg.dtype, device)

    def _rms(self, x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
        out = torch.empty_like(x)
        kernels.rms_norm(out, x, weight, self.cfg.rms_norm_eps)
        return out

    def _norm_in_proj(self, x: torch.Tensor, norm_weight: torch.Tensor, weight: Union[torch.Tensor, Fp8Weight]) -> bool:
        """Whether the projection normalises its rows itself, the same bits (us, 4096 columns, norm and projection / one launch: 6144
        rows 13.3 / 11.3 with one row of x, 13.5 / 13.3 with four; 28672 gated rows 38.6 / 37.7 with one, 38.4 / 39.4 with four, which in a
        step of eight layers comes out even: 915 / 915)."""
        return (not isinstance(weight, Fp8Weight) and x.size(0) <= kernels.RMS_NORM_LINEAR_MAX_ROWS and self.skinny_linear and self.fused_norm
                and kernels.rms_norm_linear_takes(x, norm_weight, weight))

    def _proj(self, x: torch.Tensor, weight: Union[torch.Tensor, Fp8Weight], fp8_workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x @ weight.T (llama.rs:81-83, 210).  A vocabulary's rows with more than 64 sequences stay with the library where the kernel reads
        them front to back (columns no multiple of 2048, rows none of 256), and with long rows from 97 sequences on.  us, library / C ABI:
        128256 x 4096 32 rows 197 / 161, 64 rows 209 / 176, 128 rows 233 / 219; 64 / 96 / 128 rows 65536 x 5120 118 / 115, 122 / 140, 126 / 150,
        65536 x 3072 77 / 70, 81 / 85, 84 / 91, 151936 x 4096 260 / 253, 268 / 287, 278 / 296, 131072 x 8192 0.91, 0.95, 1.05 of the library's.
        49 to 64 rows: 0.65 to 1.06 of it, 0.87 on average."""
        if isinstance(weight, Fp8Weight):
            return kernels.linear_fp8(x, weight.data, weight.scale, workspace=fp8_workspace)
        rows, (n, k) = x.size(0), weight.shape
        if self.skinny_linear and kernels.linear_takes(x, weight) and (
                rows <= 64 or n < 65536 or (n % 256 == 0 and k % 2048 == 0 and (k <= 4096 or (k <= 8192 and rows <= 96)))):
            return kernels.linear(x, weight)
        return x @ weight.t()

    def _gate_up_silu(self, h: torch.Tensor, weight: Union[torch.Tensor, Fp8Weight], fp8_workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """silu(h @ gate.T) * (h @ up.T) (llama.rs:135-142), weight = the gate rows and then the up rows."""
        if isinstance(weight, Fp8Weight):
            gu = kernels.linear_fp8(h, weight.data, weight.scale, workspace=fp8_workspace)
        elif self.skinny_linear and kernels.linear_takes(h, weight) and weight.size(0) % 32 == 0:
            return kernels.linear_silu_and_mul(h, weight)
        else:
            gu = h @ weight.t()
        act = torch.empty((h.size(0), gu.size(1) // 2), dtype=h.dtype, device=h.device)
        kernels.silu_and_mul(act, gu)
        return act

    def _proj_add_norm(self, y: torch.Tensor, weight: Union[torch.Tensor, Fp8Weight], x: torch.Tensor, norm_weight: torch.Tensor, behind=None,
                       fp8_workspace: Optional[torch.Tensor] = None):
        """x' = y @ weight.T + x (llama.rs:96 + 166, 143 + 173) and the RMS norm of x' that follows it (:169, :165 of the
        next block, :207), or None where the projection `behind` normalises its rows itself.  Few rows: the C ABI's kernel,
        which splits the inner dimension over the device and finishes the rows -- residual and norm -- in the launch that adds
        the parts up; else a library GEMM and one launch for the addition and the norm (742 x 4096: 6.3 us, two launches 5.4
        and 6.2).  The same bits either way as far as the norm goes."""
        if isinstance(weight, Fp8Weight):
            x = kernels.linear_fp8(y, weight.data, weight.scale, residual=x, workspace=fp8_workspace)
            if behind is not None and self._norm_in_proj(x, norm_weight, behind):
                return x, None
            return x, self._rms(x, norm_weight)
        if self.skinny_linear and weight.size(0) <= 8192 and kernels.linear_takes(y, weight):
            if behind is not None and self._norm_in_proj(x, norm_weight, behind):
                return kernels.linear(y, weight, residual=x), None
            if self.fused_norm:
                return kernels.linear_rms_norm(y, weight, norm_weight, self.cfg.rms_norm_eps, residual=x)
            x = kernels.linear(y, weight, residual=x)
            return x, self._rms(x, norm_weight)
        y = y @ weight.t()
        if kernels.add_rms_norm_takes(y, x, norm_weight):
            return y, kernels.add_rms_norm(y, x, norm_weight, self.cfg.rms_norm_eps)
        x = y + x
        return x, self._rms(x, norm_weight)

    def workspace_size(self, batch_info: BatchInfo) -> int:
        """Bytes of a workspace for `forward` of batches of these shapes: what attention with a window, or of trees, can make use of; 0 without either."""
        cfg = self.cfg
        if batch_info.tree_mask is not None:
            return kernels.paged_attention_tree_workspace_size(batch_info.q_multi, cfg.num_attention_heads, cfg.head_dim)
        if cfg.sliding_window is None:
            return 0
        return window_workspace_size(batch_info, cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim, cfg.dtype,
                                     cfg.sliding_window - 1, cfg.attention_sinks)

    def fp8_workspace_size(self, batch_info: BatchInfo) -> int:
        """Bytes of a workspace for what `forward` of batches of these shapes projects with weights of 8 bits; 0 without such weights."""
        rows = batch_info.tokens.numel()
        weights = {(rows, *w.data.shape): w for layer in self.layers for w in layer.values() if isinstance(w, Fp8Weight)}
        if isinstance(self.lm_head, Fp8Weight):
            weights[(batch_info.logit_idxs.numel(), *self.lm_head.data.shape)] = self.lm_head
        some = self.ln_f[:1]  # (of the projections' type; their rows' number is all that counts)
        return max((kernels.linear_fp8_workspace_size(some.expand(m, k), w.data) for (m, _, k), w in weights.items()), default=0)

    def forward(self, batch_info: BatchInfo, caches: List[Tuple[torch.Tensor, torch.Tensor]],
                paged_prefill: bool = False, fused: bool = False, workspace: Optional[torch.Tensor] = None,
                fp8_workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """batch_info on the device; caches[layer] = (key_cache, value_cache), updated in place.
        paged_prefill: multi-token rows read their context through block tables (no gather copy).
        fused: q, k, v stay views of the fused projection's output (the kernels honour the row stride) and
        rotary + cache scatter are one launch, or part of the projection's -- four or five launches fewer per layer, the same
        bits.
        workspace: uint8, `workspace_size` bytes, of a model with a window or a batch of trees: a captured step's attention is then the eager one and lies in no memory of the
        library's.  fp8_workspace: uint8, `fp8_workspace_size` bytes, on a 256-byte boundary, the same for the projections with weights of 8 bits, which
        need no eager call on the capture's stream then.  Without it, and for what has no workspace here (projections with weights of 16 bits, decode
        rows without a window), steps captured on one stream share that stream's scratch memory: their replays, and eager calls on that
        stream, must not overlap."""
        cfg = self.cfg
        Hq, Hkv, d = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
        window = {} if cfg.sliding_window is None else {"window_size_left": cfg.sliding_window - 1, "sink_tokens": cfg.attention_sinks}
        if cfg.sliding_window is not None or batch_info.tree_mask is not None:
            window["workspace"] = workspace
        x = _rows(self.wte, batch_info.tokens)                                   # llama.rs:203
        T = x.size(0)
        # h: the normalised rows, None where the projection that takes them does it
        first = self.layers[0]
        h = None if self._norm_in_proj(x, first["rms_1"], first["qkv"]) else self._rms(x, first["rms_1"])  # :165
        for li, (layer, (kc, vc)) in enumerate(zip(self.layers, caches)):
            # few rows: rotary and the cache writes happen in the projection's launch too (:85 + mod.rs:147-164)
            rotated = (fused and self.skinny_linear and not isinstance(layer["qkv"], Fp8Weight) and kc.dim() == 5 and kc.size(1) == Hkv
                       and kernels.qkv_linear_takes(x if h is None else h, layer["qkv"], self.rotary.cos_sin, kc, vc))
            if rotated:
                qkv = kernels.qkv_linear(*((x, layer["rms_1"]) if h is None else (h, None)), cfg.rms_norm_eps, layer["qkv"],
                                         batch_info.positions, self.rotary.cos_sin, kc, vc, batch_info.slot_mapping)
            elif h is None:
                qkv = kernels.rms_norm_linear(x, layer["rms_1"], cfg.rms_norm_eps, layer["qkv"])
            else:
                qkv = self._proj(h, layer["qkv"], fp8_workspace)                # :81-83
            if fused:
                q, k, v = qkv.split([Hq * d, Hkv * d, Hkv * d], dim=1)
                v = v.view(T, Hkv, d)
                if not rotated:
                    self.rotary.forward_and_cache(batch_info.positions, q, k, v, kc, vc, batch_info.slot_mapping)
                y = varlen_attn(q.view(T, Hq, d), k.view(T, Hkv, d), v, batch_info, kc, vc,
                                paged_prefill=paged_prefill, cached=True, **window)  # :93
            else:
                q, k, v = (t.contiguous() for t in qkv.split([Hq * d, Hkv * d, Hkv * d], dim=1))
                q, k = self.rotary.forward(batch_info.positions, q, k)          # :85 (in place on the copies)
                y = varlen_attn(q, k, v.reshape(T, Hkv, d), batch_info, kc, vc, paged_prefill=paged_prefill, **window)  # :93
            x, h = self._proj_add_norm(y, layer["o"], x, layer["rms_2"], layer["gate_up"], fp8_workspace)  # :96, :166, :169
            if h is None:
                act = kernels.rms_norm_linear(x, layer["rms_2"], cfg.rms_norm_eps, layer["gate_up"], silu_and_mul=True)
            else:
                act = self._gate_up_silu(h, layer["gate_up"], fp8_workspace)    # :135-142
            # the norm behind the block is the next block's first one, or the model's last (:165, :207)
            behind = self.layers[li + 1] if li + 1 < len(self.layers) else {"rms_1": self.ln_f, "qkv": None}
            x, h = self._proj_add_norm(act, layer["down"], x, behind["rms_1"], behind["qkv"], fp8_workspace)  # :143, :173
        x0 = h
        sel = _rows(x0, batch_info.logit_idxs)                                  # :209 extract_positions
        return self._proj(sel, self.lm_head, fp8_workspace)                     # :210


@dataclass
class Penalties:
    """What `kernels.penalize_logits` takes of a batch beside its logits."""
    history: torch.Tensor          # int32 [N]: every sequence's tokens, one after the other
    history_offsets: torch.Tensor  # int64 or int32 [S + 1]
    prompt_lens: Optional[torch.Tensor] = None  # int32 [S]
    repetition: Optional[torch.Tensor] = None   # f32 [S]
    frequency: Optional[torch.Tensor] = None    # f32 [S]
    presence: Optional[torch.Tensor] = None     # f32 [S]

    def apply(self, logits: torch.Tensor) -> torch.Tensor:
        return kernels.penalize_logits(logits, self.history, self.history_offsets, self.prompt_lens, self.repetition, self.frequency,
                                       self.presence)


def aici_greedy(logits: torch.Tensor, allow_masks: torch.Tensor, penalties: Optional[Penalties] = None) -> torch.Tensor:
    """The sampling half of a constrained step: every sequence's packed allow-mask (u8
    [S, 4*ceil(V/32)], bit k of byte i <-> token 8i+k; aicirt/src/api.rs:278-292) is applied
    as a 0/-inf bias and the arg-max taken (tmodel.rs:277-283, 234-236), all rows in one
    launch and without materialising f32 bias rows; `penalties` go first, in a launch of their own.  Returns int32 [S]."""
    if penalties is not None:
        logits = penalties.apply(logits)
    return kernels.bias_argmax(logits, mask=allow_masks)


def aici_sample(logits: torch.Tensor, allow_masks: torch.Tensor, temperature: torch.Tensor, top_p: torch.Tensor,
                uniforms: torch.Tensor = None, generator: torch.Generator = None,
                penalties: Optional[Penalties] = None) -> torch.Tensor:
    """The sampling half with temperature and top-p (tmodel.rs:172-194, 236-268) under the same packed
    allow-masks: rows with temperature < 1e-5 are greedy, the others are drawn with one uniform number per
    row in [0, 1) -- the caller's, or drawn here from `generator` (a seeded torch.Generator on the CPU stands
    in for the reference's per-sequence `StdRng`: the same seed gives the same tokens).  All rows in one
    call, no host round trip; `penalties` go first.  Returns int32 [S]."""
    if penalties is not None:
        logits = penalties.apply(logits)
    if uniforms is None:
        uniforms = torch.rand((logits.size(0),), generator=generator, dtype=torch.float32).to(logits.device)
    return kernels.bias_sample(logits, temperature, top_p, uniforms, mask=allow_masks)
