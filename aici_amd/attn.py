"""The attention layer pieces of rLLM's `llm` module
(rllm/rllm-cuda/src/llm/mod.rs) on top of the HIP kernels: `RotaryEmbedding`
(mod.rs:24-129), `varlen_attn` (mod.rs:318-354) and `RmsNorm` (mod.rs:367-399).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import numpy as np
import torch

from . import kernels
from .kernels import _native
from .paged import BatchInfo


class RotaryEmbedding:
    """cos/sin table built as mod.rs:41-60 does, applied in place by the HIP kernel."""

    def __init__(self, rotary_dim: int, rope_theta: float, max_sequence_length: int, num_attention_heads: int,
                 num_key_value_heads: int, head_dim: int, dtype: torch.dtype, device):
        self.num_attention_heads = num_attention_heads
        self.num_key_value_heads = num_key_value_heads
        self.head_dim = head_dim
        self.cos_sin = self.build_table(rotary_dim, rope_theta, max_sequence_length, dtype).to(device)

    @staticmethod
    def build_table(rotary_dim: int, rope_theta: float, max_len: int, dtype: torch.dtype) -> torch.Tensor:
        # theta_i = 1 / rope_theta^(i / rotary_dim), i even, in f32 (mod.rs:44-47)
        expo = np.arange(0, rotary_dim, 2, dtype=np.float32) / np.float32(rotary_dim)
        theta = torch.from_numpy(np.float32(1.0) / np.power(np.float32(rope_theta), expo, dtype=np.float32))
        idx_theta = torch.arange(max_len, dtype=torch.float32).reshape(max_len, 1).matmul(theta.reshape(1, -1))
        return torch.cat([idx_theta.cos().to(dtype), idx_theta.sin().to(dtype)], dim=-1).contiguous()

    def forward_and_cache(self, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                          key_cache: torch.Tensor, value_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
        """forward() and the scatter of the rotated keys and of v [T, Hkv, d] into the cache, in one launch;
        q [T, Hq*d] and k [T, Hkv*d] (row strides allowed) are rotated in place."""
        kernels.rotary_embedding_and_cache(positions, q, k, v, self.head_dim, self.cos_sin, True, key_cache,
                                           value_cache, slot_mapping)

    def forward(self, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        q = q.reshape(-1, self.num_attention_heads * self.head_dim)
        k = k.reshape(-1, self.num_key_value_heads * self.head_dim)
        num_tokens = q.size(0)
        assert num_tokens == k.size(0)
        kernels.rotary_embedding(positions, q, k, self.head_dim, self.cos_sin, True)
        return (q.reshape(num_tokens, self.num_attention_heads, self.head_dim),
                k.reshape(num_tokens, self.num_key_value_heads, self.head_dim))


class RmsNorm:
    """mod.rs:367-399; the reference leaves `// TODO use kernels::rms_norm`, this does."""

    def __init__(self, weight: torch.Tensor, eps: float = 1e-5):
        self.scale = weight
        self.eps = eps

    def forward(self, xs: torch.Tensor) -> torch.Tensor:
        out = torch.empty_like(xs)
        kernels.rms_norm(out, xs, self.scale, self.eps)
        return out


def _reads_through_tables(q: torch.Tensor, k: torch.Tensor, batch_info: BatchInfo, key_cache: torch.Tensor, value_cache: torch.Tensor) -> bool:
    """Whether the context of the multi-token rows need not be gathered (us, gathered / through the tables, 32 heads of 80: 120 decode rows
    of 1k..8k tokens beside 4 x 512 new ones over up to 3072 1012 / 920, 15 rows of 253 beside 4 x 65..263 103 / 39).  What the tables' route
    would not take, or would not refuse as the gather does (caches with other heads than k), is gathered."""
    tables, lens = batch_info.multi_block_tables, batch_info.multi_context_lens
    return (batch_info.q_multi > 0 and tables is not None and lens is not None and tables.size(1) * 16 >= batch_info.max_seqlen_k
            and tables.dtype == lens.dtype == torch.int32 and tables.size(0) == lens.size(0) == batch_info.seqlens_q.size(0) - 1
            and (tables.size(1) <= 1 or tables.stride(1) == 1) and lens.is_contiguous() and q.size(2) in (64, 80, 96, 112, 128)
            and q.dtype in (torch.float16, torch.bfloat16) and key_cache.dtype == q.dtype and value_cache.dtype == q.dtype
            and key_cache.dim() == 5 and value_cache.dim() == 4 and key_cache.size(3) == 16 and value_cache.size(3) == 16
            and key_cache.size(1) == k.size(1) and key_cache.is_contiguous() and value_cache.is_contiguous()
            and key_cache.data_ptr() % 16 == 0 and value_cache.data_ptr() % 16 == 0)


def window_workspace_size(batch_info: BatchInfo, num_heads: int, num_kv_heads: int, head_size: int, dtype: torch.dtype,
                          window_size_left: int, sink_tokens: int = 0) -> int:
    """Bytes of scratch memory `varlen_attn` with a window can make use of for batches of these shapes."""
    single = batch_info.tokens.numel() - batch_info.q_multi
    need = kernels.flash_attn_varlen_paged_window_workspace_size(batch_info.q_multi, num_heads, head_size)
    if single > 0:
        need = max(need, kernels.paged_attention_window_workspace_size(single, num_heads, num_kv_heads, head_size, batch_info.paged_block_size,
                                                                       batch_info.paged_max_context_len, window_size_left, sink_tokens, dtype))
    return need


def varlen_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch_info: BatchInfo, key_cache: torch.Tensor,
                value_cache: torch.Tensor, softmax_scale: Optional[float] = None,
                paged_prefill: bool = False, cached: bool = False, window_size_left: Optional[int] = None,
                sink_tokens: int = 0, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """mod.rs:318-354: q [T,Hq,d], k/v [T,Hkv,d] -> [T, Hq*d].  `cached`: the new K/V are in the cache
    already (kernels.rotary_embedding_and_cache) and the scatter is skipped.

    batch_info must already live on the GPU.  The whole composition (scatter,
    varlen prefill rows, paged decode rows) is one C-ABI call.  The multi-token
    rows read their context from the cache through block tables, or, where the
    caches are not what that takes, from a gathered copy; with `paged_prefill`
    always through the tables (needs the builder's multi_block_tables).

    window_size_left: a token sees that many tokens before it, itself and the first sink_tokens of its sequence
    (None: all of them); multi-token rows then always read through the tables.  workspace (with a window): uint8,
    `window_workspace_size` bytes, so that a captured step gives the eager step's bits and shares no scratch memory with other graphs; None: what
    the library keeps per stream, and under capture chunks whose keys are not dealt out."""
    T, Hq, d = q.shape
    Hkv = k.size(1)
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(d)
    y = torch.empty((T, Hq, d), dtype=q.dtype, device=q.device)
    if window_size_left is not None:
        has_m, has_p = batch_info.q_multi > 0, batch_info.q_multi < T
        if has_m and batch_info.multi_block_tables is None:
            raise ValueError("a window needs batch_info.multi_block_tables (slots must follow the blocks in order)")
        _native.varlen_attn_paged_window_ws(q, k, v, key_cache, value_cache, None if cached else batch_info.slot_mapping,
                                            batch_info.multi_block_tables if has_m else None, batch_info.seqlens_q if has_m else None,
                                            batch_info.multi_context_lens if has_m else None, batch_info.q_multi, batch_info.max_seqlen_q,
                                            batch_info.max_seqlen_k, batch_info.paged_block_tables if has_p else None,
                                            batch_info.paged_context_lens if has_p else None, batch_info.paged_block_size,
                                            batch_info.paged_max_context_len, softmax_scale, window_size_left, sink_tokens, y, workspace)
        return y.reshape(T, Hq * d)
    if sink_tokens != 0 or workspace is not None:
        raise ValueError(f"{'sink_tokens' if sink_tokens != 0 else 'workspace'} needs a window")
    if paged_prefill or _reads_through_tables(q, k, batch_info, key_cache, value_cache):
        if batch_info.multi_block_tables is None:
            raise ValueError("paged_prefill needs batch_info.multi_block_tables (slots must follow the blocks in order)")
        has_m, has_p = batch_info.q_multi > 0, batch_info.q_multi < T
        _native.varlen_attn_paged(q, k, v, key_cache, value_cache, None if cached else batch_info.slot_mapping,
                                  batch_info.multi_block_tables if has_m else None,
                                  batch_info.seqlens_q if has_m else None,
                                  batch_info.multi_context_lens if has_m else None, batch_info.q_multi,
                                  batch_info.max_seqlen_q, batch_info.max_seqlen_k,
                                  batch_info.paged_block_tables if has_p else None,
                                  batch_info.paged_context_lens if has_p else None,
                                  batch_info.paged_block_size, batch_info.paged_max_context_len, softmax_scale, y)
        return y.reshape(T, Hq * d)
    G = batch_info.gather_mapping.numel()
    gk = torch.empty((G, Hkv, d), dtype=q.dtype, device=q.device) if G else None
    gv = torch.empty_like(gk) if G else None
    has_multi = batch_info.q_multi > 0
    has_paged = batch_info.q_multi < T
    _native.varlen_attn(q, k, v, key_cache, value_cache, None if cached else batch_info.slot_mapping,
                        batch_info.gather_mapping if has_multi else None, batch_info.seqlens_q if has_multi else None,
                        batch_info.seqlens_k if has_multi else None, batch_info.q_multi, batch_info.max_seqlen_q,
                        batch_info.max_seqlen_k, batch_info.paged_block_tables if has_paged else None,
                        batch_info.paged_context_lens if has_paged else None, batch_info.paged_block_size,
                        batch_info.paged_max_context_len, softmax_scale, gk, gv, y)
    return y.reshape(T, Hq * d)
