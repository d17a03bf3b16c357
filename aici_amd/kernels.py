"""Host-side mirror of rLLM's `tch_cuda` kernel API (rllm/tch-cuda/src/lib.rs),
taking torch tensors that live on the GPU and calling the C ABI of libhipattn.

Function names, argument order and meaning follow the reference's safe
wrappers so the parity tests read like calls into `tch_cuda`.  PyTorch is used
only for device memory and the current stream; all computation happens in the
HIP kernels behind the C ABI.  There is no CPU implementation here: tensors on
the CPU are rejected.
"""
from __future__ import annotations

import ctypes
from typing import Dict, List, NamedTuple, Optional, Sequence

import torch

from . import _lib
from ._lib import HipAttnError, Tensor, call

try:
    from . import _native  # the hot entry points, bound without ctypes (csrc/bind/native.cpp)
except ImportError as e:
    raise ImportError("aici_amd/_native.so is missing or was built for another torch: run `python -m aici_amd.build`") from e

_DTYPES = {
    torch.float32: _lib.F32,
    torch.float16: _lib.F16,
    torch.bfloat16: _lib.BF16,
    torch.int32: _lib.I32,
    torch.int64: _lib.I64,
    torch.uint8: _lib.U8,
    torch.float8_e4m3fn: _lib.E4M3,
}


def _desc(t: Optional[torch.Tensor], name: str = "tensor", device: bool = True):
    """`hipattn_tensor` view of a torch tensor (None -> NULL)."""
    if t is None:
        return None
    if t.dtype not in _DTYPES:
        raise HipAttnError(f"{name}: unsupported dtype {t.dtype}")
    if device and not t.is_cuda:
        raise HipAttnError(f"{name}: expected a GPU tensor, got one on {t.device}")
    if t.dim() > _lib.MAX_DIMS:
        raise HipAttnError(f"{name}: at most {_lib.MAX_DIMS} dims")
    d = Tensor()
    d.data = t.data_ptr()
    d.dtype = _DTYPES[t.dtype]
    d.ndim = t.dim()
    for i in range(t.dim()):
        d.sizes[i] = t.size(i)
        d.strides[i] = t.stride(i)
    return ctypes.pointer(d)


def _stream(ref: torch.Tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(ref.device).cuda_stream)


# --------------------------------------------------------------------------- attention

def flash_attn_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seqlens_q: torch.Tensor,
                      seqlens_k: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int, softmax_scale: float,
                      causal: bool, *, return_lse: bool = False, seqused_k: Optional[torch.Tensor] = None,
                      window=(-1, -1), out_dtype: Optional[torch.dtype] = None):
    """lib.rs:69-104.  q [total_q, Hq, d], k/v [total_k, Hkv, d]; returns [total_q, Hq, d].
    window = (left, right) of mha_varlen_fwd_C (flash_api.cpp:635-636); rLLM always passes (-1, -1).
    out_dtype=torch.float32 asks for the output before its rounding to q's dtype."""
    out = torch.empty((q.size(0), q.size(1), q.size(2)), dtype=out_dtype or q.dtype, device=q.device)
    lse = None
    if return_lse:
        lse = torch.empty((seqlens_q.numel() - 1, q.size(1), max_seqlen_q), dtype=torch.float32, device=q.device)
    _native.mha_varlen_fwd(q, k, v, seqlens_q, seqlens_k, seqused_k, max_seqlen_q, max_seqlen_k, 0.0, softmax_scale,
                           False, causal, window[0], window[1], out, lse)
    return (out, lse) if return_lse else out


varlen_attn = flash_attn_varlen  # rllm-cuda/src/llm/kernels.rs:4-5


def flash_attn_varlen_paged(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                            block_tables: torch.Tensor, seqlens_q: torch.Tensor, context_lens: torch.Tensor,
                            max_seqlen_q: int, max_seqlen_k: int, softmax_scale: float, causal: bool = True,
                            return_lse: bool = False, out_dtype: Optional[torch.dtype] = None):
    """Varlen prefill whose K/V come from the paged cache through block tables -- what
    llm/mod.rs:181-238 builds from gather_cached_kv + repeat_kv + flash_attn_varlen, without the
    copies.  q [Tq,Hq,d]; block_tables int32 [b,cols]; seqlens_q int32 offsets [b+1]; context_lens
    int32 [b] (keys per sequence, the new tokens already scattered into the cache)."""
    out = torch.empty_like(q, dtype=out_dtype or q.dtype)
    lse = None
    if return_lse:
        lse = torch.empty((context_lens.numel(), q.size(1), max(int(max_seqlen_q), 1)), dtype=torch.float32,
                          device=q.device)
    _native.mha_varlen_fwd_paged(q, key_cache, value_cache, block_tables, seqlens_q, context_lens, max_seqlen_q,
                                 max_seqlen_k, softmax_scale, causal, out, lse)
    return (out, lse) if return_lse else out


def flash_attn_varlen_paged_window(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
                                   seqlens_q: torch.Tensor, context_lens: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int,
                                   softmax_scale: float, window_size_left: int, sink_tokens: int = 0, return_lse: bool = False,
                                   out_dtype: Optional[torch.dtype] = None, workspace: Optional[torch.Tensor] = None):
    """`flash_attn_varlen_paged`, causal, with a sliding window and sinks: the query at position p of its sequence sees key j iff j <= p
    and (j >= p - window_size_left or j < sink_tokens).  Blocks of keys that none of a sequence's new tokens sees may be gone.
    workspace: uint8, `flash_attn_varlen_paged_window_workspace_size` bytes, for calls that are captured and for those that must not
    allocate; None: a buffer that the library keeps per stream, and under capture none, which takes longer for few rows over long windows."""
    out = torch.empty_like(q, dtype=out_dtype or q.dtype)
    lse = None
    if return_lse:
        lse = torch.empty((context_lens.numel(), q.size(1), max(int(max_seqlen_q), 1)), dtype=torch.float32, device=q.device)
    _native.mha_varlen_fwd_paged_window(q, key_cache, value_cache, block_tables, seqlens_q, context_lens, max_seqlen_q, max_seqlen_k,
                                        softmax_scale, window_size_left, sink_tokens, out, lse, workspace)
    return (out, lse) if return_lse else out


def flash_attn_varlen_paged_window_workspace_size(total_q: int, num_heads: int, head_size: int) -> int:
    """Bytes of scratch memory flash_attn_varlen_paged_window can make use of for total_q rows."""
    n = ctypes.c_int64(0)
    call("hipattn_mha_varlen_fwd_paged_window_workspace_size", int(total_q), int(num_heads), int(head_size), ctypes.byref(n))
    return int(n.value)


def paged_attention_tree(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
                         seqlens_q: torch.Tensor, context_lens: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int, softmax_scale: float,
                         tree_mask: torch.Tensor, out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of trees of drafted tokens over the paged cache.  q [Tq,Hq,d], block_tables, seqlens_q and context_lens as for
    `flash_attn_varlen_paged` (the rows' own keys are the last of the context); a row sees every key in front of its tree and, of the tree's
    keys, those that tree_mask int64 [Tq, words] names: bit j % 64 of word j / 64 for the sequence's j-th row (`tree_rows`).  A row that sees
    nothing is zero.  out may be q.  workspace: uint8, `paged_attention_tree_workspace_size` bytes, for calls that are captured and for those that must not
    allocate; None: a buffer that the library keeps per stream, and under capture none, which takes longer for few long contexts."""
    if out is None:
        out = torch.empty_like(q)
    _native.paged_attention_tree(q, key_cache, value_cache, block_tables, seqlens_q, context_lens, max_seqlen_q, max_seqlen_k, softmax_scale,
                                 tree_mask, out, workspace)
    return out


def paged_attention_tree_workspace_size(total_q: int, num_heads: int, head_size: int) -> int:
    """Bytes of scratch memory paged_attention_tree can make use of for total_q rows."""
    n = ctypes.c_int64(0)
    call("hipattn_paged_attention_tree_workspace_size", int(total_q), int(num_heads), int(head_size), ctypes.byref(n))
    return int(n.value)


def paged_attention_window(out: torch.Tensor, query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                           num_kv_heads: int, scale: float, block_tables: torch.Tensor, context_lens: torch.Tensor, block_size: int,
                           max_context_len: int, window_size_left: int, sink_tokens: int = 0,
                           alibi_slopes: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> None:
    """`paged_attention_v1` with a sliding window and sinks: the token of a sequence of ctx tokens sees key t iff
    t >= ctx - 1 - window_size_left or t < sink_tokens.  Blocks between the two may be gone.  workspace: uint8,
    `paged_attention_window_workspace_size` bytes; None: a buffer that the library keeps per stream."""
    _native.paged_attention_window(out, query, key_cache, value_cache, num_kv_heads, scale, block_tables, context_lens, block_size,
                                   max_context_len, window_size_left, sink_tokens, alibi_slopes, workspace)


def paged_attention_window_workspace_size(num_seqs: int, num_heads: int, num_kv_heads: int, head_size: int, block_size: int,
                                          max_context_len: int, window_size_left: int, sink_tokens: int, dtype: torch.dtype) -> int:
    """Bytes of scratch memory paged_attention_window needs for these shapes on the current device."""
    n = ctypes.c_int64(0)
    call("hipattn_paged_attention_window_workspace_size", int(num_seqs), int(num_heads), int(num_kv_heads), int(head_size),
         int(block_size), int(max_context_len), int(window_size_left), int(sink_tokens), _DTYPES[dtype], ctypes.byref(n))
    return int(n.value)


def paged_attention_v1(out: torch.Tensor, query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                       num_kv_heads: int, scale: float, block_tables: torch.Tensor, context_lens: torch.Tensor,
                       block_size: int, max_context_len: int, alibi_slopes: Optional[torch.Tensor] = None) -> None:
    """lib.rs:356-391."""
    _native.paged_attention_v1(out, query, key_cache, value_cache, num_kv_heads, scale, block_tables, context_lens,
                               block_size, max_context_len, alibi_slopes)


def paged_attention_workspace_size(num_seqs: int, num_heads: int, num_kv_heads: int, head_size: int, block_size: int,
                                   max_context_len: int, dtype: torch.dtype) -> int:
    """Bytes of scratch memory paged_attention_v1 needs for these shapes on the current device."""
    n = ctypes.c_int64(0)
    call("hipattn_paged_attention_workspace_size", int(num_seqs), int(num_heads), int(num_kv_heads), int(head_size),
         int(block_size), int(max_context_len), _DTYPES[dtype], ctypes.byref(n))
    return int(n.value)


def paged_attention_v1_ws(out: torch.Tensor, query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                          num_kv_heads: int, scale: float, block_tables: torch.Tensor, context_lens: torch.Tensor,
                          block_size: int, max_context_len: int, workspace: Optional[torch.Tensor],
                          alibi_slopes: Optional[torch.Tensor] = None) -> None:
    """paged_attention_v1 on a caller-provided scratch tensor (uint8, on the GPU; None when none is needed)."""
    ptr = ctypes.c_void_p(workspace.data_ptr()) if workspace is not None else None
    nbytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    call("hipattn_paged_attention_v1_ws", _desc(out, "out"), _desc(query, "query"), _desc(key_cache, "key_cache"),
         _desc(value_cache, "value_cache"), int(num_kv_heads), float(scale), _desc(block_tables, "block_tables"),
         _desc(context_lens, "context_lens"), int(block_size), int(max_context_len), _desc(alibi_slopes, "alibi"),
         ptr, int(nbytes), _stream(query))


def paged_attention_v1_static(out: torch.Tensor, query: torch.Tensor, key_cache: torch.Tensor,
                              value_cache: torch.Tensor, num_kv_heads: int, scale: float, block_tables: torch.Tensor,
                              context_lens: torch.Tensor, block_size: int, max_context_len: int,
                              alibi_slopes: Optional[torch.Tensor] = None) -> None:
    """paged_attention_v1 on the library's built-in scratch array: allocates nothing."""
    _native.paged_attention_v1_static(out, query, key_cache, value_cache, num_kv_heads, scale, block_tables,
                                      context_lens, block_size, max_context_len, alibi_slopes)


def init() -> None:
    """Set-up for the current device ahead of the first call (hipattn_init)."""
    call("hipattn_init")


def tuning_set(name: str, value: int) -> None:
    """Sets one of the library's tuning switches (see hipattn_tuning_set in hipattn.h)."""
    call("hipattn_tuning_set", name.encode(), int(value))


def tuning_get(name: str) -> int:
    v = ctypes.c_int(0)
    call("hipattn_tuning_get", name.encode(), ctypes.byref(v))
    return int(v.value)


def paged_attention_v2(out: torch.Tensor, exp_sums: torch.Tensor, max_logits: torch.Tensor, tmp_out: torch.Tensor,
                       query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, num_kv_heads: int,
                       scale: float, block_tables: torch.Tensor, context_lens: torch.Tensor, block_size: int,
                       max_context_len: int, alibi_slopes: Optional[torch.Tensor] = None) -> None:
    """lib.rs:122-137 (declared there, no safe wrapper in the reference)."""
    _native.paged_attention_v2(out, exp_sums, max_logits, tmp_out, query, key_cache, value_cache, num_kv_heads, scale,
                               block_tables, context_lens, block_size, max_context_len, alibi_slopes)


# --------------------------------------------------------------------------- cache movement

def reshape_and_cache(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                      slot_mapping: torch.Tensor) -> None:
    """lib.rs:192-213.  The reference's wrapper widens the slots to int64; the kernels read either width, so int32 slots that
    lie end to end are taken as they are."""
    if slot_mapping.dtype != torch.int32 or not slot_mapping.is_contiguous():
        slot_mapping = slot_mapping.to(torch.int64)
    _native.reshape_and_cache(key, value, key_cache, value_cache, slot_mapping)


def gather_cached_kv(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                     slot_mapping: torch.Tensor) -> None:
    """lib.rs:215-234."""
    _native.gather_cached_kv(key, value, key_cache, value_cache, slot_mapping)


def copy_blocks(key_caches: List[torch.Tensor], value_caches: List[torch.Tensor],
                block_mapping: Dict[int, Sequence[int]]) -> None:
    """lib.rs:276-331: copy-on-write block copies in every layer's cache."""
    num_layers = len(key_caches)
    assert num_layers == len(value_caches)
    if num_layers == 0:
        return
    device = key_caches[0].device
    tsize = key_caches[0].numel()
    pairs: List[int] = []
    for src, dsts in block_mapping.items():
        for dst in dsts:
            pairs += [int(src), int(dst)]
    # addresses and pairs as arguments of the launch; False for blocks that are not whole 16-byte rows
    if _native.copy_blocks(key_caches, value_caches, pairs):
        return
    blocks = key_caches[0].size(0)
    for src, dst in zip(pairs[::2], pairs[1::2]):
        if not (0 <= src < blocks and 0 <= dst < blocks):
            raise HipAttnError(f"copy_blocks: pair {src} -> {dst} out of range, the caches have {blocks} blocks")
    for e in list(key_caches) + list(value_caches):
        assert e.device == device and e.numel() == tsize and e.is_contiguous()
        assert e.dtype in (torch.float16, torch.bfloat16)
    kp = torch.tensor([t.data_ptr() for t in key_caches], dtype=torch.int64).to(device)
    vp = torch.tensor([t.data_ptr() for t in value_caches], dtype=torch.int64).to(device)
    bm = torch.tensor(pairs, dtype=torch.int64).to(device)
    call("hipattn_copy_blocks_2", _desc(kp), _desc(vp), _desc(bm), _desc(key_caches[0], "key0"), _stream(kp))


def swap_blocks(src: torch.Tensor, dst: torch.Tensor, block_mapping: Dict[int, int], stream=None) -> None:
    """cache_kernels.cu:12-50 (the reference's Rust wrapper is `todo!()`, lib.rs:236-243)."""
    pairs: List[int] = []
    for s, d in block_mapping.items():
        pairs += [int(s), int(d)]
    arr = (ctypes.c_int64 * max(1, len(pairs)))(*pairs)
    dev = src if src.is_cuda else dst
    raw = ctypes.c_void_p(stream.raw) if stream is not None else _stream(dev)
    call("hipattn_swap_blocks", _desc(src, "src", device=False), int(src.is_cuda), _desc(dst, "dst", device=False),
         int(dst.is_cuda), arr, len(pairs) // 2, raw)


# --------------------------------------------------------------------------- small ops

def rotary_embedding(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, head_size: int,
                     cos_sin_cache: torch.Tensor, is_neox: bool) -> None:
    """lib.rs:333-354; query/key [T, H*d] are rotated in place."""
    _native.rotary_embedding(positions, query, key, head_size, cos_sin_cache, is_neox)


def rotary_embedding_and_cache(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                               head_size: int, cos_sin_cache: torch.Tensor, is_neox: bool, key_cache: torch.Tensor,
                               value_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """rotary_embedding (llm/mod.rs:88-114) and reshape_and_cache (mod.rs:147-164) of a step's new tokens in
    one launch: query/key [T, H*d] rotated in place, rotated keys and value [T, Hkv, d] written to the cache."""
    _native.rotary_embedding_and_cache(positions, query, key, value, head_size, cos_sin_cache, is_neox, key_cache,
                                       value_cache, slot_mapping)


def rms_norm(out: torch.Tensor, input: torch.Tensor, weight: torch.Tensor, epsilon: float) -> None:
    _native.rms_norm(out, input, weight, epsilon)


def fused_add_rms_norm(input: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, epsilon: float) -> None:
    _native.fused_add_rms_norm(input, residual, weight, epsilon)


def add_rms_norm_takes(input: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor) -> bool:
    """Whether `add_rms_norm` accepts these operands (else a caller makes the two calls)."""
    return (input.dtype in (torch.float16, torch.bfloat16) and input.size(1) % 8 == 0 and input.size(1) <= 8192
            and all(t.dtype == input.dtype and t.is_contiguous() and t.data_ptr() % 16 == 0 for t in (input, residual, weight)))


def add_rms_norm(input: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, epsilon: float) -> torch.Tensor:
    """input += residual and rms_norm of the sum, in one launch with the bits of the two calls (llama.rs:166 + 169, 173 + 165): returns
    the norm; input [rows, hidden] holds the sum."""
    out = torch.empty_like(input)
    _native.add_rms_norm(out, input, residual, weight, epsilon)
    return out


LINEAR_MAX_ROWS = 128


def linear_takes(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """Whether `linear` accepts these operands (else a caller multiplies with a library GEMM)."""
    return (x.dim() == 2 and weight.dim() == 2 and 0 < x.size(0) <= LINEAR_MAX_ROWS and x.size(1) % 256 == 0
            and weight.size(0) % 16 == 0 and x.dtype in (torch.float16, torch.bfloat16) and weight.dtype == x.dtype
            and x.stride(1) == 1 and weight.stride(1) == 1 and x.stride(0) % 8 == 0 and weight.stride(0) % 8 == 0
            and x.data_ptr() % 16 == 0 and weight.data_ptr() % 16 == 0)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
           workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = x @ weight.T (+ bias) (+ residual) for at most 128 rows of x: `nn::Linear::forward` as rLLM calls
    it for the rows of a generation step (llm/mod.rs:401-416; llama.rs:81-83, 96, 135-143, 210)."""
    if out is None:
        out = torch.empty((x.size(0), weight.size(0)), dtype=x.dtype, device=x.device)
    _native.linear(out, x, weight, bias, residual, workspace)
    return out


def linear_fp8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = x @ (weight * its scales).T (+ bias) (+ residual) for any number of rows of x [M, K], f16 or bf16: weight [N, K] float8_e4m3fn,
    weight_scale f32 [ceil(N / 128), ceil(K / 128)], one for each 128 x 128 of weight (`quantize_weight_fp8`).  The rows of x are rounded to
    e4m3 in blocks of 128 columns, scaled by powers of two.  out may lie over x, and be the residual.  workspace: uint8,
    `linear_fp8_workspace_size` bytes; None: a buffer that the library keeps per stream."""
    if out is None:
        out = torch.empty((x.size(0), weight.size(0)), dtype=x.dtype, device=x.device)
    _native.linear_fp8(out, x, weight, weight_scale, bias, residual, workspace)
    return out


def linear_fp8_workspace_size(x: torch.Tensor, weight: torch.Tensor) -> int:
    n = ctypes.c_int64(0)
    call("hipattn_linear_fp8_workspace_size", _desc(x, "x"), _desc(weight, "weight"), ctypes.byref(n))
    return int(n.value)


def quantize_weight_fp8(weight: torch.Tensor):
    """(weight in float8_e4m3fn, f32 scales [ceil(N / 128), ceil(K / 128)]) of a weight [N, K] for `linear_fp8`: in each 128 x 128 of it the
    largest magnitude becomes 448.  For loading, a strip of 128 rows at a time: nothing of the weight's size is held in 32 bits."""
    n, k = weight.shape
    nb, kb = (n + 127) // 128, (k + 127) // 128
    data = torch.empty((n, k), dtype=torch.float8_e4m3fn, device=weight.device)
    scale = torch.empty((nb, kb), dtype=torch.float32, device=weight.device)
    largest = torch.full((1,), 448.0, device=weight.device)  # (a tensor: by a number a GPU multiplies with the reciprocal, and a CPU divides)
    for b in range(nb):
        rows = weight[128 * b:128 * b + 128]
        strip = torch.zeros((rows.size(0), kb * 128), dtype=torch.float32, device=weight.device)
        strip[:, :k] = rows
        strip = strip.view(-1, kb, 128)
        most = strip.abs().amax((0, 2)) / largest
        scale[b] = torch.where(most > 0, most, torch.ones_like(most))
        data[128 * b:128 * b + 128] = (strip / scale[b][None, :, None]).clamp(-448.0, 448.0).view(rows.size(0), -1)[:, :k].to(torch.float8_e4m3fn)
    return data, scale


def linear_silu_and_mul(x: torch.Tensor, weight: torch.Tensor, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """silu_and_mul(x @ weight.T) for at most 128 rows of x, weight [2 n, K] with the gate rows first (llama.rs:135-142):
    the bits of `linear` followed by `silu_and_mul`, without the [M, 2 n] product in memory."""
    out = torch.empty((x.size(0), weight.size(0) // 2), dtype=x.dtype, device=x.device)
    _native.linear_silu_and_mul(out, x, weight, workspace)
    return out


def linear_rms_norm(x: torch.Tensor, weight: torch.Tensor, norm_weight: torch.Tensor, epsilon: float,
                    bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None):
    """`linear` and the RMS norm of its rows in the launch that finishes them: returns (out, rms_norm(out)),
    the same bits as `linear` followed by `rms_norm`."""
    out = torch.empty((x.size(0), weight.size(0)), dtype=x.dtype, device=x.device)
    normed = torch.empty_like(out)
    _native.linear_rms_norm(out, normed, x, weight, bias, residual, norm_weight, epsilon, workspace)
    return out, normed


RMS_NORM_LINEAR_MAX_ROWS = 4


def rms_norm_linear_takes(x: torch.Tensor, norm_weight: torch.Tensor, weight: torch.Tensor) -> bool:
    """Whether `rms_norm_linear` accepts these operands (else a caller makes the two calls)."""
    return (linear_takes(x, weight) and x.size(0) <= RMS_NORM_LINEAR_MAX_ROWS and x.size(1) <= 8192
            and norm_weight.dtype == x.dtype and norm_weight.numel() == x.size(1) and norm_weight.is_contiguous()
            and norm_weight.data_ptr() % 16 == 0 and (x.size(0) + 1) * ((x.size(1) * 2 + 1023) // 1024) <= 40
            and weight.size(0) < 65536 and weight.size(0) % 32 == 0
            and 0 < weight.stride(0) < 1 << 28 and (x.size(0) == 1 or 0 <= x.stride(0) < 1 << 28))


def rms_norm_linear(x: torch.Tensor, norm_weight: torch.Tensor, epsilon: float, weight: torch.Tensor,
                    silu_and_mul: bool = False) -> torch.Tensor:
    """rms_norm(x) @ weight.T, or with silu_and_mul behind it (weight [2 n, K], the gate rows first), in one launch for the few
    rows of a small step (llama.rs:165 + 81-83, 169 + 135-142): the bits of the two calls."""
    out = torch.empty((x.size(0), weight.size(0) // 2 if silu_and_mul else weight.size(0)), dtype=x.dtype, device=x.device)
    _native.rms_norm_linear(out, x, norm_weight, epsilon, weight, silu_and_mul)
    return out


def qkv_linear_takes(x: torch.Tensor, weight: torch.Tensor, cos_sin_cache: torch.Tensor, key_cache: torch.Tensor,
                     value_cache: torch.Tensor) -> bool:
    """Whether `qkv_linear` accepts these operands without a norm (else a caller makes the two calls)."""
    d = cos_sin_cache.size(1)
    return (linear_takes(x, weight) and weight.size(0) < (65536 if x.size(0) <= 16 else 16384) and d % 16 == 0
            and key_cache.dim() == 5 and key_cache.size(2) * key_cache.size(4) == d and weight.size(0) % d == 0
            and weight.size(0) // d > 2 * key_cache.size(1) > 0
            and 0 < weight.stride(0) < 1 << 28 and (x.size(0) == 1 or 0 <= x.stride(0) < 1 << 28)
            and cos_sin_cache.dtype == key_cache.dtype == value_cache.dtype == x.dtype and cos_sin_cache.is_contiguous()
            and cos_sin_cache.data_ptr() % 16 == 0 and key_cache.data_ptr() % 16 == 0 and key_cache.stride(0) % 8 == 0
            and key_cache.stride(1) % 8 == 0)


def qkv_linear(x: torch.Tensor, norm_weight: Optional[torch.Tensor], epsilon: float, weight: torch.Tensor, positions: torch.Tensor,
               cos_sin_cache: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
               slot_mapping: torch.Tensor) -> torch.Tensor:
    """x @ weight.T, behind rms_norm of the rows where norm_weight is given, and rotary_embedding_and_cache of its heads (llama.rs:81-85 +
    mod.rs:147-164) in the projection's own launches (wide weights and heads that do not divide 128: one more): returns [M, (Hq + 2 Hkv) d]
    with the bits of the calls."""
    out = torch.empty((x.size(0), weight.size(0)), dtype=x.dtype, device=x.device)
    _native.qkv_linear(out, x, norm_weight, epsilon, weight, positions, cos_sin_cache, key_cache, value_cache, slot_mapping)
    return out


def linear_rms_norm_workspace_size(x: torch.Tensor, weight: torch.Tensor) -> int:
    n = ctypes.c_int64(0)
    call("hipattn_linear_rms_norm_workspace_size", _desc(x, "x"), _desc(weight, "weight"), ctypes.byref(n))
    return int(n.value)


def linear_workspace_size(x: torch.Tensor, weight: torch.Tensor) -> int:
    n = ctypes.c_int64(0)
    call("hipattn_linear_workspace_size", _desc(x, "x"), _desc(weight, "weight"), ctypes.byref(n))
    return int(n.value)


def silu_and_mul(out: torch.Tensor, input: torch.Tensor) -> None:
    _native.silu_and_mul(out, input)


def gelu_new(out: torch.Tensor, input: torch.Tensor) -> None:
    _native.gelu_new(out, input)


def gelu_fast(out: torch.Tensor, input: torch.Tensor) -> None:
    _native.gelu_fast(out, input)


def bias_argmax(logits: torch.Tensor, bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                bias_rows: Optional[torch.Tensor] = None, return_logits: bool = False):
    """Greedy token after the AICI bias (tmodel.rs:277-283 + 234-236) for every row at once.

    bias: f32 [R, >=V] rows of 0/-inf; mask: u8 [R, bytes] packed allow-bits.  Returns int32 [S]."""
    S = logits.size(0)
    tokens = torch.empty((S,), dtype=torch.int32, device=logits.device)
    best = torch.empty((S,), dtype=torch.float32, device=logits.device) if return_logits else None
    _native.bias_argmax(logits, bias, mask, bias_rows, tokens, best)
    return (tokens, best) if return_logits else tokens


def bias_sample(logits: torch.Tensor, temperature: torch.Tensor, top_p: torch.Tensor, uniforms: torch.Tensor,
                bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                bias_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """AICI bias, temperature, top-p and the draw (tmodel.rs:277-283, 172-194, 236-268) for every row at once.
    temperature / top_p / uniforms: f32 [S]; rows with temperature < 1e-5 are greedy; uniforms in [0, 1) are
    the caller's random numbers (one per row).  Returns int32 [S]."""
    S = logits.size(0)
    tokens = torch.empty((S,), dtype=torch.int32, device=logits.device)
    _native.bias_sample(logits, bias, mask, bias_rows, temperature, top_p, uniforms, tokens)
    return tokens


def penalize_logits(logits: torch.Tensor, history: torch.Tensor, history_offsets: torch.Tensor,
                    prompt_lens: Optional[torch.Tensor] = None, repetition: Optional[torch.Tensor] = None,
                    frequency: Optional[torch.Tensor] = None, presence: Optional[torch.Tensor] = None,
                    bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None, bias_rows: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Penalties for what every row's sequence has said, bias and allow-mask on the logits [S, V], in front of `bias_argmax` /
    `bias_sample`.  history int32 [N]: the sequences' tokens one after the other, from history_offsets [S + 1] on, the first
    prompt_lens [S] of each its prompt.  A token that the sequence holds: x / repetition where x > 0, else x * repetition; then
    - frequency * count - presence * (count > 0), counted behind the prompt; + bias; -inf where the mask bars it.  Returns `out`, by
    default a new tensor of out_dtype (that of logits, or float32); out=logits works in place."""
    if out is None:
        out = torch.empty_like(logits, dtype=out_dtype)
    _native.penalize_logits(out, logits, history, history_offsets, prompt_lens, repetition, frequency, presence, bias, mask, bias_rows)
    return out


# --------------------------------------------------------------------------- a step's blocks on the device

class StepBlocks(NamedTuple):
    """What `step_blocks` makes of a step."""
    state: torch.Tensor         # int32 [R, 2]: tokens in the cache, columns gone
    ends: torch.Tensor          # int64 [2]: head and tail of the ring of free blocks
    served: torch.Tensor        # int32 [R]: tokens given; -1: no blocks or rows left, -2: does not fit its table or its rows
    context_lens: torch.Tensor  # int32 [R]: keys of a request that is served, else 0
    seqlens_q: torch.Tensor     # int32 [R + 1]: sums of the tokens given
    logit_idxs: torch.Tensor    # int32 [R]: a served request's last row, else 0
    positions: torch.Tensor     # int64 [T]
    slot_mapping: torch.Tensor  # int32 [T], -1: no token
    totals: torch.Tensor        # int32 [4]: tokens given, requests not served, blocks free, blocks taken


STEP_BLOCKS_MAX_REQUESTS = 4096


def step_blocks(new_lens: torch.Tensor, state: torch.Tensor, block_tables: torch.Tensor, free_ring: torch.Tensor, ring_ends: torch.Tensor,
                block_size: int, num_rows: int, rows_per_request: int = 0, window_size_left: int = -1, sink_tokens: int = 0,
                state_out: Optional[torch.Tensor] = None, ring_ends_out: Optional[torch.Tensor] = None) -> StepBlocks:
    """A step's block bookkeeping on the device (hipattn_step_blocks in hipattn.h): new_lens int32 [R] tokens per request (0: idle,
    negative: ended); blocks that ended requests and windows let go return to free_ring, blocks that are needed come from it into
    block_tables, both updated in place, and num_rows rows get their positions and slots.  state_out / ring_ends_out default to new
    tensors; they may be state / ring_ends themselves."""
    R = new_lens.size(0)
    # One allocation for what a step hands out, cut into pieces on the boundaries they need: the host's time per call is what a small step
    # waits for (a piece costs some 0.4 us, an allocation more).
    T = int(num_rows)
    pool = new_lens.new_empty(10 * R + 13 + 3 * T)
    work, new_state, positions, new_ends, served, context_lens, seqlens_q, logit_idxs, slots, totals = torch.unsafe_split_with_sizes(
        pool, (4 * R + 4, 2 * R, 2 * T, 4, R, R, R + 1, R, T, 4))
    positions = positions.view(torch.int64)
    if state_out is None:
        state_out = new_state.view(R, 2)
    if ring_ends_out is None:
        ring_ends_out = new_ends.view(torch.int64)
    _native.step_blocks(new_lens, state, block_tables, free_ring, ring_ends, block_size, rows_per_request, window_size_left, sink_tokens,
                        state_out, ring_ends_out, served, context_lens, seqlens_q, logit_idxs, positions, slots, totals, work)
    return StepBlocks(state_out, ring_ends_out, served, context_lens, seqlens_q, logit_idxs, positions, slots, totals)


# --------------------------------------------------------------------------- trees of drafted tokens

class TreeRows(NamedTuple):
    """What `tree_rows` says of a step's trees."""
    positions: torch.Tensor  # int64 [T]
    mask: torch.Tensor       # int64 [T, (max_seqlen_q + 63) / 64]: bits of the rows of its tree that a row sees


def tree_rows(parents: torch.Tensor, seqlens_q: torch.Tensor, context_lens: torch.Tensor, max_seqlen_q: int) -> TreeRows:
    """Positions and masks of trees of drafted tokens (hipattn_tree_rows in hipattn.h): parents int32 [T], the row of its own tree that a
    row continues, negative: none; a row sees itself and its ancestors and lies behind as many of them.  At most 1024 rows a tree."""
    T = parents.size(0)
    rows = TreeRows(torch.empty((T,), dtype=torch.int64, device=parents.device),
                    torch.empty((T, (int(max_seqlen_q) + 63) // 64), dtype=torch.int64, device=parents.device))
    _native.tree_rows(parents, seqlens_q, context_lens, max_seqlen_q, rows.positions, rows.mask)
    return rows


class CacheList:
    """Every layer's key and value cache as `tree_accept` takes them: made once, when the caches are, and kept with them."""

    def __init__(self, key_caches: Sequence[torch.Tensor], value_caches: Sequence[torch.Tensor]):
        self.key_caches, self.value_caches = list(key_caches), list(value_caches)
        if not self.key_caches or len(self.key_caches) != len(self.value_caches):
            raise HipAttnError(f"CacheList: {len(self.key_caches)} key caches and {len(self.value_caches)} value caches")
        for caches in (self.key_caches, self.value_caches):
            first = caches[0]
            for t in caches:
                if not t.is_cuda or t.device != self.key_caches[0].device:
                    raise HipAttnError(f"CacheList: expected GPU tensors of one device, got one on {t.device}")
                if t.dtype != self.key_caches[0].dtype or t.size() != first.size() or t.stride() != first.stride() or t.data_ptr() % 16 != 0:
                    raise HipAttnError("CacheList: the layers' caches must have one type, one shape and the same strides, and start on 16-byte boundaries")
        # (layers that share a cache have it once in the list: two moves of the same rows at a time would take from each other what they have moved)
        if self.key_caches[0].numel() > 0 and len({t.data_ptr() for t in self.key_caches + self.value_caches}) < 2 * len(self.key_caches):
            raise HipAttnError("CacheList: the same cache twice")
        device = self.key_caches[0].device
        self.key_ptrs = torch.tensor([t.data_ptr() for t in self.key_caches], dtype=torch.int64).to(device)
        self.value_ptrs = torch.tensor([t.data_ptr() for t in self.value_caches], dtype=torch.int64).to(device)


class TreeAccept(NamedTuple):
    """What `tree_accept` keeps of a step's trees."""
    lens: torch.Tensor         # int32 [R]: rows kept, the root among them; 0 without rows
    path: torch.Tensor         # int32 [R, max_seqlen_q]: which, counted in the tree; -1 behind the last
    next_tokens: torch.Tensor  # int32 [R]: the token that follows the last of them; -1 without rows


def tree_accept(tokens: torch.Tensor, parents: torch.Tensor, chosen: torch.Tensor, seqlens_q: torch.Tensor, max_seqlen_q: int,
                slot_mapping: Optional[torch.Tensor] = None, caches: Optional[CacheList] = None) -> TreeAccept:
    """The drafted tokens that the model's choices confirm (hipattn_tree_accept in hipattn.h): tokens, parents, chosen int32 [T], `chosen`
    what `bias_argmax` or `bias_sample` gives for every row.  With slot_mapping [T] and caches the kept rows' keys and values move to the slots of
    the tree's first rows, in every layer."""
    R, device = seqlens_q.size(0) - 1, tokens.device
    kept = TreeAccept(torch.empty((max(R, 0),), dtype=torch.int32, device=device),
                      torch.empty((max(R, 0), int(max_seqlen_q)), dtype=torch.int32, device=device),
                      torch.empty((max(R, 0),), dtype=torch.int32, device=device))
    if caches is None:
        _native.tree_accept(tokens, parents, chosen, seqlens_q, max_seqlen_q, slot_mapping, None, None, None, None, kept.lens, kept.path,
                            kept.next_tokens)
    else:
        _native.tree_accept(tokens, parents, chosen, seqlens_q, max_seqlen_q, slot_mapping, caches.key_ptrs, caches.value_ptrs,
                            caches.key_caches[0], caches.value_caches[0], kept.lens, kept.path, kept.next_tokens)
    return kept


# --------------------------------------------------------------------------- runtime plumbing

class Stats:
    """lib.rs:393-400."""

    def __init__(self, s: _lib.MemStats):
        self.current, self.peak, self.allocated, self.freed = s.current, s.peak, s.allocated, s.freed

    def __str__(self) -> str:
        G = 1024.0 ** 3
        return (f"current: {self.current / G:.3f}GiB, peak: {self.peak / G:.3f}GiB, "
                f"allocated: {self.allocated / G:.3f}GiB, freed: {self.freed / G:.3f}GiB")


def cuda_reset_peak_memory_stats(device: int) -> None:
    call("hipattn_reset_peak_memory_stats", int(device))


def cuda_empty_cache() -> None:
    call("hipattn_empty_cache")


def cuda_get_stats_allocated_bytes(device: int) -> Stats:
    s = _lib.MemStats()
    call("hipattn_get_stats_allocated_bytes", int(device), ctypes.byref(s))
    return Stats(s)


def cuda_get_device_properties(device: int) -> _lib.DeviceProps:
    p = _lib.DeviceProps()
    call("hipattn_get_device_properties", int(device), ctypes.byref(p))
    return p


class CudaStream:
    """stream.rs:30-151 over hipStream_t."""
    DEFAULT, CURRENT, HIGH_PRI, LOW_PRI = range(4)

    def __init__(self, typ: int = LOW_PRI, device: int = 0, _handle=None):
        if _handle is None:
            h = ctypes.c_void_p()
            call("hipattn_stream_get", int(typ), int(device), ctypes.byref(h))
            _handle = h
        self._h = _handle

    @classmethod
    def default(cls, device: int = 0) -> "CudaStream":
        return cls(cls.DEFAULT, device)

    @classmethod
    def current(cls, device: int = 0) -> "CudaStream":
        return cls(cls.CURRENT, device)

    def clone(self) -> "CudaStream":
        h = ctypes.c_void_p()
        call("hipattn_stream_clone", self._h, ctypes.byref(h))
        return CudaStream(_handle=h)

    def query(self) -> bool:
        done = ctypes.c_int()
        call("hipattn_stream_query", self._h, ctypes.byref(done))
        return bool(done.value)

    def synchronize(self) -> None:
        call("hipattn_stream_synchronize", self._h)

    def set_current(self) -> None:
        call("hipattn_stream_set_current", self._h)

    def device_index(self) -> int:
        i = ctypes.c_int()
        call("hipattn_stream_device_index", self._h, ctypes.byref(i))
        return i.value

    def id(self) -> int:
        i = ctypes.c_int64()
        call("hipattn_stream_id", self._h, ctypes.byref(i))
        return i.value

    @property
    def raw(self) -> int:
        r = ctypes.c_void_p()
        call("hipattn_stream_raw", self._h, ctypes.byref(r))
        return r.value or 0

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h:
            try:
                call("hipattn_stream_free", h)
            except Exception:
                pass


class CudaEvent:
    """event.rs:34-138 over hipEvent_t."""

    def __init__(self, timing: bool = False, blocking: bool = False):
        h = ctypes.c_void_p()
        call("hipattn_event_create", bool(timing), bool(blocking), ctypes.byref(h))
        self._h = h

    def record(self, stream: CudaStream) -> None:
        call("hipattn_event_record", self._h, stream._h)

    def wait(self, stream: CudaStream) -> None:
        call("hipattn_event_block", self._h, stream._h)

    def elapsed_time(self, end: "CudaEvent") -> float:
        ms = ctypes.c_float()
        call("hipattn_event_elapsed_time", self._h, end._h, ctypes.byref(ms))
        return ms.value

    def query(self) -> bool:
        done = ctypes.c_int()
        call("hipattn_event_query", self._h, ctypes.byref(done))
        return bool(done.value)

    def synchronize(self) -> None:
        call("hipattn_event_synchronize", self._h)

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h:
            try:
                call("hipattn_event_free", h)
            except Exception:
                pass
