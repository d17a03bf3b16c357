/*
 * hipattn — C ABI of the MI355X (gfx950) attention path for rLLM.
 *
 * This header is the drop-in boundary: every entry point replaces one of the
 * `extern "C"` functions that rLLM's `tch-cuda` crate binds
 * (rllm/tch-cuda/src/lib.rs:29-47,107-190,426-431, src/stream.rs:18-28,
 * src/event.rs:12-28; implemented in rllm/tch-cuda/kernels/vllm_bindings.cpp:15-90,
 * kernels/flash_attn/flash_api.cpp:621-655, kernels/cuda.cpp:32-149).
 *
 * Differences from the reference ABI, all forced by dropping libtorch:
 *   - a tensor is a plain descriptor (`hipattn_tensor`: device pointer, dtype,
 *     sizes, strides in elements) instead of `torch::Tensor*`;
 *   - every op takes the HIP stream it enqueues on as its last argument
 *     (`hipStream_t` passed as `void*`; NULL = the thread's current stream as
 *     set by hipattn_stream_set_current, initially the device's default stream);
 *     the reference launches on torch's implicit current stream;
 *   - outputs are caller-allocated, including the one output the reference
 *     allocates itself (`mha_varlen_fwd_C`'s `outp`).
 *
 * Conventions kept from the reference:
 *   - every call returns `char*`: NULL on success, otherwise a malloc'd,
 *     NUL-terminated message that the caller releases with `free()` (or
 *     hipattn_free_error); nothing is thrown across the ABI
 *     (vllm_bindings.cpp:7-13);
 *   - ops only enqueue work, they never synchronise the device;
 *   - index dtypes: slot_mapping int64 for reshape_and_cache and int32 for
 *     gather_cached_kv (lib.rs:199-200), positions int64, block_tables /
 *     context_lens / cu_seqlens int32.  Where it is harmless both widths are
 *     accepted.
 */
#ifndef HIPATTN_H
#define HIPATTN_H

#include <stdbool.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HIPATTN_MAX_DIMS 5

typedef enum hipattn_dtype {
  HIPATTN_F32 = 0,
  HIPATTN_F16 = 1,
  HIPATTN_BF16 = 2,
  HIPATTN_I32 = 3,
  HIPATTN_I64 = 4,
  HIPATTN_U8 = 5
} hipattn_dtype;

/* Borrowed view of device (or, for host-side builders, host) memory.
 * strides are in elements, as torch reports them. */
typedef struct hipattn_tensor {
  void *data;
  int32_t dtype; /* hipattn_dtype */
  int32_t ndim;
  int64_t sizes[HIPATTN_MAX_DIMS];
  int64_t strides[HIPATTN_MAX_DIMS];
} hipattn_tensor;

void hipattn_free_error(char *msg);
/* "major.minor.patch" of this library; static storage. */
const char *hipattn_version(void);

/* ---------------------------------------------------------------------------
 * Attention
 * ------------------------------------------------------------------------- */

/* Replaces mha_varlen_fwd_C (lib.rs:29-47; flash_api.cpp:447-655).
 * q [total_q, Hq, d], k/v [total_k, Hkv, d] (last dim contiguous, row and head
 * strides honoured), cu_seqlens_* int32 [b+1], seqused_k int32 [b] or NULL,
 * out [total_q, Hq, d] caller-allocated, in q's dtype or f32 (the accumulators
 * divided by the row sums and not rounded again: the form in which the
 * kernel's arithmetic can be checked apart from the rounding of its output),
 * softmax_lse f32 [b, Hq, max_seqlen_q] or NULL.  fp16/bf16 inputs, d % 8 == 0, d <= 256, Hq % Hkv == 0.  Causal masking is
 * bottom-right aligned: key j is visible to query i iff j <= i + (Lk - Lq)
 * (flash_attn/softmax.h:159-160).  window_size_left / window_size_right as in
 * the reference (flash_api.cpp:113-120,466; softmax.h:155-166): with bounds
 * (l, r) key j is visible iff i + (Lk - Lq) - l <= j <= i + (Lk - Lq) + r, a
 * negative bound is no bound, is_causal forces r = 0; rLLM passes (-1,-1).
 * p_dropout must be 0; zero_tensors clears out (and lse) first. */
char *hipattn_mha_varlen_fwd(const hipattn_tensor *q, const hipattn_tensor *k,
                             const hipattn_tensor *v,
                             const hipattn_tensor *cu_seqlens_q,
                             const hipattn_tensor *cu_seqlens_k,
                             const hipattn_tensor *seqused_k, int max_seqlen_q,
                             int max_seqlen_k, float p_dropout,
                             float softmax_scale, bool zero_tensors,
                             bool is_causal, int window_size_left,
                             int window_size_right, hipattn_tensor *out,
                             hipattn_tensor *softmax_lse, void *stream);

/* Varlen prefill over the paged cache.  No counterpart in tch-cuda: it replaces
 * the sequence gather_cached_kv -> repeat_kv -> flash_attn_varlen that
 * rllm-cuda/src/llm/mod.rs:181-238 runs for multi-token rows (K/V of the whole
 * context copied out of the cache, kv heads repeated) by one kernel that reads
 * K/V through block tables, like paged_attention does for single tokens.
 * q/out [total_q, Hq, d]; key_cache [nb, Hkv, d/8, BS, 8], value_cache
 * [nb, Hkv, d, BS] with BS = 8, 16 or 32 (read from the caches' shapes; 16,
 * what rLLM runs, has the fast kernels); block_tables int32 [b, cols]: key
 * position p of sequence i is in block block_tables[i][p / BS] at offset p % BS
 * (the new tokens' K/V must already be in the cache); cu_seqlens_q int32 [b+1]; context_lens int32
 * [b] = keys per sequence; causal mask bottom-right aligned as in
 * hipattn_mha_varlen_fwd; out in q's dtype or f32 as there.  fp16/bf16, d % 8 == 0, d <= 256 (what
 * flash_api.cpp:522-523 serves). */
char *hipattn_mha_varlen_fwd_paged(const hipattn_tensor *q, const hipattn_tensor *key_cache,
                                   const hipattn_tensor *value_cache, const hipattn_tensor *block_tables,
                                   const hipattn_tensor *cu_seqlens_q, const hipattn_tensor *context_lens,
                                   int max_seqlen_q, int max_seqlen_k, float softmax_scale, bool is_causal,
                                   hipattn_tensor *out, hipattn_tensor *softmax_lse, void *stream);

/* hipattn_mha_varlen_fwd_paged with a sliding window and sinks: always causal, and the query at position p of its sequence sees key j
 * iff j <= p and (j >= p - window_size_left or j < sink_tokens) -- window_size_left + 1 tokens with its own, as the window of
 * hipattn_mha_varlen_fwd counts them, and the first sink_tokens of the sequence.  No counterpart in tch-cuda (its windows have no sinks
 * and read rows of k / v).  Sinks are keys like others, as the cache holds them: nothing is rotated anew, and no term is added to the softmax.
 * window_size_left >= 0, sink_tokens >= 0; everything else as there, any of its types, head and block sizes.
 * max_seqlen_q and max_seqlen_k bound every sequence's new tokens and keys: rows and keys beyond them may be left out.
 * Keys that no new token of a sequence sees may be gone: table columns that hold only such keys may name any block or none (a negative
 * or large number), and their blocks may hold anything.  Values of a key that some of a sequence's new tokens see are taken to be finite,
 * also where others do not see it.  A row that sees nothing (its position is negative) is zero, its LSE +inf.
 * Where few workgroups would leave compute units idle a row's keys are dealt out to several (not with an f32 out or an LSE), by way of
 * workspace: u8, 256-byte aligned, hipattn_mha_varlen_fwd_paged_window_workspace_size bytes (at most 64 MiB), not shared by calls that overlap,
 * replays of captured ones included; where no keys can be dealt out (as well: head sizes other than 64, 80, 96, 112, 128 and 256, and rows of
 * which two pieces exceed 64 MiB) nothing is asked of it.  NULL: a buffer of 64 MiB that the library allocates once per stream; under capture, on
 * hipStreamPerThread and without that memory keys are then not dealt out, so that last bits, and the time of few long rows, may differ. */
char *hipattn_mha_varlen_fwd_paged_window(const hipattn_tensor *q, const hipattn_tensor *key_cache,
                                          const hipattn_tensor *value_cache, const hipattn_tensor *block_tables,
                                          const hipattn_tensor *cu_seqlens_q, const hipattn_tensor *context_lens,
                                          int max_seqlen_q, int max_seqlen_k, float softmax_scale,
                                          int window_size_left, int sink_tokens, hipattn_tensor *out,
                                          hipattn_tensor *softmax_lse, const hipattn_tensor *workspace, void *stream);
char *hipattn_mha_varlen_fwd_paged_window_workspace_size(int64_t total_q, int num_heads, int head_size, int64_t *bytes);

/* Replaces paged_attention_v1_C (lib.rs:107-120; attention_kernels.cu:679-700).
 * out/query [S, Hq, d]; key_cache [nb, Hkv, d/x, BS, x]; value_cache
 * [nb, Hkv, d, BS]; block_tables int32 [S, max_blocks]; context_lens int32 [S].
 * alibi_slopes f32 [Hq] or NULL.  A context length above max_context_len is
 * cut there.  Runs the split-K kernels on scratch memory the library owns: one
 * buffer per (device, stream), so calls on different streams may overlap, and
 * threads may share a stream (a call has the buffer to itself until its
 * launches are enqueued; hipStreamPerThread counts as one stream per thread, each
 * with a buffer until hipattn_shutdown); it
 * grows with hipMalloc when a call needs more than it has (the old buffer stays
 * alive until hipattn_shutdown, nothing is synchronised); a stream that is being
 * captured into a graph cannot grow it -- run the call once with the largest
 * shapes before capturing, or use hipattn_paged_attention_v1_ws.
 * x = 16 / sizeof(dtype).  The reference's support matrix is accepted: f16,
 * bf16 and f32; BS 8, 16 and 32; d in {64, 80, 96, 112, 128, 256}.  The
 * 2-byte types take the MFMA kernels at every block size; f32 caches, and
 * BS 8 / 32 at other head sizes (any d <= 256 that is a multiple of x), take
 * a plain fp32 kernel. */
char *hipattn_paged_attention_v1(hipattn_tensor *out,
                                 const hipattn_tensor *query,
                                 const hipattn_tensor *key_cache,
                                 const hipattn_tensor *value_cache,
                                 int num_kv_heads, float scale,
                                 const hipattn_tensor *block_tables,
                                 const hipattn_tensor *context_lens,
                                 int block_size, int max_context_len,
                                 const hipattn_tensor *alibi_slopes,
                                 void *stream);

/* hipattn_paged_attention_v1 on scratch memory the caller provides: the
 * "workspace-size query + caller-allocated split-K scratch" form of the call
 * (the reference's v1 signature has no such argument, lib.rs:107-120; its v2
 * passes three tensors).  workspace: device memory, 256-byte aligned, of at
 * least the number of bytes hipattn_paged_attention_workspace_size reports for
 * these shapes (NULL is fine when that is 0); its contents need not be
 * preserved or cleared between calls.  Calls that overlap in time need
 * workspaces of their own. */
char *hipattn_paged_attention_v1_ws(hipattn_tensor *out,
                                    const hipattn_tensor *query,
                                    const hipattn_tensor *key_cache,
                                    const hipattn_tensor *value_cache,
                                    int num_kv_heads, float scale,
                                    const hipattn_tensor *block_tables,
                                    const hipattn_tensor *context_lens,
                                    int block_size, int max_context_len,
                                    const hipattn_tensor *alibi_slopes,
                                    void *workspace, int64_t workspace_bytes,
                                    void *stream);

/* hipattn_paged_attention_v1 for callers that cannot allocate (code under HIP
 * graph capture, tight serving loops, harnesses that forbid hipMalloc); it has
 * no counterpart in the reference.  Same arguments and results as
 * hipattn_paged_attention_v1, but the split-K scratch memory is a 16 MiB array
 * built into the library's code object (each device the library runs on holds
 * it until the process ends), so the call allocates and frees nothing.  A call
 * whose shapes need more (hipattn_paged_attention_workspace_size) is refused
 * with a message.  Every call on a device uses that device's one array: calls
 * that overlap in time on one device (two streams, two threads) race.  The
 * first call on a device asks the runtime for the array's address and for the
 * decode kernels' occupancy; hipattn_init does that ahead of time. */
char *hipattn_paged_attention_v1_static(hipattn_tensor *out,
                                        const hipattn_tensor *query,
                                        const hipattn_tensor *key_cache,
                                        const hipattn_tensor *value_cache,
                                        int num_kv_heads, float scale,
                                        const hipattn_tensor *block_tables,
                                        const hipattn_tensor *context_lens,
                                        int block_size, int max_context_len,
                                        const hipattn_tensor *alibi_slopes,
                                        void *stream);

/* Optional set-up for the current device: everything the decode entry points
 * would otherwise ask the runtime on their first call (the address of the
 * built-in scratch array, kernel occupancy).  Allocates nothing; safe to call
 * more than once. */
char *hipattn_init(void);

/* Scratch bytes hipattn_paged_attention_v1* needs on the current device for
 * num_seqs sequences of at most max_context_len tokens (0 when the call needs
 * none).  Depends on the shapes only, not on the context lengths of a step. */
char *hipattn_paged_attention_workspace_size(int64_t num_seqs, int num_heads,
                                             int num_kv_heads, int head_size,
                                             int block_size,
                                             int max_context_len, int32_t dtype,
                                             int64_t *bytes);

/* hipattn_paged_attention_v1 with a sliding window and sinks: the token of a sequence of ctx tokens sees key t iff t < ctx and
 * (t >= ctx - 1 - window_size_left or t < sink_tokens).  No counterpart in tch-cuda.  Reads those keys alone: table columns between the
 * sinks and the window may name any block or none, and their blocks hold anything.  f16 and bf16 caches, head sizes 64, 80, 96, 112, 128
 * and 256, block sizes 8, 16 and 32; window_size_left >= 0, sink_tokens >= 0; arguments else as for hipattn_paged_attention_v1.
 * workspace: u8, 256-byte aligned, hipattn_paged_attention_window_workspace_size bytes -- a function of the shapes, max_context_len, the
 * window and the sinks -- or NULL for a buffer that the library keeps per stream, with what hipattn_paged_attention_v1 says about captures,
 * threads and overlapping calls. */
char *hipattn_paged_attention_window(hipattn_tensor *out, const hipattn_tensor *query,
                                     const hipattn_tensor *key_cache, const hipattn_tensor *value_cache,
                                     int num_kv_heads, float scale, const hipattn_tensor *block_tables,
                                     const hipattn_tensor *context_lens, int block_size, int max_context_len,
                                     int window_size_left, int sink_tokens, const hipattn_tensor *alibi_slopes,
                                     const hipattn_tensor *workspace, void *stream);
char *hipattn_paged_attention_window_workspace_size(int64_t num_seqs, int num_heads, int num_kv_heads,
                                                    int head_size, int block_size, int max_context_len,
                                                    int window_size_left, int sink_tokens, int32_t dtype,
                                                    int64_t *bytes);

/* Replaces paged_attention_v2_C (lib.rs:122-137; attention_kernels.cu:421-546,
 * 729-874).  Same as v1 with caller-provided split-K workspaces: exp_sums and
 * max_logits f32 [S, Hq, P], tmp_out [S, Hq, P, d] in the cache dtype.  The
 * partition length is ceil(max_context_len / P) rounded up to a multiple of 32
 * tokens, so a caller that sizes P for the reference's 512-token partitions
 * gets 512-token partitions (other block sizes and f32: a multiple of the
 * block size, at most 8192 tokens). */
char *hipattn_paged_attention_v2(
    hipattn_tensor *out, hipattn_tensor *exp_sums, hipattn_tensor *max_logits,
    hipattn_tensor *tmp_out, const hipattn_tensor *query,
    const hipattn_tensor *key_cache, const hipattn_tensor *value_cache,
    int num_kv_heads, float scale, const hipattn_tensor *block_tables,
    const hipattn_tensor *context_lens, int block_size, int max_context_len,
    const hipattn_tensor *alibi_slopes, void *stream);

/* ---------------------------------------------------------------------------
 * KV-cache data movement (bit-exact)
 * ------------------------------------------------------------------------- */

/* Replaces reshape_and_cache_C (lib.rs:168-174; cache_kernels.cu:168-253).
 * key/value [T, Hkv, d]; slot_mapping int64 (int32 accepted) [T]; slot < 0
 * skips the token. */
char *hipattn_reshape_and_cache(const hipattn_tensor *key,
                                const hipattn_tensor *value,
                                hipattn_tensor *key_cache,
                                hipattn_tensor *value_cache,
                                const hipattn_tensor *slot_mapping,
                                void *stream);

/* Replaces gather_cached_kv_C (lib.rs:176-182; cache_kernels.cu:301-413).
 * slot_mapping int32 (int64 accepted) [T]. */
char *hipattn_gather_cached_kv(hipattn_tensor *key, hipattn_tensor *value,
                               const hipattn_tensor *key_cache,
                               const hipattn_tensor *value_cache,
                               const hipattn_tensor *slot_mapping,
                               void *stream);

/* Replaces copy_blocks_2_C (lib.rs:184-189; cache_kernels.cu:55-81,141-163).
 * key_cache_ptrs/value_cache_ptrs: int64 [layers] device arrays of cache base
 * addresses; block_mapping int64 [2*pairs] (src,dst,...); key0: the first
 * layer's key cache (gives dtype and elements per block). */
char *hipattn_copy_blocks_2(const hipattn_tensor *key_cache_ptrs,
                            const hipattn_tensor *value_cache_ptrs,
                            const hipattn_tensor *block_mapping,
                            const hipattn_tensor *key0, void *stream);

/* The same from host arrays: the caches' base addresses of every layer and the
 * (src,dst) pairs are read before the call returns and travel as arguments of
 * the launches (64 layers x 256 pairs each), so that no upload goes in front
 * of the copy and the call may be captured.  Caches must start on 16-byte
 * boundaries, bytes_per_block be a multiple of 16 (at most 64 MiB) and block
 * numbers lie between 0 and what 32 bits hold; a negative one is refused before
 * any launch.  That they lie within the caches is the caller's to see to: the
 * call does not know how many blocks there are. */
char *hipattn_copy_blocks_host(void *const *key_caches, void *const *value_caches,
                               int64_t layers, const int64_t *block_mapping,
                               int64_t n_pairs, int64_t bytes_per_block,
                               void *stream);

/* Replaces swap_blocks (cache_kernels.cu:12-50; the Rust wrapper is a stub,
 * lib.rs:236-243).  src/dst are whole caches of equal block shape; direction
 * is given by where each lives (0 = host, 1 = device); block_mapping is a host
 * array of n_pairs (src,dst) int64 pairs; one hipMemcpyAsync per pair. */
char *hipattn_swap_blocks(const hipattn_tensor *src, int src_on_device,
                          hipattn_tensor *dst, int dst_on_device,
                          const int64_t *block_mapping, int64_t n_pairs,
                          void *stream);

/* ---------------------------------------------------------------------------
 * Positional encoding, normalisation, activations
 * ------------------------------------------------------------------------- */

/* Replaces rotary_embedding_C (lib.rs:153-160; pos_encoding_kernels.cu:9-128).
 * positions int64 (int32 accepted) [T]; query [T, Hq*d], key [T, Hkv*d] rotated
 * in place (row stride honoured); cos_sin_cache [max_pos, rot_dim] in the
 * query dtype.  Arithmetic rounds to the tensor dtype after every operation,
 * like the reference kernel (pos_encoding_kernels.cu:33-36). */
char *hipattn_rotary_embedding(const hipattn_tensor *positions,
                               hipattn_tensor *query, hipattn_tensor *key,
                               int head_size,
                               const hipattn_tensor *cos_sin_cache,
                               bool is_neox, void *stream);

/* hipattn_rotary_embedding followed by hipattn_reshape_and_cache of the same
 * keys, in one launch: what a layer does with a step's new tokens
 * (llm/mod.rs:88-114 then 147-164).  No counterpart in the reference's FFI;
 * same results as the two calls, bit for bit.  query [T, Hq*d] and key
 * [T, Hkv*d] are rotated in place, the rotated keys and value [T, Hkv, d] go to
 * the slots of slot_mapping (int64 or int32; negative = not cached).  NeoX
 * layout on a 2-byte type takes the fused kernel; anything else runs the two
 * calls one after the other. */
char *hipattn_rotary_embedding_and_cache(
    const hipattn_tensor *positions, hipattn_tensor *query, hipattn_tensor *key,
    const hipattn_tensor *value, int head_size,
    const hipattn_tensor *cos_sin_cache, bool is_neox,
    hipattn_tensor *key_cache, hipattn_tensor *value_cache,
    const hipattn_tensor *slot_mapping, void *stream);

/* Replaces rms_norm_C (lib.rs:139-144; layernorm_kernels.cu:10-35,69-92). */
char *hipattn_rms_norm(hipattn_tensor *out, const hipattn_tensor *input,
                       const hipattn_tensor *weight, float epsilon,
                       void *stream);

/* Replaces fused_add_rms_norm_C (lib.rs:146-151; layernorm_kernels.cu:38-117):
 * residual += input; input = rms_norm(residual) * weight. */
char *hipattn_fused_add_rms_norm(hipattn_tensor *input,
                                 hipattn_tensor *residual,
                                 const hipattn_tensor *weight, float epsilon,
                                 void *stream);

/* The residual addition and the norm behind it (llama.rs:166 + 169, 173 + 165) as the two calls round them: input = T(input + residual),
 * out = rms_norm(input) * weight, the variance that of the rounded sum (hipattn_fused_add_rms_norm takes the unrounded one).
 * [rows, hidden] f16 or bf16, contiguous, on 16-byte boundaries, hidden a multiple of 8, at most 8192; input must not share memory with
 * the others. */
char *hipattn_add_rms_norm(hipattn_tensor *out, hipattn_tensor *input,
                           const hipattn_tensor *residual,
                           const hipattn_tensor *weight, float epsilon,
                           void *stream);

/* A linear layer applied to at most 128 rows: out = x . weight^T (+ bias)
 * (+ residual), the projections of a generation step.  Replaces the
 * `nn::Linear::forward` calls that rLLM makes through `linear_no_bias` /
 * `linear` (rllm/rllm-cuda/src/llm/mod.rs:401-416): llama.rs:81-83, 96,
 * 135-143, 210 and phi.rs:73-75, 99, 131, 147, which reach at::linear through
 * the tch crate rather than through the reference's own extern "C" block.
 * x [M, K] (row stride honoured, e.g. a slice of a wider activation), weight
 * [N, K] in the layout of a checkpoint (row stride honoured), bias [N] or
 * NULL, residual [M, N] or NULL (row stride honoured), out [M, N]; f16 or
 * bf16 throughout; M <= 128, K a multiple of 256, N a multiple of 16, rows of
 * x and weight on 16-byte boundaries -- anything else is refused with a
 * message (a caller then uses a library GEMM, as it does for the rows of a
 * prompt).  Rounding: fp32 sums over K, + bias in fp32, rounded to the data
 * type; with a residual, that value + residual rounded again (the separate
 * addition of llama.rs:166, 173).  The same bits on every run.  When weight has
 * too few rows to occupy the device the inner dimension is split, and from 17
 * rows of x on a second launch adds the parts, in fp32, from `workspace` (u8,
 * hipattn_linear_workspace_size bytes: a function of weight alone, 0 when no
 * split is needed, so that a buffer sized with any number of rows serves every
 * other) or, when that is NULL, from a scratch buffer that the library keeps
 * per stream (with what hipattn_paged_attention_v1 says about captures and
 * overlapping calls).  Up to 16 rows take one launch and no workspace.  out
 * may lie over x, in this call and in the two below: the sums then go through
 * the workspace whatever the shape (splits x 128 x N x 4 bytes; a caller's own
 * that is smaller is refused). */
char *hipattn_linear(hipattn_tensor *out, const hipattn_tensor *x,
                     const hipattn_tensor *weight, const hipattn_tensor *bias,
                     const hipattn_tensor *residual,
                     const hipattn_tensor *workspace, void *stream);
char *hipattn_linear_workspace_size(const hipattn_tensor *x,
                                    const hipattn_tensor *weight,
                                    int64_t *bytes);

/* hipattn_linear with silu_and_mul behind it (llama.rs:135-142): weight [2 n, K] holds the gate rows and then
 * the up rows, out [M, n] = silu_and_mul(x . weight^T), the bits of the two calls; the [M, 2 n] product is not
 * written to memory.  Workspace: hipattn_linear_workspace_size of the same x and weight. */
char *hipattn_linear_silu_and_mul(hipattn_tensor *out, const hipattn_tensor *x,
                                  const hipattn_tensor *weight,
                                  const hipattn_tensor *workspace, void *stream);

/* hipattn_linear followed by the RMS norm of the finished rows, from 17 rows of
 * x on (and for rows of out or norm_out that lie apart) in the launch that adds
 * up the ranges of the inner dimension, below in a launch of its own: out = x . weight^T (+ bias) (+ residual) as above, norm_out = rms_norm(out, norm_weight, epsilon) with the
 * arithmetic of hipattn_rms_norm -- the same bits as the two calls one after
 * the other.  It is the pair that closes every residual branch of the decoder
 * (llama.rs:166 + 169, 173 + 165 of the next block, 173 + 207), with no
 * counterpart of its own in the reference's extern "C" block.  Operands as
 * for hipattn_linear, and: N a multiple of 8, at most 8192; norm_weight [N],
 * norm_out [M, N]; rows of out, norm_out and residual on 16-byte boundaries.
 * The workspace (hipattn_linear_rms_norm_workspace_size bytes, a function of
 * weight alone, or the library's per-stream scratch when NULL) is used
 * whatever the weight, from 17 rows of x on and for rows that lie apart. */
char *hipattn_linear_rms_norm(hipattn_tensor *out, hipattn_tensor *norm_out,
                              const hipattn_tensor *x,
                              const hipattn_tensor *weight,
                              const hipattn_tensor *bias,
                              const hipattn_tensor *residual,
                              const hipattn_tensor *norm_weight, float epsilon,
                              const hipattn_tensor *workspace, void *stream);
char *hipattn_linear_rms_norm_workspace_size(const hipattn_tensor *x,
                                             const hipattn_tensor *weight,
                                             int64_t *bytes);

/* hipattn_rms_norm of the rows of x and the linear layer behind it (llama.rs:165 + 81-83, 169 + 135-142) in one launch, for the few
 * rows that a workgroup can hold: out = rms_norm(x, norm_weight, epsilon) . weight^T, or with silu_and_mul as in
 * hipattn_linear_silu_and_mul; the bits of the two calls; the normalised rows are not written to memory.  Operands as for
 * hipattn_linear, and: x at most HIPATTN_RMS_NORM_LINEAR_ROWS rows of at most 8192 (rows and norm_weight together at most 40 KB),
 * fewer than 65536 rows of weight, norm_weight [K] on a 16-byte boundary, out not over x.  No workspace. */
#define HIPATTN_RMS_NORM_LINEAR_ROWS 4
char *hipattn_rms_norm_linear(hipattn_tensor *out, const hipattn_tensor *x,
                              const hipattn_tensor *norm_weight, float epsilon,
                              const hipattn_tensor *weight, bool silu_and_mul,
                              void *stream);

/* The projection of q, k and v with hipattn_rotary_embedding_and_cache (NeoX) behind it (llama.rs:81-85 + mod.rs:147-164), for the
 * rows of a small step: out [M, (Hq + 2 Hkv) d] = x . weight^T, query and key heads rotated, the keys and values written to the cache;
 * the bits of the calls, and the calls themselves where d does not divide 128 and hipattn_linear turns the weight's ranges.  With norm_weight not NULL hipattn_rms_norm of the rows of x comes first, as in hipattn_rms_norm_linear and
 * within its limits.  d and Hkv are the cache's; d a multiple of 16, cos_sin_cache [positions, d]; fewer than 65536 rows of weight, and
 * than 16384 with more than 16 rows of x; operands else, and scratch, as for hipattn_linear and hipattn_rotary_embedding_and_cache. */
char *hipattn_qkv_linear(hipattn_tensor *out, const hipattn_tensor *x,
                         const hipattn_tensor *norm_weight, float epsilon,
                         const hipattn_tensor *weight,
                         const hipattn_tensor *positions,
                         const hipattn_tensor *cos_sin_cache,
                         hipattn_tensor *key_cache, hipattn_tensor *value_cache,
                         const hipattn_tensor *slot_mapping, void *stream);

/* Replace silu_and_mul_C / gelu_new_C / gelu_fast_C (lib.rs:162-166;
 * activation_kernels.cu:15-115). */
char *hipattn_silu_and_mul(hipattn_tensor *out, const hipattn_tensor *input,
                           void *stream);
char *hipattn_gelu_new(hipattn_tensor *out, const hipattn_tensor *input,
                       void *stream);
char *hipattn_gelu_fast(hipattn_tensor *out, const hipattn_tensor *input,
                        void *stream);

/* ---------------------------------------------------------------------------
 * AICI logit-mask step
 * ------------------------------------------------------------------------- */

/* The bias-add + greedy pick that rLLM performs per sequence
 * (rllm-cuda/src/llm/tmodel.rs:277-283 `TchAiciBias::apply`, :234-236
 * `sample_argmax`) for all rows in one launch.  logits [S, V] (f32/f16/bf16).
 * Exactly one of bias / mask is non-NULL:
 *   bias: f32 [R, Vb] rows as produced by aicirt (0 / -inf, Vb >= V);
 *   mask: u8 [R, mask_bytes] packed allow-bits, bit k of byte i (LSB first) is
 *         token 8*i+k, set = allowed (aicirt/src/api.rs:278-292); tokens past
 *         8*mask_bytes are disallowed.
 * bias_rows int32 [S] or NULL selects the row for each sequence (identity when
 * NULL).  out_tokens int32 [S]; out_logits f32 [S] or NULL receives the
 * winning biased logit.  Ties resolve to the lowest token id.
 * For large vocabularies the call keeps a few bytes of state per row in a
 * library-owned buffer that belongs to the stream it runs on (cleared by the
 * call itself, so no call depends on an earlier one).  Calls that share that
 * buffer must not overlap: a graph captured from this call replays onto the
 * buffer of the stream it was captured on, so two replays of such graphs on
 * different streams at once, or a replay beside eager calls on the capture
 * stream, give wrong tokens for the overlapping calls (never for later ones). */
char *hipattn_bias_argmax(const hipattn_tensor *logits,
                          const hipattn_tensor *bias,
                          const hipattn_tensor *mask,
                          const hipattn_tensor *bias_rows,
                          hipattn_tensor *out_tokens,
                          hipattn_tensor *out_logits, void *stream);

/* Penalties for what a sequence has said, bias and allow-mask on the logits of all rows, in front of hipattn_bias_argmax /
 * hipattn_bias_sample (rLLM applies the bias alone, tmodel.rs:277-283):
 *   x = logits; a token that the sequence holds: x = x > 0 ? x / repetition : x * repetition;
 *   x -= frequency * count + presence * (count > 0), count: how often the token stands behind the prompt; x += bias; not allowed: x = -inf.
 * history int32 [N]: the tokens of all sequences one after the other, sequence s those from history_offsets[s] (int64 or int32 [S + 1]) on,
 * the first prompt_lens[s] (int32 [S] or NULL: none) of them its prompt; tokens outside the vocabulary count for nothing.  repetition,
 * frequency, presence f32 [S], NULL: 1, 0, 0.  bias f32 rows, mask packed allow-bits and bias_rows as for hipattn_bias_argmax, but any of
 * them, both or none.  out [S, V] in the type of logits or f32, rounded once from fp32; it may be logits itself (same type and strides)
 * and lies over no other input. */
char *hipattn_penalize_logits(hipattn_tensor *out, const hipattn_tensor *logits, const hipattn_tensor *history,
                              const hipattn_tensor *history_offsets, const hipattn_tensor *prompt_lens,
                              const hipattn_tensor *repetition, const hipattn_tensor *frequency,
                              const hipattn_tensor *presence, const hipattn_tensor *bias,
                              const hipattn_tensor *mask, const hipattn_tensor *bias_rows, void *stream);

/* Bias + temperature + nucleus (top-p) sampling for all rows in one call:
 * `TchAiciBias::apply` followed by `TModel::sample` / `sample_topp` /
 * `sample_multinomial` (rllm-cuda/src/llm/tmodel.rs:277-283, 172-194, 236-268),
 * which the reference runs per sequence on the host side of a device sync.
 * logits, bias / mask and bias_rows as for hipattn_bias_argmax.  temperature,
 * top_p, uniforms: f32 [S].  A row whose temperature is below 1e-5 (the
 * reference's SAMPLING_EPS) takes the arg-max.  Otherwise p = softmax((logits
 * + bias) / temperature) in f32; with 0 < top_p < 1 tokens are taken in
 * descending order of p (equal values by ascending id) and kept while the mass
 * of those before them is below top_p, the others get weight 0; the token
 * returned is the first whose cumulative weight in id order exceeds
 * uniforms[s] * (sum of weights), which is what rand's WeightedIndex returns
 * for that draw.  uniforms[s] in [0, 1) comes from the caller, who keeps the
 * random generators (one per sequence in the reference); values outside are
 * clamped.  A token with bias -inf is never drawn, whatever the temperature.
 * A row that holds +inf (where the reference's softmax has no answer) yields
 * the first such token, a row with nothing allowed token 0.
 * out_tokens int32 [S].
 * bf16 rows of 24576 to 262144 tokens under a mask are read by several
 * workgroups each, which leave their counts in a buffer of the library's that
 * belongs to the stream (38 MB from the first such call on, kept until
 * hipattn_shutdown).  While the stream
 * is being captured, or without memory for the buffer, one workgroup reads the
 * row, as for other rows: the same tokens. */
char *hipattn_bias_sample(const hipattn_tensor *logits,
                          const hipattn_tensor *bias,
                          const hipattn_tensor *mask,
                          const hipattn_tensor *bias_rows,
                          const hipattn_tensor *temperature,
                          const hipattn_tensor *top_p,
                          const hipattn_tensor *uniforms,
                          hipattn_tensor *out_tokens, void *stream);

/* ---------------------------------------------------------------------------
 * Device runtime plumbing
 * ------------------------------------------------------------------------- */

/* Mirror `Stats` / `CudaProps` (lib.rs:393-411; cuda.cpp:17-30). */
typedef struct hipattn_mem_stats {
  int64_t current;
  int64_t peak;
  int64_t allocated;
  int64_t freed;
} hipattn_mem_stats;

typedef struct hipattn_device_props {
  int32_t major;
  int32_t minor;
  int32_t multi_processor_count;
  int32_t max_threads_per_multi_processor;
  int64_t total_memory;
} hipattn_device_props;

/* Replace cuda_reset_peak_memory_stats_C / cuda_empty_cache_C /
 * cuda_get_stats_allocated_bytes_C / cuda_get_device_properties_C
 * (cuda.cpp:34-60).  Without a caching allocator the figures come from
 * hipMemGetInfo: current = total - free on the device, peak = the largest
 * `current` seen by any stats call since the last reset; allocated / freed =
 * the bytes of scratch memory this library itself has allocated on the device
 * and released again (hipattn_shutdown) since it was loaded. */
char *hipattn_reset_peak_memory_stats(int device);
char *hipattn_empty_cache(void); /* nothing to release: no caching allocator; see hipattn_shutdown */
char *hipattn_get_stats_allocated_bytes(int device, hipattn_mem_stats *outp);
char *hipattn_get_device_properties(int device, hipattn_device_props *outp);

typedef struct hipattn_stream hipattn_stream;
typedef struct hipattn_event hipattn_event;

#define HIPATTN_STREAM_DEFAULT 0
#define HIPATTN_STREAM_CURRENT 1
#define HIPATTN_STREAM_HIGH_PRI 2
#define HIPATTN_STREAM_LOW_PRI 3

/* Replace cuda_stream_*_C (cuda.cpp:62-107; stream.rs:18-28).  Pool streams
 * (HIGH_PRI / LOW_PRI) are new non-blocking streams at the default priority. */
char *hipattn_stream_get(int typ, int device, hipattn_stream **outp);
char *hipattn_stream_free(hipattn_stream *s);
char *hipattn_stream_clone(hipattn_stream *s, hipattn_stream **outp);
char *hipattn_stream_query(hipattn_stream *s, int *done);
char *hipattn_stream_synchronize(hipattn_stream *s);
char *hipattn_stream_set_current(hipattn_stream *s);
char *hipattn_stream_device_index(hipattn_stream *s, int *id);
char *hipattn_stream_id(hipattn_stream *s, int64_t *id);
/* The raw hipStream_t, to pass as an op's `stream` argument. */
char *hipattn_stream_raw(hipattn_stream *s, void **raw);

/* Replace cuda_event_*_C (cuda.cpp:113-147; event.rs:12-28). */
char *hipattn_event_create(bool timing, bool blocking, hipattn_event **outp);
char *hipattn_event_record(hipattn_event *e, hipattn_stream *s);
char *hipattn_event_block(hipattn_event *e, hipattn_stream *s);
char *hipattn_event_elapsed_time(hipattn_event *e, hipattn_event *e2,
                                 float *elapsed_ms);
char *hipattn_event_query(hipattn_event *e, int *done);
char *hipattn_event_synchronize(hipattn_event *e);
char *hipattn_event_free(hipattn_event *e);

/* Releases the scratch buffers the library owns, on every device, after
 * waiting for the devices to drain.  Graphs captured from calls that used them
 * must not be replayed afterwards. */
char *hipattn_shutdown(void);

/* Switches for tuning and for tests that want one particular kernel.  Each is
 * read from the environment once, when the library is loaded (HIPATTN_ + the
 * name in capitals); ops never read the environment.  Names: decode_flat
 * (-1 library's choice, 0 partitioned launch, 1 flat split), decode_flat_wgs
 * (0 = what the device holds at once), decode_part_blocks (0 = chosen per
 * call, else 2..64), prefill_kernel (0 library's choice, 1 workgroups of eight
 * wavefronts, 5 the same kernel in workgroups of four -- the bits of 1 -- 2 / 3
 * another of four wavefronts with 2 / 1 row tiles, 4 three groups of four
 * wavefronts; what a kernel does not cover, the one that does takes),
 * paged_prefill_dma (-1 library's
 * choice, 0 staged tiles), cache_move_lds (-1 library's choice, 0 never the
 * LDS-transposing kernels), prefill_wg_heads (query heads of one kv group per
 * workgroup of prefill_kernel 1 and, up to four, 5, at most; 0 library's
 * choice -- up to four -- 1: one),
 * prefill_rescale_log2 (0..16, default 8: the prefill
 * kernels move a row's reference maximum only when the row outgrows it by
 * more than 2^value; 0 follows the row maximum exactly, as the reference
 * does), window_parts (prefill over a window: 0 library's choice, else the
 * number of workgroups, at most 16, that a row block's keys are dealt out to
 * where there is a merge for the head size), linear_tiles (0 library's choice,
 * 1 / 2: workgroups of 64 / 128 rows of the weight in hipattn_linear), linear_splits (0 library's choice, else
 * the number of ranges the inner dimension is cut into, at most 32).  Every
 * setting computes the same results -- prefill_kernel 2 to 4 (over a window any
 * but 0), prefill_rescale_log2, window_parts and linear_splits up to rounding.  Not
 * synchronised with running calls: set them between calls. */
char *hipattn_tuning_set(const char *name, int value);
char *hipattn_tuning_get(const char *name, int *value);

/* ---------------------------------------------------------------------------
 * Host side of the paged KV cache (no GPU needed)
 * ------------------------------------------------------------------------- */

typedef struct hipattn_block_allocator hipattn_block_allocator;

/* `BlockAllocator` (rllm-cuda/src/llm/paged/blocks.rs:32-257): free list seeded
 * (0..n).rev() and popped from the back, reference counts, fork / trim /
 * copy-on-write. */
char *hipattn_block_allocator_new(int64_t block_size, int64_t num_blocks,
                                  hipattn_block_allocator **outp);
void hipattn_block_allocator_free(hipattn_block_allocator *a);
int64_t hipattn_block_allocator_num_free(const hipattn_block_allocator *a);
/* blocks.rs:157-165 (number of blocks held by seq; 0 if unknown). */
int64_t hipattn_block_allocator_num_allocated(const hipattn_block_allocator *a,
                                              int64_t seq_id);
/* blocks.rs:167-176 `alloc_seq`. */
char *hipattn_block_allocator_alloc_seq(hipattn_block_allocator *a,
                                        int64_t seq_id, int64_t seq_len);
/* blocks.rs:213-243 `append_slots`: grows seq to seq_len tokens, replacing
 * shared blocks at or after num_kv_computed by fresh ones.  Each replacement
 * appends (old,new) to copy_pairs (capacity max_pairs pairs); *n_pairs
 * receives the count. */
char *hipattn_block_allocator_append_slots(hipattn_block_allocator *a,
                                           int64_t seq_id,
                                           int64_t num_kv_computed,
                                           int64_t seq_len, int64_t *copy_pairs,
                                           int64_t max_pairs, int64_t *n_pairs);
/* blocks.rs:245-256 `copy` (fork src's first `length` tokens into dst),
 * `trim`, `delete`. */
char *hipattn_block_allocator_copy(hipattn_block_allocator *a, int64_t src,
                                   int64_t dst, int64_t length);
char *hipattn_block_allocator_trim(hipattn_block_allocator *a, int64_t seq_id,
                                   int64_t length);
char *hipattn_block_allocator_delete(hipattn_block_allocator *a,
                                     int64_t seq_id);
/* blocks.rs:152-155 `get_block_idxes`: slot of every position < len. */
char *hipattn_block_allocator_get_block_idxes(const hipattn_block_allocator *a,
                                              int64_t seq_id, int64_t len,
                                              int64_t *out_slots);

/* blocks.rs:176-189 `swap_out`: copies the sequence's physical block numbers
 * (logical order) to out_blocks and releases them.  With out_blocks == NULL
 * only *n_out is set (nothing is released).
 * blocks.rs:191-210 `swap_in`: one block of this allocator per entry of
 * block_idxs (blocks of the other allocator); `mapping` holds *n_pairs pairs
 * (other-side block, this-side block) and is shared by the sequences of a
 * group: an already mapped block is forked, new pairs are appended. */
char *hipattn_block_allocator_swap_out(hipattn_block_allocator *a,
                                       int64_t seq_id, int64_t *out_blocks,
                                       int64_t capacity, int64_t *n_out);
char *hipattn_block_allocator_swap_in(hipattn_block_allocator *a,
                                      int64_t seq_id,
                                      const int64_t *block_idxs, int64_t n,
                                      int64_t *mapping, int64_t pair_capacity,
                                      int64_t *n_pairs);

/* Admission policy of `BlockSpaceManager` over the GPU allocator
 * (blocks.rs:260-283, 321-343): `watermark_blocks = (watermark * num_blocks) as
 * usize` blocks are held back from new sequences so that running ones can keep
 * growing.  can_allocate: a new sequence of seq_len tokens fits on top of the
 * watermark (`can_allocate`, :267-270); can_append_slot: one free block per
 * running sequence (`can_append_slot`, :278-282).  Both return 0 / 1. */
char *hipattn_block_allocator_set_watermark(hipattn_block_allocator *a,
                                            float watermark);
int hipattn_block_allocator_can_allocate(const hipattn_block_allocator *a,
                                         int64_t seq_len);
int hipattn_block_allocator_can_append_slot(const hipattn_block_allocator *a,
                                            int64_t num_running_seqs);

typedef struct hipattn_batch_builder hipattn_batch_builder;

/* What `BatchInfoBuilder::finish` produces (batch_info.rs:18-43,196-315).  All
 * arrays are host memory owned by the builder, valid until the next finish()
 * or free(). */
typedef struct hipattn_batch_info {
  int64_t num_tokens;
  const int32_t *tokens;       /* [num_tokens] */
  const int64_t *positions;    /* [num_tokens] */
  const int32_t *slot_mapping; /* [num_tokens] */
  int64_t num_seqs;
  const int32_t *logit_idxs; /* [num_seqs] */
  const int64_t *seq_ids;    /* [num_seqs] entry order after multi-first sort */
  int64_t num_multi;         /* seqlen_multi: entries on the varlen path */
  const int32_t *seqlens_q;  /* [num_multi+1] offsets (kernels.rs:10-21) */
  const int32_t *seqlens_k;  /* [num_multi+1] */
  int64_t max_seqlen_q;
  int64_t max_seqlen_k;
  int64_t num_gather;
  const int32_t *gather_mapping; /* [num_gather] */
  int64_t q_multi;               /* tokens belonging to multi-token entries */
  int64_t num_paged;             /* single-token entries */
  int64_t paged_max_blocks;
  const int32_t *paged_block_tables; /* [num_paged, paged_max_blocks] 0-padded */
  const int32_t *paged_context_lens; /* [num_paged] */
  int64_t paged_block_size;
  int64_t paged_max_context_len;
  /* Extension (not in batch_info.rs): block tables and key counts of the
   * multi-token entries, for hipattn_mha_varlen_fwd_paged.  multi_tables_valid
   * is 1 when every multi-token entry's slots follow its blocks in order
   * (slot(p) = table[p / BS] * BS + p % BS, which is how blocks.rs:122-127 hands
   * them out); otherwise 0 and the gather route must be used. */
  int32_t multi_tables_valid;
  int64_t multi_max_blocks;
  const int32_t *multi_block_tables; /* [num_multi, multi_max_blocks] 0-padded */
  const int32_t *multi_context_lens; /* [num_multi] */
} hipattn_batch_info;

/* paged_attn_kernel_v > 0 sends single-token entries to the paged kernel
 * (sorted to the back); 0 keeps every entry on the varlen path, as CPU builds
 * do (rllm-cuda/src/llm/config.rs:155-158). */
char *hipattn_batch_builder_new(int64_t block_size, int64_t max_model_len,
                                int paged_attn_kernel_v,
                                hipattn_batch_builder **outp);
void hipattn_batch_builder_free(hipattn_batch_builder *b);
/* One `BatchEntry` (batch_info.rs:109-113,141-148): the query tokens with
 * their positions, and the slot of every token of the sequence. */
char *hipattn_batch_builder_add(hipattn_batch_builder *b, int64_t seq_id,
                                const int64_t *query_positions,
                                const int32_t *query_tokens, int64_t q_len,
                                const int64_t *kv_slots, int64_t k_len);
/* `sched_out` for one running sequence (batch_info.rs:115-152): q_len =
 * seq_len - num_kv_computed (1 if that is 0), slots from the allocator. */
char *hipattn_batch_builder_add_seq(hipattn_batch_builder *b,
                                    const hipattn_block_allocator *a,
                                    int64_t seq_id, const int32_t *seq_tokens,
                                    int64_t seq_len, int64_t num_kv_computed);
char *hipattn_batch_builder_finish(hipattn_batch_builder *b,
                                   hipattn_batch_info *outp);

/* The single-token rows of a running batch, kept across steps.  No counterpart
 * in the reference, whose BatchInfoBuilder::finish rebuilds every vector from
 * the sequences' full slot lists at every step (batch_info.rs:196-315,
 * blocks.rs:152-155: O(sum of contexts)); between two generation steps a running
 * sequence only gains one token, which costs O(1) here.  hipattn_decode_batch_info
 * hands out what finish() would for the same sequences in the same order
 * (num_multi = 0), value for value.  Rows keep the order in which they were
 * added.
 *   add:     a sequence of seq_len tokens whose last token is last_token and is
 *            the one to be computed (the others are in the cache); the
 *            allocator holds its blocks.
 *   advance: the sequence gained new_token (the allocator's append_slots for
 *            the longer sequence has been called).
 *   remove:  the sequence left the batch (finished, preempted, swapped out). */
typedef struct hipattn_decode_batch hipattn_decode_batch;
char *hipattn_decode_batch_new(int64_t block_size, int64_t max_model_len,
                               hipattn_decode_batch **outp);
void hipattn_decode_batch_free(hipattn_decode_batch *b);
int64_t hipattn_decode_batch_size(const hipattn_decode_batch *b);
char *hipattn_decode_batch_add(hipattn_decode_batch *b,
                               const hipattn_block_allocator *a, int64_t seq_id,
                               int32_t last_token, int64_t seq_len);
char *hipattn_decode_batch_advance(hipattn_decode_batch *b,
                                   const hipattn_block_allocator *a,
                                   int64_t seq_id, int32_t new_token);
/* advance for every row at once: new_tokens[i] goes to row i (n = rows). */
char *hipattn_decode_batch_advance_all(hipattn_decode_batch *b,
                                       const hipattn_block_allocator *a,
                                       const int32_t *new_tokens, int64_t n);
char *hipattn_decode_batch_remove(hipattn_decode_batch *b, int64_t seq_id);
/* Arrays are owned by the batch and valid until its next change. */
char *hipattn_decode_batch_info(hipattn_decode_batch *b,
                                hipattn_batch_info *outp);

/* One generation step's block bookkeeping with preemption by recomputation,
 * for sequence groups of one sequence: Scheduler::step_generation + _preempt
 * (rllm-base/src/scheduler.rs:304-337, 357-380) over can_append_slot /
 * append_slots (blocks.rs:278-286).  seq_ids in arrival order (earliest
 * first), seq_lens the lengths to grow to, num_kv_computed as for
 * append_slots.  Sequences are served earliest first; while no block is free
 * the latest arrival not yet served is preempted -- its blocks are released
 * (seq.rs:115-125) and it must be admitted and recomputed later -- and when
 * nobody else is left the sequence itself is preempted and the walk stops.
 * scheduled / preempted (capacity n each) receive the ids in the order of
 * events, copy_pairs the copy-on-write pairs of all append_slots calls. */
char *hipattn_block_allocator_step_generation(
    hipattn_block_allocator *a, const int64_t *seq_ids, const int64_t *seq_lens,
    const int64_t *num_kv_computed, int64_t n, int64_t *scheduled,
    int64_t *n_scheduled, int64_t *preempted, int64_t *n_preempted,
    int64_t *copy_pairs, int64_t max_pairs, int64_t *n_pairs);

/* The same step for sequence groups of any size over the two allocators of a
 * BlockSpaceManager (device `gpu`, host `cpu`): Scheduler::step_generation,
 * _append_slots and _preempt (rllm-base/src/scheduler.rs:304-337, 346-380)
 * over BlockSpaceManager::{can_append_slot, append_slots, can_swap_out,
 * swap_out} (rllm-cuda/src/llm/paged/blocks.rs:278-286, 307-322).
 *
 * Groups are given in arrival order (earliest first): group g owns sequences
 * group_start[g] .. group_start[g+1]-1 of the four sequence arrays
 * (group_start has n_groups+1 entries, the first 0); seq_phase holds
 * HIPATTN_SEQ_* (SchedulingPhase, seq.rs:44-51), seq_lens / num_kv_computed
 * are as for append_slots and read for running sequences only;
 * max_running_seqs[g] is the group's get_max_num_running_seqs()
 * (seq.rs:275-292), which picks the way it would be preempted.
 *
 * The walk: the earliest group not yet handled is served.  A group whose
 * sequences are all suspended or finished (seq.rs:324-328) is set aside --
 * HIPATTN_GROUP_SUSPENDED: it keeps its blocks and takes no part in the step.
 * Any other group goes on once one device block per running sequence is free
 * (needed or not); until then the latest arrival still queued, suspended or
 * not, is preempted, and with nobody queued the group itself, which ends the
 * walk.  A group that goes on has append_slots applied to each running
 * sequence (HIPATTN_GROUP_SCHEDULED; copy-on-write pairs are appended to
 * copy_pairs).  Preemption: max_running_seqs == 1 -> HIPATTN_GROUP_RECOMPUTE,
 * every sequence's blocks are released on both sides and the group has to be
 * admitted again (it is an error if one of its sequences has finished,
 * scheduler.rs:477); otherwise -> HIPATTN_GROUP_SWAPPED_OUT: the running
 * sequences' device blocks are released and each gets as many host blocks, a
 * block shared inside the group once; (device block, host block) pairs are
 * appended to swap_out_pairs for `CacheEngine::swap_out`.  The host must have
 * room for every block the group holds (can_swap_out) or the call fails with
 * the reference's message.
 *
 * group_fate[g] receives HIPATTN_GROUP_*.  On an error the allocators keep
 * what the walk did up to that point (the reference panics there);
 * group_fate, *n_copy_pairs and *n_swap_pairs describe it, groups not yet
 * handled read HIPATTN_GROUP_NOT_REACHED.
 *
 * Where the reference's text is not followed: its group-level swap_out hands
 * the sequence to the allocators the other way round (blocks.rs:310-313, which
 * trips the assert of blocks.rs:192 on any sequence that holds device blocks);
 * this moves device -> host, as the name and scheduler.rs:371-372 say.  Blocks
 * are released on recomputation whatever num_kv_computed is (the reference
 * skips the release at 0, seq.rs:116).  And groups set aside as suspended keep
 * that fate when the walk ends early (the reference drops its list of them on
 * that return, scheduler.rs:326-327). */
enum {
  HIPATTN_SEQ_RUNNING = 0,
  HIPATTN_SEQ_SUSPENDED = 1,
  HIPATTN_SEQ_SWAPPED = 2,
  HIPATTN_SEQ_WAITING = 3,
  HIPATTN_SEQ_FINISHED = 4
};
enum {
  HIPATTN_GROUP_NOT_REACHED = -1,
  HIPATTN_GROUP_SCHEDULED = 0,
  HIPATTN_GROUP_SUSPENDED = 1,
  HIPATTN_GROUP_RECOMPUTE = 2,
  HIPATTN_GROUP_SWAPPED_OUT = 3
};
char *hipattn_block_space_step_generation(
    hipattn_block_allocator *gpu, hipattn_block_allocator *cpu,
    int64_t n_groups, const int64_t *group_start,
    const int64_t *max_running_seqs, const int64_t *seq_ids,
    const int32_t *seq_phase, const int64_t *seq_lens,
    const int64_t *num_kv_computed, int32_t *group_fate, int64_t *copy_pairs,
    int64_t max_copy_pairs, int64_t *n_copy_pairs, int64_t *swap_out_pairs,
    int64_t max_swap_pairs, int64_t *n_swap_pairs);

/* The block bookkeeping of a step on the device, for sequences that share no blocks: what append_slots and the batch builder give on the
 * host, from device arrays alone, so that a step can be captured and replayed.  R requests (at most 4096), a pool of nb blocks.
 *   new_lens int32 [R]: tokens that request r brings; 0: it idles; negative: it has ended and its blocks go back.
 *   state int32 [R, 2]: its tokens in the cache, and the table columns in front of which everything but the sinks is gone.  state_out may
 *     be the same memory.
 *   block_tables int32 [R, cols] (rows may lie apart), updated in place: columns of blocks that are taken; the others stay as they are.
 *   free_ring int32 [nb]: the free blocks, in a ring: the next to be taken is free_ring[ring_ends[0] % nb], the place of the next that comes
 *     back free_ring[ring_ends[1] % nb] (int64 [2], both only grow; ring_ends_out may be the same memory).
 * Blocks go back first: those of ended requests and, with window_size_left >= 0, columns that hold only tokens in front of the window of
 * a request's next token and behind its sink_tokens; in the order of requests and columns.  Then requests are served in their order, as long
 * as the pool and the rows last: one that does not get all it needs gets nothing, nor do those behind it (served -1).  One whose tokens
 * exceed its table row, its rows or all rows is passed over (served -2).
 * rows_per_request 0: the rows of the T = positions' length lie one request behind the other, from seqlens_q[r] on; q > 0: request r has
 * rows q r .. q r + q - 1 whether it uses them or not (R q <= T).
 * Outputs: served int32 [R], the tokens given or the codes above; context_lens int32 [R]: keys of a request that is served, else 0;
 * seqlens_q int32 [R + 1]: sums of the tokens given; logit_idxs int32 [R]: a served request's last row, else 0; positions int64 [T] and
 * slot_mapping int32 [T], of rows without a token 0 and -1; totals int32 [4]: tokens given, requests not served (-1 and -2), blocks
 * free afterwards, blocks taken.  workspace int32 [4 (R + 1)], 16-byte aligned.  No output but the
 * two named lies over an input. */
char *hipattn_step_blocks(const hipattn_tensor *new_lens, const hipattn_tensor *state,
                          hipattn_tensor *block_tables, hipattn_tensor *free_ring,
                          const hipattn_tensor *ring_ends, int block_size, int rows_per_request,
                          int window_size_left, int sink_tokens, hipattn_tensor *state_out,
                          hipattn_tensor *ring_ends_out, hipattn_tensor *served, hipattn_tensor *context_lens,
                          hipattn_tensor *seqlens_q, hipattn_tensor *logit_idxs, hipattn_tensor *positions,
                          hipattn_tensor *slot_mapping, hipattn_tensor *totals, hipattn_tensor *workspace,
                          void *stream);

/* Cache geometry (`CacheEngine`, cache_engine.rs:81-100,165-175):
 * x = 16 / elt_size; key block [Hkv, d/x, BS, x], value block [Hkv, d, BS];
 * bytes per block over all layers = 2*BS*Hkv*d*elt*layers. */
int64_t hipattn_cache_x(int32_t dtype);
int64_t hipattn_cache_block_bytes(int64_t block_size, int64_t num_kv_heads,
                                  int64_t head_size, int64_t num_layers,
                                  int32_t dtype);

/* ---------------------------------------------------------------------------
 * Per-layer attention as rLLM composes it
 * ------------------------------------------------------------------------- */

/* `llm::varlen_attn` (rllm-cuda/src/llm/mod.rs:318-354): scatter all new K/V
 * into the cache, gather the context of multi-token sequences, run varlen
 * causal attention for the first q_multi rows and paged attention for the
 * rest; y [T, Hq, d] receives both parts in batch order.  Device inputs:
 * q [T,Hq,d], k/v [T,Hkv,d], slot_mapping int32|int64 [T], gather_mapping
 * int32 [G], seqlens_q/k int32 [num_multi+1], paged_block_tables,
 * paged_context_lens.  gather_k/gather_v [G, Hkv, d] are scratch for the
 * gathered context.  The GQA head mapping is done inside the kernels; no
 * repeat_kv copy (mod.rs:357-365) is made.  slot_mapping NULL = the new K/V are
 * in the cache already (hipattn_rotary_embedding_and_cache put them there) and
 * the scatter is skipped; the same holds for hipattn_varlen_attn_paged. */
char *hipattn_varlen_attn(
    const hipattn_tensor *q, const hipattn_tensor *k, const hipattn_tensor *v,
    hipattn_tensor *key_cache, hipattn_tensor *value_cache,
    const hipattn_tensor *slot_mapping, const hipattn_tensor *gather_mapping,
    const hipattn_tensor *seqlens_q, const hipattn_tensor *seqlens_k,
    int64_t q_multi, int max_seqlen_q, int max_seqlen_k,
    const hipattn_tensor *paged_block_tables,
    const hipattn_tensor *paged_context_lens, int paged_block_size,
    int paged_max_context_len, float softmax_scale, hipattn_tensor *gather_k,
    hipattn_tensor *gather_v, hipattn_tensor *y, void *stream);

/* The same composition without the gather copy: multi-token rows read their
 * context from the cache through multi_block_tables int32 [num_multi, cols] and
 * multi_context_lens int32 [num_multi] (hipattn_mha_varlen_fwd_paged).  No
 * counterpart in the reference, which always gathers (mod.rs:181-197).  Head
 * sizes up to 256.  Steps of f16 / bf16 over 16-token blocks with head sizes
 * 64, 80, 96, 112 or 128 take one launch for both kinds of rows and one that
 * merges partial results, where that is faster: its 64 MiB of scratch memory
 * are allocated once per stream.  Under capture, on hipStreamPerThread and
 * where there is no such memory the two go by themselves, as
 * hipattn_mha_varlen_fwd_paged and hipattn_paged_attention_v1 would, with the
 * latter's scratch memory, which an eager call on the stream allocates
 * whichever way it goes: one is all that a capture of the same shapes needs.
 * A replay's last bits may differ from the eager call's, whose keys are added
 * up in other pieces. */
char *hipattn_varlen_attn_paged(
    const hipattn_tensor *q, const hipattn_tensor *k, const hipattn_tensor *v,
    hipattn_tensor *key_cache, hipattn_tensor *value_cache,
    const hipattn_tensor *slot_mapping, const hipattn_tensor *multi_block_tables,
    const hipattn_tensor *seqlens_q, const hipattn_tensor *multi_context_lens,
    int64_t q_multi, int max_seqlen_q, int max_seqlen_k,
    const hipattn_tensor *paged_block_tables,
    const hipattn_tensor *paged_context_lens, int paged_block_size,
    int paged_max_context_len, float softmax_scale, hipattn_tensor *y,
    void *stream);

/* The same for a model with a sliding window and sinks: hipattn_reshape_and_cache (slot_mapping not NULL),
 * hipattn_mha_varlen_fwd_paged_window for the first q_multi rows, hipattn_paged_attention_window for the rest.  _ws: with a workspace for both, which
 * run one after the other -- the larger of their two sizes, or NULL -- so that a captured step is the eager one and shares no scratch memory. */
char *hipattn_varlen_attn_paged_window(
    const hipattn_tensor *q, const hipattn_tensor *k, const hipattn_tensor *v,
    hipattn_tensor *key_cache, hipattn_tensor *value_cache,
    const hipattn_tensor *slot_mapping, const hipattn_tensor *multi_block_tables,
    const hipattn_tensor *seqlens_q, const hipattn_tensor *multi_context_lens,
    int64_t q_multi, int max_seqlen_q, int max_seqlen_k,
    const hipattn_tensor *paged_block_tables,
    const hipattn_tensor *paged_context_lens, int paged_block_size,
    int paged_max_context_len, float softmax_scale, int window_size_left,
    int sink_tokens, hipattn_tensor *y, void *stream);
char *hipattn_varlen_attn_paged_window_ws(
    const hipattn_tensor *q, const hipattn_tensor *k, const hipattn_tensor *v,
    hipattn_tensor *key_cache, hipattn_tensor *value_cache,
    const hipattn_tensor *slot_mapping, const hipattn_tensor *multi_block_tables,
    const hipattn_tensor *seqlens_q, const hipattn_tensor *multi_context_lens,
    int64_t q_multi, int max_seqlen_q, int max_seqlen_k,
    const hipattn_tensor *paged_block_tables,
    const hipattn_tensor *paged_context_lens, int paged_block_size,
    int paged_max_context_len, float softmax_scale, int window_size_left,
    int sink_tokens, hipattn_tensor *y, const hipattn_tensor *workspace,
    void *stream);

#ifdef __cplusplus
}
#endif
#endif /* HIPATTN_H */
