// Paged decode over a sliding window with sinks: one query token per sequence against the last window_left + 1 tokens of its context
// and the first sink_tokens ones.  rLLM has no such models (it passes no window, rllm/tch-cuda/src/lib.rs:96-97); the reference's flash
// kernel knows windows for the rows of a prompt alone (rllm/tch-cuda/kernels/flash_attn/flash_api.cpp:113-120).
//
//   out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),  s_t = scale q . k_t,  over t < ctx with t >= ctx - 1 - window_left or t < sinks.
//
// What bounds it: the bytes of the keys and values that are seen, 4 d per (token, kv head), like all of paged decode.  So these are the
// kernels of paged decode -- query heads of a kv group as MFMA columns, K and V blocks as operands straight from the cache, the flat
// split or partitions, a merge -- over the 32-token pairs that hold a seen key, numbered without the gap between the sinks and the
// window (SeenKeys); columns of the gap are not read, so that their blocks may have gone back to the pool.  A launch is planned as one
// over contexts of that many tokens (seen_tokens).  The pair at either end of the gap is masked in its scores and its values are cleared:
// a NaN there meets a probability of zero otherwise.  Probabilities are rounded to the cache's type as operands of the second product, as in all paged
// decode; scores, sums, partitions and the merge are fp32.
//
// Measured, 128 sequences of up to 16k tokens, 32 / 8 x 128 bf16, a window of 4096: 314 us, 1.99 GB at 6.3 TB/s (a read kernel with the same hint
// gets 6.5), 6.6 of them the merge.  With few keys it is latency: 48 sequences, 39.7 MB, 11.8 us in one launch (lengths, table, keys one
// after the other; 8.3 at a copy's rate); one sequence that sees 1028 keys 8.1 us, 5.7 + 3.1 of merge by the trace, whatever the number of partitions.
#include <algorithm>

#include "paged_decode_parts.h"
#include "workspace.h"

namespace hipattn {

namespace {

// Tokens of the pairs that a sequence can see keys in, at most.
int64_t seen_tokens(int max_context_len, int window_left, int sinks) {
  const int64_t window_pairs = ((int64_t)window_left + 31) / 32 + 1, sink_pairs = ((int64_t)sinks + 31) / 32;
  return std::min<int64_t>(max_context_len, 32 * (window_pairs + sink_pairs));
}

void check_window(const char *op, int window_left, int sinks) {
  HA_CHECK(window_left >= 0, "%s: window_size_left must not be negative here, got %d", op, window_left);
  HA_CHECK(sinks >= 0, "%s: sink_tokens must not be negative, got %d", op, sinks);
}

void check_head_size(const char *op, int hd) {
  HA_CHECK(hd == 64 || hd == 80 || hd == 96 || hd == 112 || hd == 128 || hd == 256,
           "%s: unsupported head size %d (supported: 64, 80, 96, 112, 128, 256)", op, hd);
}

template <typename T, int HD>
void launch_head(const DecodeParams &p, const DecodePlan &pl, int block_size, char *ws, hipStream_t stream) {
  if (pl.flat) {
    launch_decode_flat<T, HD, WindowKeys>(p, pl, block_size, ws, stream);
    return;
  }
  switch (block_size) {
    case 8: launch_decode<T, HD, false, 8, WindowKeys>(p, p.num_seqs, stream); break;
    case 32: launch_decode<T, HD, false, 32, WindowKeys>(p, p.num_seqs, stream); break;
    default: launch_decode<T, HD, false, kBlockSize, WindowKeys>(p, p.num_seqs, stream); break;
  }
}

template <typename T>
void dispatch_window(const DecodeParams &p, const DecodePlan &pl, int head_size, int block_size, char *ws, hipStream_t stream) {
  switch (head_size) {
    case 64: launch_head<T, 64>(p, pl, block_size, ws, stream); break;
    case 80: launch_head<T, 80>(p, pl, block_size, ws, stream); break;
    case 96: launch_head<T, 96>(p, pl, block_size, ws, stream); break;
    case 112: launch_head<T, 112>(p, pl, block_size, ws, stream); break;
    case 128: launch_head<T, 128>(p, pl, block_size, ws, stream); break;
    case 256: launch_head<T, 256>(p, pl, block_size, ws, stream); break;
    default: fail("paged_attention_window: unsupported head size %d (supported: 64, 80, 96, 112, 128, 256)", head_size);
  }
}

void paged_attention_window_impl(hipattn_tensor *out, const hipattn_tensor *query, const hipattn_tensor *key_cache,
                                 const hipattn_tensor *value_cache, int num_kv_heads, float scale, const hipattn_tensor *block_tables,
                                 const hipattn_tensor *context_lens, int block_size, int max_context_len, int window_left, int sinks,
                                 const hipattn_tensor *alibi, const hipattn_tensor *workspace, void *stream_arg) {
  const char *op = "paged_attention_window";
  check_window(op, window_left, sinks);
  check_tensor(query, "query", 3);
  HA_CHECK(query->dtype == HIPATTN_F16 || query->dtype == HIPATTN_BF16, "%s: unsupported data type %s (supported: f16, bf16)", op,
           dtype_name(query->dtype));
  const int hd = (int)query->sizes[2];
  check_head_size(op, hd);
  if (workspace) {
    check_tensor(workspace, "workspace", 1);
    HA_CHECK(workspace->dtype == HIPATTN_U8, "%s: workspace must be u8", op);
    check_contiguous(workspace, "workspace");
  }
  DecodeParams p;
  if (!decode_params(DecodeCall{query, key_cache, value_cache, num_kv_heads, scale, block_tables, context_lens, block_size, max_context_len,
                                alibi, op},
                     out, p))
    return;
  p.window_left = std::min(window_left, p.max_ctx);  // (what ctx - 1 - window_left stays within 32 bits with)
  p.sinks = std::min(sinks, p.max_ctx);
  hipStream_t stream = resolve_stream(stream_arg);
  const DecodePlan pl = plan_decode(p.num_seqs, p.Hq, num_kv_heads, hd, block_size, query->dtype,
                                    (int)seen_tokens(p.max_ctx, window_left, sinks));
  char *ws = nullptr;
  HeldWorkspace held;  // over both launches
  if (pl.bytes > 0 && workspace) {
    HA_CHECK(workspace->data != nullptr && (reinterpret_cast<uintptr_t>(workspace->data) & 255) == 0,
             "%s: workspace must be 256-byte aligned", op);
    HA_CHECK((size_t)workspace->sizes[0] >= pl.bytes,
             "%s: workspace of %lld bytes is too small, %zu are needed (hipattn_paged_attention_window_workspace_size)", op,
             (long long)workspace->sizes[0], pl.bytes);
    ws = static_cast<char *>(workspace->data);
  } else if (pl.bytes > 0) {
    held = library_workspace(WS_WINDOW_ATTENTION, pl.bytes, stream);
    ws = static_cast<char *>(held.ptr);
  }
  if (!pl.flat) {
    p.part_blocks = pl.part_blocks;
    p.num_parts = pl.num_parts;
    p.waves = pl.waves;
    if (pl.num_parts > 1) {
      p.ws_acc = reinterpret_cast<float *>(ws);
      p.ws_m = p.ws_acc + pl.slots * hd;
      p.ws_l = p.ws_m + pl.slots;
    }
  }
  if (query->dtype == HIPATTN_F16) dispatch_window<half_t>(p, pl, hd, block_size, ws, stream);
  else dispatch_window<bf16_t>(p, pl, hd, block_size, ws, stream);
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" char *hipattn_paged_attention_window(hipattn_tensor *out, const hipattn_tensor *query, const hipattn_tensor *key_cache,
                                                const hipattn_tensor *value_cache, int num_kv_heads, float scale,
                                                const hipattn_tensor *block_tables, const hipattn_tensor *context_lens, int block_size,
                                                int max_context_len, int window_size_left, int sink_tokens,
                                                const hipattn_tensor *alibi_slopes, const hipattn_tensor *workspace, void *stream) {
  HA_PROTECT(paged_attention_window_impl(out, query, key_cache, value_cache, num_kv_heads, scale, block_tables, context_lens, block_size,
                                         max_context_len, window_size_left, sink_tokens, alibi_slopes, workspace, stream));
}

extern "C" char *hipattn_paged_attention_window_workspace_size(int64_t num_seqs, int num_heads, int num_kv_heads, int head_size,
                                                               int block_size, int max_context_len, int window_size_left,
                                                               int sink_tokens, int32_t dtype, int64_t *bytes) {
  HA_PROTECT({
    const char *op = "paged_attention_window_workspace_size";
    HA_CHECK(bytes != nullptr, "%s: bytes is NULL", op);
    HA_CHECK(num_seqs >= 0 && num_heads >= 0 && max_context_len >= 0, "%s: negative size", op);
    HA_CHECK(dtype == HIPATTN_F16 || dtype == HIPATTN_BF16, "%s: unsupported data type %s (supported: f16, bf16)", op, dtype_name(dtype));
    HA_CHECK(block_size == 8 || block_size == 16 || block_size == 32, "%s: unsupported block size %d (supported: 8, 16, 32)", op, block_size);
    HA_CHECK(num_kv_heads > 0 && num_heads % num_kv_heads == 0, "%s: %d query heads not divisible by %d kv heads", op, num_heads, num_kv_heads);
    check_window(op, window_size_left, sink_tokens);
    check_head_size(op, head_size);
    *bytes = (int64_t)plan_decode(num_seqs, num_heads, num_kv_heads, head_size, block_size, dtype,
                                  (int)seen_tokens(max_context_len, window_size_left, sink_tokens))
                 .bytes;
  });
}
