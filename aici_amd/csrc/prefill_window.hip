// Varlen prefill over the paged cache with a sliding window and sinks: new tokens of a sequence, causal, each against the window_left
// tokens before it, itself and the sequence's first sink_tokens ones.  The reference has windows without sinks and over rows of k / v alone
// (rllm/tch-cuda/kernels/flash_attn/flash_api.cpp:113-120, softmax.h:142-179); rLLM passes none.
//
//   row r of the sequence, at position r + Lk - Lq, sees key j iff j <= r + Lk - Lq and (j >= r + Lk - Lq - window_left or j < sinks).
//
// The kernels are those of hipattn_mha_varlen_fwd_paged -- block images of the cache copied into LDS, two wavefronts of a SIMD that alternate
// between the matrix pipe and the vector ALU, or workgroups of four wavefronts several to a compute unit -- over the 64-key tiles that hold a
// key some row of the workgroup sees (prefill_w8.h, STEP::window).  What bounds them is the matrix pipe and the vector unit on
// (window + rows of a block) keys a row, and with few workgroups the chain of a row block's tiles.
#include <algorithm>

#include "prefill_parts.h"
#include "prefill_w8.h"

namespace hipattn {

namespace {

struct PrefillWindow {
  struct Params : PrefillParams {
    int n_parts, part_tiles;    // pieces of a row block's keys at most, and 64-key tiles in each
    float *part_acc, *part_ml;  // of piece i of row r and head h, at (i * total_q + r) * Hq + h: d sums; maximum and sum
  };
  static constexpr bool value = false, parts = true, window = true;
};

template <typename T, int HDP, int MODE, int NW>
void launch_window_nw(PrefillWindow::Params p, int hl, hipStream_t stream) {
  static bool attr_set = false;  // benign race: setting twice is harmless
  auto kernel = prefill_varlen_w8_kernel<T, HDP, MODE, PrefillWindow, NW>;
  constexpr size_t lds_bytes = (size_t)w8_stages(HDP, NW) * 2 * BN * HDP * 2;
  if (!attr_set) {
    HA_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_bytes));
    attr_set = true;
  }
  p.wg_heads_log2 = hl;
  const int bm = (NW * 32) >> hl;
  p.n_qblocks = (p.max_q + bm - 1) / bm;
  const int64_t n_wg = (int64_t)p.n_qblocks * p.batch * (p.Hq >> hl) * p.n_parts;
  HA_CHECK(n_wg <= 0x7fffffff, "mha_varlen_fwd_paged_window: too many workgroups");
  kernel<<<dim3((unsigned)n_wg), NW * 64, lds_bytes, stream>>>(p);
  check_launch("mha_varlen_fwd_paged_window");
}

template <typename T, int HDP, int MODE>
void launch_window(const PrefillWindow::Params &p, hipStream_t stream) {
  const int force = tuning().prefill_kernel;
  const bool four = force == 5 || force == 0;
  if (four) launch_window_nw<T, HDP, MODE, 4>(p, prefill_heads_log2(p, 2), stream);
  else launch_window_nw<T, HDP, MODE, 8>(p, prefill_heads_log2(p, 3), stream);
}

template <typename T>
void dispatch_window(const PrefillWindow::Params &p, hipStream_t stream) {
  switch ((p.d + 31) / 32 * 32) {
    case 32: launch_window<T, 32, W8_PAGED_DMA>(p, stream); break;
#define HA_W8W(H)                                                     \
  case H:                                                             \
    if (p.d == H) launch_window<T, H, W8_PAGED_DMA>(p, stream);       \
    else launch_window<T, H, W8_PAGED_DMA_PART>(p, stream);           \
    break
    HA_W8W(64);
    HA_W8W(96);
    HA_W8W(128);
#undef HA_W8W
    default: fail("mha_varlen_fwd_paged_window: head size %d not supported by this kernel", p.d);
  }
}

void mha_varlen_fwd_paged_window_impl(const hipattn_tensor *q, const hipattn_tensor *key_cache, const hipattn_tensor *value_cache,
                                      const hipattn_tensor *block_tables, const hipattn_tensor *cu_q, const hipattn_tensor *context_lens,
                                      int max_q, int max_k, float scale, int window_left, int sinks, hipattn_tensor *out,
                                      hipattn_tensor *lse, void *stream_arg) {
  const char *op = "mha_varlen_fwd_paged_window";
  HA_CHECK(window_left >= 0, "%s: window_size_left must not be negative here, got %d", op, window_left);
  HA_CHECK(sinks >= 0, "%s: sink_tokens must not be negative, got %d", op, sinks);
  PrefillWindow::Params p;
  if (!paged_prefill_params(PagedPrefillCall{q, key_cache, value_cache, block_tables, cu_q, context_lens, max_q, max_k, scale, true, op}, out,
                            lse, p))
    return;
  // (no context is longer than its table: what lies beyond that sees everything, and row + Lk - Lq - window_left stays within 32 bits)
  const int64_t longest = (int64_t)p.table_cols << p.block_log2;
  p.win_left = (int)std::min<int64_t>(window_left, std::min<int64_t>(longest, 1 << 30));
  p.sinks = (int)std::min<int64_t>(sinks, std::min<int64_t>(longest, 1 << 30));
  p.win_right = 0;
  p.causal = 1;
  p.n_parts = 1;
  p.part_tiles = 1 << 24;
  p.part_acc = p.part_ml = nullptr;
  hipStream_t stream = resolve_stream(stream_arg);
  // Block images go into LDS as they are where they fill most of their place there; else tiles are staged through registers.
  if (!paged_prefill_copies_images(p) || p.d > 128 || (p.d < 64 && p.d != 32)) {
    launch_staged_window(p, q->dtype, stream);
    return;
  }
  if (q->dtype == HIPATTN_F16) dispatch_window<half_t>(p, stream);
  else dispatch_window<bf16_t>(p, stream);
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" char *hipattn_mha_varlen_fwd_paged_window(const hipattn_tensor *q, const hipattn_tensor *key_cache,
                                                     const hipattn_tensor *value_cache, const hipattn_tensor *block_tables,
                                                     const hipattn_tensor *cu_seqlens_q, const hipattn_tensor *context_lens,
                                                     int max_seqlen_q, int max_seqlen_k, float softmax_scale, int window_size_left,
                                                     int sink_tokens, hipattn_tensor *out, hipattn_tensor *softmax_lse, void *stream) {
  HA_PROTECT(mha_varlen_fwd_paged_window_impl(q, key_cache, value_cache, block_tables, cu_seqlens_q, context_lens, max_seqlen_q,
                                              max_seqlen_k, softmax_scale, window_size_left, sink_tokens, out, softmax_lse, stream));
}
