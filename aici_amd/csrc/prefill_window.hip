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

#include "paged_decode.h"
#include "prefill_parts.h"
#include "prefill_w8.h"

namespace hipattn {

namespace {

struct PrefillWindow {
  struct Params : PrefillParams {
    int block_rows;             // rows of a row block
    int n_parts, part_tiles;    // pieces of a row block's keys at most, and 64-key tiles in each
    float *part_acc, *part_ml;  // of piece i of row r and head h, at (i * total_q + r) * Hq + h: d sums; maximum and sum
  };
  static constexpr bool value = false, parts = true, window = true;
};

// The merge of row blocks whose keys were dealt out, a workgroup per (row, kMergeHeads heads).
template <typename T, int HD>
__global__ __launch_bounds__(128) void window_merge_kernel(PrefillWindow::Params p) {
  const int groups = (p.Hq + kMergeHeads - 1) / kMergeHeads, lane = threadIdx.x & 63;
  const int r = blockIdx.x / groups, h0 = blockIdx.x % groups * kMergeHeads;
  int b = -1;
  for (int s0 = 0; s0 < p.batch && b < 0; s0 += 64) {
    const unsigned long long past = __ballot(s0 + lane < p.batch && p.cu_q[min(s0 + lane, p.batch - 1) + 1] > r);
    if (past != 0) b = s0 + __builtin_ctzll(past);
  }
  if (b < 0) return;
  const int q_begin = p.cu_q[b], Lq = p.cu_q[b + 1] - q_begin, Lk = p.context_lens[b];
  if (r < q_begin) return;
  const int first_row = (r - q_begin) / p.block_rows * p.block_rows, last_row = min(first_row + p.block_rows, Lq) - 1;  // of the row's block
  int tiles = (max(min(Lk, last_row + Lk - Lq + 1), 0) + BN - 1) / BN;
  const int seen_from = max(first_row + Lk - Lq - p.win_left, 0);  // (the kernel's arithmetic)
  tiles -= max(seen_from / BN - (min(p.sinks, seen_from) + BN - 1) / BN, 0);
  if (tiles <= p.part_tiles) return;  // whole, and written
  merge_parts<T, HD>(p, r, h0, min((tiles + p.part_tiles - 1) / p.part_tiles, p.n_parts));
}

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
  const int bm = p.block_rows = (NW * 32) >> hl;
  p.n_qblocks = (p.max_q + bm - 1) / bm;
  const int64_t n_wg = (int64_t)p.n_qblocks * p.batch * (p.Hq >> hl) * p.n_parts;
  HA_CHECK(n_wg <= 0x7fffffff, "mha_varlen_fwd_paged_window: too many workgroups");
  kernel<<<dim3((unsigned)n_wg), NW * 64, lds_bytes, stream>>>(p);
  check_launch("mha_varlen_fwd_paged_window");
  if (p.n_parts > 1) {
    const int64_t merges = p.total_q * ((p.Hq + kMergeHeads - 1) / kMergeHeads);
    HA_CHECK(merges <= 0x7fffffff, "mha_varlen_fwd_paged_window: too many rows");
    switch (p.d) {
      case 64: window_merge_kernel<T, 64><<<dim3((unsigned)merges), 128, 0, stream>>>(p); break;
      case 80: window_merge_kernel<T, 80><<<dim3((unsigned)merges), 128, 0, stream>>>(p); break;
      case 96: window_merge_kernel<T, 96><<<dim3((unsigned)merges), 128, 0, stream>>>(p); break;
      case 112: window_merge_kernel<T, 112><<<dim3((unsigned)merges), 128, 0, stream>>>(p); break;
      case 128: window_merge_kernel<T, 128><<<dim3((unsigned)merges), 128, 0, stream>>>(p); break;
      default: fail("mha_varlen_fwd_paged_window: no merge for head size %d", p.d);
    }
    check_launch("mha_varlen_fwd_paged_window (merge)");
  }
}

// Tiles of the longest chain: what a row block of `rows` rows sees at most.
int64_t most_tiles(const PrefillParams &p, int rows) {
  return std::min<int64_t>(((int64_t)p.max_k + BN - 1) / BN, ((int64_t)p.sinks + BN - 1) / BN + ((int64_t)p.win_left + rows + BN - 1) / BN + 1);
}

// Workgroups of `waves` wavefronts with work to do, about.
int64_t busy_workgroups(const PrefillParams &p, int waves, int hl) {
  return std::max<int64_t>(p.total_q / ((waves * 32) >> hl) + (p.batch + 1) / 2, 1) * (p.Hq >> hl);
}

// Workgroups of eight wavefronts instead of four: where windows are long enough for what their alternation between the pipes gains a tile, and
// there is one of them for nearly every compute unit, or several, of more than one head.  us, eight / four: 32 / 8 x 128, 2 x 4096 new tokens
// with a window of 4096 549 / 574, 16 x 512 of 2048 327 / 333, 1 x 2000 of 4096 (250 workgroups) 145 / 154, 4 x 2048 of 1024 182 / 174; 32 / 32 x 80,
// 1 x 2000 of 4096 133 / 152, 2 x 4096 502 / 493; 16 / 2 x 64, 2 x 4096 215 / 228, 1 x 2000 of 4096 (125) 108 / 88; 12 / 4 x 112, 16 x 512 of 2048 173 /
// 151, 2 x 4096 277 / 275.
bool eight_wavefronts_pay(const PrefillParams &p) {
  const int hl = prefill_heads_log2(p, 3);
  const int64_t wgs = busy_workgroups(p, 8, hl);
  return most_tiles(p, 256 >> hl) >= 32 && wgs >= 200 && (wgs <= 256 || hl > 0);
}

// Pieces that a row block's keys are dealt out in (workgroups of four wavefronts).  A workgroup's chain of tiles is bound by its own
// instructions, some 1.4 us a tile with a wavefront per SIMD (five tiles in LDS instead of two change nothing), so where compute units are idle
// more of them take a part each.  All in us: a tile, which takes longer from one workgroup per compute unit on, but less than in proportion,
// as two or three of them fill each other's gaps; the merge's launch, and what writing and reading the pieces costs.  In 56 measured shapes (16
// x 4 new tokens to 2 x 4096, windows of 100 to 4096) the choice among 1, 2, 3, 4, 6, 10 and 16, which asks for a tenth before it cuts, is 0.7 % off the best on average.  us, whole / best:
// 32 / 8 x 128, 1 x 16 over 4096 keys 102 / 25 (16 pieces), 1 x 300 106 / 47 (6), 4 x 64 over 2048 62 / 33 (4), 16 x 20 over 4096 104 / 63 (4);
// 16 / 2 x 64, 1 x 45 over 256 17.5 / 11.1 (7); 32 / 8 x 128, 4 x 8 over 100 10.5 / 10.5 (1; in 2 13.7).
int choose_parts(const PrefillParams &p) {
  const int hl = prefill_heads_log2(p, 2);
  const int64_t tiles = most_tiles(p, 128 >> hl), wgs = busy_workgroups(p, 4, hl);
  const double tile = p.d > 96 ? 1.45 : (p.d > 64 ? 1.55 : 1.25), share = (p.d > 96 ? 0.6 : 0.4) / compute_units();
  const double piece = (double)p.total_q * p.Hq * (p.d + 2) * 2e-6;
  double best = 0;
  int parts = 1;
  for (int n = 1; n <= kMostParts && n <= tiles; n++) {
    const int64_t part_tiles = (tiles + n - 1) / n;
    if ((tiles + part_tiles - 1) / part_tiles != n) continue;
    const double t = (double)part_tiles * tile * std::max(1.0, share * (double)(wgs * n)) + (n > 1 ? 3.0 + n * piece : 0.0);
    if (n == 1) {
      best = 0.9 * t;
    } else if (t < best) {
      best = t;
      parts = n;
    }
  }
  return parts;
}

// A stream's buffer, allocated once; row blocks whose pieces do not fit go whole.
constexpr size_t kWindowScratchBytes = (size_t)64 << 20;

template <typename T, int HDP, int MODE>
void launch_window(PrefillWindow::Params p, bool lse_or_f32, hipStream_t stream) {
  const int force = tuning().prefill_kernel;
  if (force == 1 || (force != 5 && eight_wavefronts_pay(p))) {
    launch_window_nw<T, HDP, MODE, 8>(p, prefill_heads_log2(p, 3), stream);
    return;
  }
  const int hl = prefill_heads_log2(p, 2);
  // (whole where the merge has no form, or a switch asks for a kernel)
  int parts = lse_or_f32 || force != 0 || (p.d != 64 && p.d != 80 && p.d != 96 && p.d != 112 && p.d != 128) || stream == hipStreamPerThread ? 1 : choose_parts(p);
  const size_t rows = (size_t)p.total_q * p.Hq, piece_bytes = rows * (p.d + 2) * sizeof(float);
  if ((size_t)parts * piece_bytes > kWindowScratchBytes) parts = (int)(kWindowScratchBytes / piece_bytes);
  HeldWorkspace ws;
  if (parts > 1) ws = try_library_workspace(WS_WINDOW_CHUNKS, kWindowScratchBytes, stream);
  if (ws.ptr != nullptr) {
    const int64_t tiles = most_tiles(p, 128 >> hl);
    p.part_tiles = (int)((tiles + parts - 1) / parts);
    p.n_parts = (int)((tiles + p.part_tiles - 1) / p.part_tiles);
    p.part_acc = static_cast<float *>(ws.ptr);
    p.part_ml = p.part_acc + p.n_parts * rows * p.d;
  }
  launch_window_nw<T, HDP, MODE, 4>(p, hl, stream);
}

template <typename T>
void dispatch_window(const PrefillWindow::Params &p, bool lse_or_f32, hipStream_t stream) {
  switch ((p.d + 31) / 32 * 32) {
    case 32: launch_window<T, 32, W8_PAGED_DMA>(p, lse_or_f32, stream); break;
#define HA_W8W(H)                                                     \
  case H:                                                             \
    if (p.d == H) launch_window<T, H, W8_PAGED_DMA>(p, lse_or_f32, stream);       \
    else launch_window<T, H, W8_PAGED_DMA_PART>(p, lse_or_f32, stream);           \
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
  const bool lse_or_f32 = lse != nullptr || p.out_f32;  // (the merge has neither)
  if (q->dtype == HIPATTN_F16) dispatch_window<half_t>(p, lse_or_f32, stream);
  else dispatch_window<bf16_t>(p, lse_or_f32, stream);
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
