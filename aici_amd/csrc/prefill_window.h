// The launches of windowed prefill (prefill_window.hip) for caches of one block size; a translation unit for each.  Device code.
#pragma once

#include "prefill_parts.h"
#include "prefill_w8.h"
#include "prefill_window_params.h"

namespace hipattn {

namespace {

template <int BS>
struct PrefillWindow {
  typedef WindowParams Params;
  static constexpr bool value = false, parts = true, window = true;
  static constexpr int block = BS;
};

// The merge of row blocks whose keys were dealt out, a workgroup per (row, kMergeHeads heads).
template <typename T, int HD>
__global__ __launch_bounds__(128) void window_merge_kernel(WindowParams p) {
  const int groups = (p.Hq + kMergeHeads - 1) / kMergeHeads;
  const int r = blockIdx.x / groups, h0 = blockIdx.x % groups * kMergeHeads;
  const int b = sequence_of_row(p.cu_q, p.batch, r);
  if (b < 0) return;
  const int q_begin = p.cu_q[b], Lq = p.cu_q[b + 1] - q_begin, Lk = p.context_lens[b];
  if ((r - q_begin) / p.block_rows >= p.n_qblocks) return;  // beyond max_seqlen_q: left out
  const int first_row = (r - q_begin) / p.block_rows * p.block_rows, last_row = min(first_row + p.block_rows, Lq) - 1;  // of the row's block
  int tiles = (max(min(Lk, last_row + Lk - Lq + 1), 0) + BN - 1) / BN;
  const int seen_from = max(first_row + Lk - Lq - p.win_left, 0);  // (the kernel's arithmetic)
  tiles -= max(seen_from / BN - (min(p.sinks, seen_from) + BN - 1) / BN, 0);
  if (tiles <= p.part_tiles) return;  // whole, and written
  merge_parts<T, HD>(p, r, h0, min((tiles + p.part_tiles - 1) / p.part_tiles, p.n_parts));
}

template <typename T, int BS, int HDP, int MODE, int NW>
void launch_window_nw(WindowParams p, int hl, hipStream_t stream) {
  static bool attr_set = false;  // benign race: setting twice is harmless
  auto kernel = prefill_varlen_w8_kernel<T, HDP, MODE, PrefillWindow<BS>, NW>;
  constexpr size_t lds_bytes = (size_t)w8_stages(HDP, NW) * 2 * BN * HDP * 2;
  if (!attr_set) {
    HA_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_bytes));
    attr_set = true;
  }
  p.wg_heads_log2 = hl;
  const int bm = p.block_rows = (NW * 32) >> hl;
  p.n_qblocks = (p.max_q + bm - 1) / bm;
  const int64_t listed = row_blocks_of(p.total_q, p.batch, bm, p.n_qblocks);
  const int64_t n_wg = (listed > 0 ? listed : (int64_t)p.n_qblocks * p.batch) * (p.Hq >> hl) * p.n_parts;
  HA_CHECK(n_wg <= 0x7fffffff, "mha_varlen_fwd_paged_window: too many workgroups");
  p.row_blocks = (int)listed;
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

template <typename T, int BS, int HDP, int MODE>
void launch_window(const WindowParams &p, int waves, hipStream_t stream) {
  if (waves == 8) launch_window_nw<T, BS, HDP, MODE, 8>(p, prefill_heads_log2(p, 3), stream);
  else launch_window_nw<T, BS, HDP, MODE, 4>(p, prefill_heads_log2(p, 2), stream);
}

template <typename T, int BS>
void dispatch_window(const WindowParams &p, int waves, hipStream_t stream) {
  switch ((p.d + 31) / 32 * 32) {
    case 32: launch_window<T, BS, 32, W8_PAGED_DMA>(p, waves, stream); break;
#define HA_W8W(H)                                                     \
  case H:                                                             \
    if (p.d == H) launch_window<T, BS, H, W8_PAGED_DMA>(p, waves, stream);       \
    else launch_window<T, BS, H, W8_PAGED_DMA_PART>(p, waves, stream);           \
    break
    HA_W8W(64);
    HA_W8W(96);
    HA_W8W(128);
#undef HA_W8W
    default: fail("mha_varlen_fwd_paged_window: head size %d not supported by this kernel", p.d);
  }
}

template <int BS>
void launch_window_images(const WindowParams &p, int waves, int dtype, hipStream_t stream) {
  if (dtype == HIPATTN_F16) dispatch_window<half_t, BS>(p, waves, stream);
  else dispatch_window<bf16_t, BS>(p, waves, stream);
}

}  // namespace
}  // namespace hipattn
