// Few new tokens of a sequence (a draft to be verified, the end of a prompt) over a window of its paged cache.
//
// A workgroup of the prefill kernel takes 128 or 256 rows of a head through one tile of 64 keys after the other; with few rows most of its
// rows are empty and the chain is long.  Here the rows are columns of the decode kernel's products, 16 at a time -- whole rows with the query
// heads of a kv group, as many as fit -- so that the keys a column group sees can be dealt out to many wavefronts, 32 at a time, and the merge
// adds up what they leave.  The keys are read once per column group, from L2 but for the first.
//
// Numerics are those of paged decode: scores and sums in fp32, probabilities rounded to the cache's type as operands of the second product,
// the normaliser not.
#include <algorithm>

#include "paged_decode.h"
#include "prefill_parts.h"
#include "window_rows.h"

namespace hipattn {

namespace {

struct RowsParams {
  DecodeParams cache;  // the caches, tables, context lengths, scale, window and sinks
  const void *q;
  void *out;
  int64_t q_row, q_head, o_row, o_head, total_q;
  const int32_t *cu_q;
  int batch, Hq, Hkv, G;
  int rows_per_group, head_groups;  // columns: that many rows with all G heads, or one row with 16 of them
  int row_groups;                   // groups of rows of a sequence, at most
  int listed;                       // 0, or the groups of rows of the grid, one sequence's behind the other's (row_block_of)
  int part_pairs, num_parts, waves;
  float *part_acc, *part_ml;  // of part i of row r and head h, at (i * total_q + r) * Hq + h: d sums; maximum and sum
};

// The keys that rows [i0, i1] of a sequence see.
__device__ __forceinline__ SeenKeys rows_see(const RowsParams &p, int Lq, int Lk, int i0, int i1) {
  return SeenKeys(p.cache, Lk - Lq + i1 + 1, i1 - i0 + 1);
}
// Runs of 16 tokens that hold them.  The parts hold what max_seqlen_k allows: of a context beyond that the last ones are left out, as there is
// neither a part nor scratch memory for them.
__device__ __forceinline__ int seen_runs(const RowsParams &p, const SeenKeys &s) {
  return s.ctx > 0 ? min((s.ctx + kBlockSize - 1) / kBlockSize - 2 * s.skip, 2 * p.part_pairs * p.num_parts) : 0;
}

template <typename T, int HD, int BS, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void window_rows_kernel(RowsParams p) {
  typedef typename Vec8<T>::type vec8;
  constexpr int NCH = HD / 8, NSTEP = (HD + 31) / 32, NDT = HD / 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, kg = lane >> 4, col = lane & 15;
  // Workgroup -> (part, sequence, column group, kv head), the kv head fastest: the column groups that read the same keys share an XCD's L2.
  int id = blockIdx.x;
  const int kvh = id % p.Hkv;
  id /= p.Hkv;
  const int hg = id % p.head_groups;
  id /= p.head_groups;
  const int all_groups = p.listed > 0 ? p.listed : p.row_groups * p.batch, part = id / all_groups;
  id %= all_groups;
  RowBlock blk;
  if (p.listed > 0) {
    blk = row_block_of(p.cu_q, p.cache.context_lens, p.cache.window_left / 2, p.batch, p.rows_per_group, p.row_groups, id);
  } else {
    blk.seq = id / p.row_groups;
    blk.block = id % p.row_groups;
    blk.begin = p.cu_q[blk.seq];
    blk.rows = p.cu_q[blk.seq + 1] - blk.begin;
  }
  const int seq = blk.seq, q_begin = blk.begin, Lq = blk.rows;
  const int i0 = blk.block * p.rows_per_group;  // the group's first row
  if (i0 < 0 || i0 >= Lq) return;
  const int i1 = min(i0 + p.rows_per_group, Lq) - 1;
  const int Lk = p.cache.context_lens[seq];
  const SeenKeys seen = rows_see(p, Lq, Lk, i0, i1);
  const int nblk = seen_runs(p, seen), b0 = part * p.part_pairs * 2;
  if (b0 >= nblk && part > 0) return;
  const int nb = min(b0 + p.part_pairs * 2, nblk) - b0;  // runs of this part
  const int t0 = b0 * kBlockSize / BS, tn = p.part_pairs * 2 * kBlockSize / BS;
  const int32_t *table = p.cache.block_tables + seq * p.cache.max_blocks;
  int tbl = 0, tbl_hi = 0;
  if (lane < tn && seen.column(t0 + lane, BS) < p.cache.table_cols) tbl = table[seen.column(t0 + lane, BS)];
  if (BS == 8 && 64 + lane < tn && seen.column(t0 + 64 + lane, BS) < p.cache.table_cols) tbl_hi = table[seen.column(t0 + 64 + lane, BS)];

  const int row = i0 + (p.head_groups > 1 ? 0 : col / p.G), g = p.head_groups > 1 ? hg * 16 + col : col % p.G;
  const bool col_ok = row <= i1 && g < p.G && (p.head_groups > 1 || col < p.rows_per_group * p.G);
  const int qh = kvh * p.G + g;
  const KeyRange mine = rows_see(p, Lq, Lk, row, row);
  vec8 qreg[NSTEP];
  {
    const T *qp = static_cast<const T *>(p.q) + (int64_t)(q_begin + row) * p.q_row + qh * p.q_head;
#pragma unroll
    for (int s = 0; s < NSTEP; s++) {
      const int ch = 4 * s + kg;
      u32x4_t raw = {0u, 0u, 0u, 0u};
      if (col_ok && ch < NCH) raw = *reinterpret_cast<const u32x4_t *>(qp + ch * 8);
      qreg[s] = bit_cast<vec8>(raw);
    }
  }
  const T *kbase = static_cast<const T *>(p.cache.kc) + (int64_t)kvh * p.cache.k_head_stride;
  const T *vbase = static_cast<const T *>(p.cache.vc) + (int64_t)kvh * p.cache.v_head_stride;
  float m_run = -INFINITY, l_run = 0.f;
  f32x4_t acc[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; dt++) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto load = [&](int it, PairRegs<HD> &r) {
    int64_t i0 = 0, i1 = 0, i2 = 0, i3 = 0;
    if constexpr (BS == 16) {
      i0 = __builtin_amdgcn_readlane(tbl, it);
      i1 = __builtin_amdgcn_readlane(tbl, it + 1 < nb ? it + 1 : it);
    } else if constexpr (BS == 32) {
      i0 = __builtin_amdgcn_readlane(tbl, it >> 1);
    } else {
      const int c = (2 * it) & 63, src = 2 * it < 64 ? tbl : tbl_hi;
      i0 = __builtin_amdgcn_readlane(src, c);
      i1 = __builtin_amdgcn_readlane(src, c + 1);
      i2 = __builtin_amdgcn_readlane(src, c + 2);
      i3 = __builtin_amdgcn_readlane(src, c + 3);
    }
    pair_load_bs<T, HD, BS, false>(p.cache, kbase, vbase, i0, i1, i2, i3, r);
  };
  // (a second pair on its way costs the registers that let a compute unit hold several workgroups: 32 / 8 x 128, 4 x 64 rows over 2048 keys 45 us ->
  // 70, 1 x 128 over 1024 21 -> 26)
  for (int it = 2 * wave; it < nb; it += 2 * WAVES) {
    PairRegs<HD> r;
    load(it, r);
    pair_compute<T, HD, WindowKeys>(p.cache, r, seen.run(b0 + it), it + 1 < nb, mine, seen, 0.f, qreg, m_run, l_run, acc);
  }

  float l_tot = l_run + __shfl_xor(l_run, 16, 64);
  l_tot += __shfl_xor(l_tot, 32, 64);
  // The wavefronts' states: common maximum, rescale, sum into wavefront 0.
  __shared__ float s_m[WAVES][16], s_l[WAVES][16];
  __shared__ f32x4_t s_acc[WAVES - 1][NDT][64];
  if (kg == 0) s_m[wave][col] = m_run;
  __syncthreads();
  float m_all = s_m[0][col];
#pragma unroll
  for (int w = 1; w < WAVES; w++) m_all = fmaxf(m_all, s_m[w][col]);
  const float wscale = fast_exp2(m_run - (m_all == -INFINITY ? 0.f : m_all));  // 0 for a wavefront that saw no key
  if (kg == 0) s_l[wave][col] = l_tot * wscale;
  if (wave > 0) {
#pragma unroll
    for (int dt = 0; dt < NDT; dt++) s_acc[wave - 1][dt][lane] = acc[dt] * wscale;
  }
  __syncthreads();
  if (wave > 0 || !col_ok) return;
  l_tot = s_l[0][col];
#pragma unroll
  for (int w = 1; w < WAVES; w++) l_tot += s_l[w][col];
#pragma unroll
  for (int dt = 0; dt < NDT; dt++) {
    acc[dt] = acc[dt] * wscale;
#pragma unroll
    for (int w = 0; w < WAVES - 1; w++) acc[dt] = acc[dt] + s_acc[w][dt][lane];
  }
  if (nblk <= p.part_pairs * 2) {  // nothing to merge
    const float inv = l_tot > 0.f ? 1.0f / l_tot : 0.f;
    T *op = static_cast<T *>(p.out) + (int64_t)(q_begin + row) * p.o_row + qh * p.o_head + kg * 4;
#pragma unroll
    for (int dt = 0; dt < NDT; dt++) {
      T r[4];
#pragma unroll
      for (int i = 0; i < 4; i++) r[i] = from_float<T>(acc[dt][i] * inv);
      *reinterpret_cast<u32x2_t *>(op + dt * 16) = *reinterpret_cast<u32x2_t *>(r);
    }
    return;
  }
  const int64_t at = ((int64_t)part * p.total_q + q_begin + row) * p.Hq + qh;
#pragma unroll
  for (int dt = 0; dt < NDT; dt++) *reinterpret_cast<f32x4_t *>(p.part_acc + at * HD + dt * 16 + kg * 4) = acc[dt];
  if (kg == 0) *reinterpret_cast<float2 *>(p.part_ml + 2 * at) = make_float2(m_all, l_tot);
}

// The merge, a workgroup per (row, kMergeHeads heads).
template <typename T, int HD>
__global__ __launch_bounds__(128) void window_rows_merge_kernel(RowsParams p) {
  const int head_blocks = (p.Hq + kMergeHeads - 1) / kMergeHeads;
  const int r = blockIdx.x / head_blocks, h0 = blockIdx.x % head_blocks * kMergeHeads;
  const int b = sequence_of_row(p.cu_q, p.batch, r);
  if (b < 0) return;
  const int q_begin = p.cu_q[b], Lq = p.cu_q[b + 1] - q_begin, group = (r - q_begin) / p.rows_per_group, i0 = group * p.rows_per_group;
  if (group >= p.row_groups) return;  // beyond max_seqlen_q: left out
  const int nblk = seen_runs(p, rows_see(p, Lq, p.cache.context_lens[b], i0, min(i0 + p.rows_per_group, Lq) - 1));
  if (nblk <= p.part_pairs * 2) return;  // written
  merge_parts<T, HD>(p, r, h0, (nblk + p.part_pairs * 2 - 1) / (p.part_pairs * 2));
}

template <typename T, int HD>
void launch_rows(const RowsParams &p, int block_size, hipStream_t stream) {
  const int64_t n_wg = (int64_t)p.num_parts * (p.listed > 0 ? p.listed : (int64_t)p.batch * p.row_groups) * p.head_groups * p.Hkv;
  HA_CHECK(n_wg <= 0x7fffffff, "mha_varlen_fwd_paged_window: too many workgroups");
  const dim3 grid((unsigned)n_wg);
#define HA_ROWS(BS)                                                                       \
  if (p.waves == 8) window_rows_kernel<T, HD, BS, 8><<<grid, 512, 0, stream>>>(p);        \
  else window_rows_kernel<T, HD, BS, 4><<<grid, 256, 0, stream>>>(p)
  switch (block_size) {
    case 8: HA_ROWS(8); break;
    case 32: HA_ROWS(32); break;
    default: HA_ROWS(kBlockSize); break;
  }
#undef HA_ROWS
  check_launch("mha_varlen_fwd_paged_window");
  if (p.num_parts > 1) {
    const int64_t merges = p.total_q * ((p.Hq + kMergeHeads - 1) / kMergeHeads);
    HA_CHECK(merges <= 0x7fffffff, "mha_varlen_fwd_paged_window: too many rows");
    window_rows_merge_kernel<T, HD><<<dim3((unsigned)merges), 128, 0, stream>>>(p);
    check_launch("mha_varlen_fwd_paged_window (merge)");
  }
}

template <typename T>
void dispatch_rows(const RowsParams &p, int head_size, int block_size, hipStream_t stream) {
  switch (head_size) {
    case 64: launch_rows<T, 64>(p, block_size, stream); break;
    case 80: launch_rows<T, 80>(p, block_size, stream); break;
    case 96: launch_rows<T, 96>(p, block_size, stream); break;
    case 112: launch_rows<T, 112>(p, block_size, stream); break;
    case 128: launch_rows<T, 128>(p, block_size, stream); break;
    case 256: launch_rows<T, 256>(p, block_size, stream); break;
    default: fail("mha_varlen_fwd_paged_window: head size %d not supported by this kernel", head_size);
  }
}

}  // namespace

// All in us, for each form: a launch, the chain of a wavefront's pairs, each longer where more workgroups run than some per compute unit (1.4 of
// four wavefronts, 0.68 of eight), and the merge (prefill_window.hip's choose_parts says how far off the choice is).  us, prefill / here:
// 32 / 8 x 128, 1 x 2 over 64 keys 10.7 / 6.3, 16 x 5 over 500 21.6 / 10.0, 1 x 45 over 256 18.3 / 8.3, 2 x 2 over 2048 22.0 / 14.9, 8 x 16 over 512 23.8 / 10.0, 1 x 300 over
// 4096 47 / 86; 12 / 4 x 112, 64 x 4 over 1024 75 / 27, 4 x 64 over 2048 29 / 24; 16 / 2 x 64, 1 x 16 over 4096 16.0 / 10.2.
bool plan_window_rows(const PrefillParams &p, int most_parts, RowsPlan &plan) {
  if (p.d != 64 && p.d != 80 && p.d != 96 && p.d != 112 && p.d != 128 && p.d != 256) return false;
  const int per = p.G <= 16 ? 16 / p.G : 1;
  const int64_t pairs = std::max<int64_t>(
      std::min<int64_t>(((int64_t)p.max_k + 31) / 32, ((int64_t)p.win_left + per + 30) / 32 + 1 + ((int64_t)p.sinks + 31) / 32), 1);
  const double wgs = (double)((p.G + 15) / 16) * ((double)((p.total_q + per - 1) / per) + 1.1 * p.batch) * p.Hkv;
  const double pair = 1.5 * (0.2 + 0.8 * p.d / 128), piece = (double)p.total_q * p.Hq * (p.d + 2) * 1.9e-6;
  plan.us = 0;
  for (int waves : {4, 8})
    for (int64_t part : {4, 8, 12, 16, 24, 32}) {  // (the columns of 32 pairs' blocks lie in the lanes)
      const int64_t parts = (pairs + part - 1) / part;
      if (parts > most_parts) continue;
      const double load = std::max(1.0, wgs * (double)parts / compute_units() / (waves == 4 ? 1.4 : 0.68));
      const double us = 6.6 + (double)((std::min(part, pairs) + waves - 1) / waves) * pair * load + (parts > 1 ? 3.7 + (double)parts * piece : 0.0);
      if (plan.us == 0 || us < plan.us) plan = RowsPlan{waves, (int)part, (int)parts, us};
    }
  return plan.us > 0;
}

void launch_window_rows(const PrefillParams &pp, const RowsPlan &plan, int dtype, void *scratch, hipStream_t stream) {
  RowsParams p;
  memset(&p, 0, sizeof p);
  p.cache.kc = pp.k;
  p.cache.vc = pp.v;
  p.cache.k_block_stride = pp.kc_block;
  p.cache.k_head_stride = pp.kc_head;
  p.cache.v_block_stride = pp.vc_block;
  p.cache.v_head_stride = pp.vc_head;
  p.cache.num_blocks = pp.num_blocks;
  p.cache.block_tables = pp.block_tables;
  p.cache.max_blocks = pp.table_stride;
  p.cache.table_cols = pp.table_cols;
  p.cache.context_lens = pp.context_lens;
  p.cache.scale_log2 = pp.scale_log2;
  p.cache.window_left = pp.win_left;
  p.cache.sinks = pp.sinks;
  p.q = pp.q;
  p.out = pp.out;
  p.q_row = pp.q_row;
  p.q_head = pp.q_head;
  p.o_row = pp.o_row;
  p.o_head = pp.o_head;
  p.total_q = pp.total_q;
  p.cu_q = pp.cu_q;
  p.batch = pp.batch;
  p.Hq = pp.Hq;
  p.Hkv = pp.Hkv;
  p.G = pp.G;
  p.rows_per_group = pp.G <= 16 ? 16 / pp.G : 1;
  p.head_groups = (pp.G + 15) / 16;
  p.row_groups = (pp.max_q + p.rows_per_group - 1) / p.rows_per_group;
  p.listed = (int)row_blocks_of(pp.total_q, pp.batch, p.rows_per_group, p.row_groups);
  p.part_pairs = plan.part_pairs;
  p.num_parts = plan.num_parts;
  p.waves = plan.waves;
  p.part_acc = static_cast<float *>(scratch);
  p.part_ml = p.part_acc + (size_t)plan.num_parts * pp.total_q * pp.Hq * pp.d;
  if (dtype == HIPATTN_F16) dispatch_rows<half_t>(p, pp.d, 1 << pp.block_log2, stream);
  else dispatch_rows<bf16_t>(p, pp.d, 1 << pp.block_log2, stream);
}

}  // namespace hipattn
