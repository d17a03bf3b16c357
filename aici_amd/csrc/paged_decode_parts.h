// The launches of paged decode, partitioned and as one flat split, each with the merge behind it, for all of a context's keys
// (paged_decode.hip) and for a window with sinks (window_decode.hip).  Device code; included by those two.
#pragma once

#include "paged_decode.h"

namespace hipattn {

namespace {

// V2FMT: write partials in the reference's v2 layout (normalised T outputs,
// natural-log maxima) instead of the internal fp32 one.
// BS: tokens per block of the cache; inside, a "block" is a run of 16 tokens whatever BS is.
// KEYS: all of a context, or the runs of it that hold a key its token sees, one after the other.
// WAVES: wavefronts that share a partition.  Eight take a whole context of up to 1024 tokens, their next pair's loads under way
// while the one in hand is folded in, so that no second launch has to merge partitions (see plan_decode).
template <typename T, int HD, bool V2FMT, int BS, int WAVES, typename KEYS = AllKeys>
__global__ __launch_bounds__(WAVES * 64) void paged_decode_kernel(DecodeParams p) {
  typedef typename Vec8<T>::type vec8;
  constexpr int NCH = HD / 8;             // 16-byte chunks per K row
  constexpr int NSTEP = (HD + 31) / 32;   // q.k MFMA steps (32 head elements each)
  constexpr int NDT = HD / 16;            // output tiles of 16 head elements
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int kg = lane >> 4;   // k-group of MFMA operands / row group of results
  const int col = lane & 15;  // operand row (A) or result column (query head)
  // Linear workgroup id -> (partition, sequence, kv head), kv head fastest.
  // Consecutive ids go to the 8 XCDs round-robin; with the kv head fastest
  // every XCD gets the same mix of sequences and partitions (partition-major
  // ids would hand the rarely populated tail partitions to the same XCDs).
  const int hk = p.Hkv * p.col_groups;
  const int kvh = (blockIdx.x % hk) / p.col_groups;
  const int cg = (blockIdx.x % hk) % p.col_groups;
  const int seq = (blockIdx.x / hk) % p.num_seqs;
  const int part = (blockIdx.x / hk) / p.num_seqs;
  // The block-table slice of this partition, one entry per lane, is fetched
  // before the context length is known (rows are zero-padded to max_blocks),
  // so the two round trips overlap.
  const int b0 = part * p.part_blocks;
  const int t0 = b0 * kBlockSize / BS;            // the partition's first table column (b0 is even)
  const int tn = p.part_blocks * kBlockSize / BS;  // and how many it has: at most 64, with 8-token blocks 128
  int tbl = 0, tbl_hi = 0;
  auto load_table = [&](auto column) {
    if (lane < tn && column(t0 + lane) < p.table_cols) tbl = p.block_tables[seq * p.max_blocks + column(t0 + lane)];
    if (BS == 8 && 64 + lane < tn && column(t0 + 64 + lane) < p.table_cols) tbl_hi = p.block_tables[seq * p.max_blocks + column(t0 + 64 + lane)];
  };
  if constexpr (!KEYS::window) load_table([](int c) { return c; });
  const int ctx = min(p.context_lens[seq], p.max_ctx);
  const SeenKeys seen(p, ctx);
  if constexpr (KEYS::window) load_table([&](int c) { return seen.column(c, BS); });
  const int nblk = (ctx + kBlockSize - 1) / kBlockSize - (KEYS::window ? 2 * seen.skip : 0);
  const int g_idx = cg * 16 + col;  // query head within the GQA group
  const bool col_ok = g_idx < p.G;
  const int qh = kvh * p.G + g_idx;
  T *out = static_cast<T *>(p.out);

  if (b0 >= nblk) {
    // Empty partition (uniform over the workgroup).  With a single partition
    // nobody else writes the row.
    if (p.num_parts == 1 && col_ok && wave == 0) {
#pragma unroll
      for (int dt = 0; dt < NDT; dt++)
#pragma unroll
        for (int i = 0; i < 4; i++) out[seq * p.out_stride + (int64_t)qh * HD + dt * 16 + kg * 4 + i] = from_float<T>(0.f);
    }
    return;
  }
  const int b1 = min(b0 + p.part_blocks, nblk);
  const int nb = b1 - b0;

  // Query operand: lane (kg, col) holds q[head col][32*step + 8*kg .. +8].
  vec8 qreg[NSTEP];
  {
    const T *qp = static_cast<const T *>(p.q) + seq * p.q_stride + (int64_t)qh * HD;
#pragma unroll
    for (int s = 0; s < NSTEP; s++) {
      const int ch = 4 * s + kg;
      u32x4_t raw = {0u, 0u, 0u, 0u};
      if (col_ok && ch < NCH) raw = *reinterpret_cast<const u32x4_t *>(qp + ch * 8);
      qreg[s] = bit_cast<vec8>(raw);
    }
  }
  const float slope = (p.alibi != nullptr && col_ok) ? p.alibi[qh] * kLog2e : 0.f;

  const T *kbase = static_cast<const T *>(p.kc) + (int64_t)kvh * p.k_head_stride;
  const T *vbase = static_cast<const T *>(p.vc) + (int64_t)kvh * p.v_head_stride;

  float m_run = -INFINITY;  // running max (log2 domain), uniform per column
  float l_run = 0.f;        // this lane's share of the running sum
  f32x4_t acc[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; dt++) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  auto load = [&](int it, PairRegs<HD> &r) {
    int64_t i0, i1 = 0, i2 = 0, i3 = 0;
    if constexpr (BS == 16) {
      i0 = __builtin_amdgcn_readlane(tbl, it);
      i1 = __builtin_amdgcn_readlane(tbl, it + 1 < nb ? it + 1 : it);
    } else if constexpr (BS == 32) {
      i0 = __builtin_amdgcn_readlane(tbl, it >> 1);
    } else {
      const int c = (2 * it) & 63;  // four columns that never straddle the two registers
      const int src = 2 * it < 64 ? tbl : tbl_hi;
      i0 = __builtin_amdgcn_readlane(src, c);
      i1 = __builtin_amdgcn_readlane(src, c + 1);
      i2 = __builtin_amdgcn_readlane(src, c + 2);
      i3 = __builtin_amdgcn_readlane(src, c + 3);
    }
    pair_load_bs<T, HD, BS>(p, kbase, vbase, i0, i1, i2, i3, r);
  };
  auto fold = [&](int it, PairRegs<HD> &r) {
    pair_compute<T, HD, KEYS>(p, r, KEYS::window ? seen.run(b0 + it) : b0 + it, it + 1 < nb, seen, seen, slope, qreg, m_run, l_run, acc);
  };
  constexpr int STEP = 2 * WAVES;
  if constexpr (WAVES == 4) {
    for (int it = 2 * wave; it < nb; it += STEP) {
      PairRegs<HD> r;
      load(it, r);
      fold(it, r);
    }
  } else {
    PairRegs<HD> ra, rb;
    int it = 2 * wave;
    if (it < nb) load(it, ra);
    for (; it < nb; it += 2 * STEP) {
      if (it + STEP < nb) load(it + STEP, rb);
      fold(it, ra);
      if (it + 2 * STEP < nb) load(it + 2 * STEP, ra);
      if (it + STEP < nb) fold(it + STEP, rb);
    }
  }

  float l_tot = l_run + __shfl_xor(l_run, 16, 64);
  l_tot += __shfl_xor(l_tot, 32, 64);

  // Merge the wavefronts' states: common maximum, rescale, sum into wave 0.
  __shared__ float s_m[WAVES][16];
  __shared__ float s_l[WAVES][16];
  __shared__ f32x4_t s_acc[WAVES - 1][NDT][64];
  if (kg == 0) s_m[wave][col] = m_run;
  __syncthreads();
  float m_all = s_m[0][col];
#pragma unroll
  for (int w = 1; w < WAVES; w++) m_all = fmaxf(m_all, s_m[w][col]);
  const float m_all_safe = m_all == -INFINITY ? 0.f : m_all;
  const float wscale = fast_exp2(m_run - m_all_safe);  // 0 for a wave that saw no token
  l_tot *= wscale;
  if (kg == 0) s_l[wave][col] = l_tot;
  if (wave > 0) {
#pragma unroll
    for (int dt = 0; dt < NDT; dt++) s_acc[wave - 1][dt][lane] = acc[dt] * wscale;
  }
  __syncthreads();
  if (wave > 0 || !col_ok) return;
  m_run = m_all;
  l_tot = s_l[0][col];
#pragma unroll
  for (int w = 1; w < WAVES; w++) l_tot += s_l[w][col];
#pragma unroll
  for (int dt = 0; dt < NDT; dt++) {
    acc[dt] = acc[dt] * wscale;
#pragma unroll
    for (int w = 0; w < WAVES - 1; w++) acc[dt] = acc[dt] + s_acc[w][dt][lane];
  }

  if (p.num_parts == 1) {
    const float inv = l_tot > 0.f ? 1.0f / l_tot : 0.f;
    T *op = out + seq * p.out_stride + (int64_t)qh * HD + kg * 4;
#pragma unroll
    for (int dt = 0; dt < NDT; dt++) {
      T r[4];
#pragma unroll
      for (int i = 0; i < 4; i++) r[i] = from_float<T>(acc[dt][i] * inv);
      *reinterpret_cast<u32x2_t *>(op + dt * 16) = *reinterpret_cast<u32x2_t *>(r);
    }
    return;
  }

  const int64_t pidx = ((int64_t)seq * p.Hq + qh) * p.num_parts + part;
  if (V2FMT) {
    const float inv = l_tot > 0.f ? 1.0f / l_tot : 0.f;
    T *tp = static_cast<T *>(p.tmp_out) + pidx * HD + kg * 4;
#pragma unroll
    for (int dt = 0; dt < NDT; dt++) {
      T r[4];
#pragma unroll
      for (int i = 0; i < 4; i++) r[i] = from_float<T>(acc[dt][i] * inv);
      *reinterpret_cast<u32x2_t *>(tp + dt * 16) = *reinterpret_cast<u32x2_t *>(r);
    }
    if (kg == 0) {
      p.ws_m[pidx] = m_run * kLn2;
      p.ws_l[pidx] = l_tot;
    }
  } else {
    float *ap = p.ws_acc + pidx * HD + kg * 4;
#pragma unroll
    for (int dt = 0; dt < NDT; dt++) *reinterpret_cast<f32x4_t *>(ap + dt * 16) = acc[dt];
    if (kg == 0) {
      p.ws_m[pidx] = m_run;
      p.ws_l[pidx] = l_tot;
    }
  }
}

// Merge of the partitions of one (sequence, query head): grid (Hq, S).  A long context of a small batch
// is cut into hundreds of partitions (the main launch wants a few thousand workgroups), so the merge is
// spread over the workgroup: thread (slice, d) sums the partitions slice, slice + SLICES, ... of head element
// d, four loads in flight, and the slices meet in LDS (one slice when there are few partitions).
template <typename T, int HD, bool V2FMT, int THREADS, typename KEYS = AllKeys>
__global__ __launch_bounds__(THREADS) void paged_decode_reduce_kernel(DecodeParams p) {
  constexpr int HDT = HD <= 64 ? 64 : (HD <= 128 ? 128 : 256);  // threads per slice
  static_assert(THREADS % HDT == 0 && THREADS % 64 == 0, "whole slices, whole wavefronts");
  constexpr int SLICES = THREADS / HDT;
  constexpr int WAVES = THREADS / 64;
  __shared__ float s_red[WAVES];
  __shared__ float s_o[SLICES][HDT];
  const int qh = blockIdx.x, seq = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int ctx = min(p.context_lens[seq], p.max_ctx);
  const int nblk = (ctx + kBlockSize - 1) / kBlockSize - (KEYS::window ? 2 * SeenKeys(p, ctx).skip : 0);
  const int np = (nblk + p.part_blocks - 1) / p.part_blocks;  // partitions that ran
  const int64_t base = ((int64_t)seq * p.Hq + qh) * p.num_parts;
  T *op = static_cast<T *>(p.out) + seq * p.out_stride + (int64_t)qh * HD;
  const float mscale = V2FMT ? kLog2e : 1.0f;  // v2 maxima are natural-log
  auto block_reduce = [&](float v, bool is_max) -> float {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float t = __shfl_xor(v, o, 64);
      v = is_max ? fmaxf(v, t) : v + t;
    }
    __syncthreads();  // s_red may still be read from the previous reduction
    if (lane == 0) s_red[wave] = v;
    __syncthreads();
    v = s_red[0];
#pragma unroll
    for (int i = 1; i < WAVES; i++) v = is_max ? fmaxf(v, s_red[i]) : v + s_red[i];
    return v;
  };
  float mmax = -INFINITY;
  for (int i = tid; i < np; i += THREADS) mmax = fmaxf(mmax, p.ws_m[base + i] * mscale);
  mmax = block_reduce(mmax, true);
  float denom = 0.f;
  for (int i = tid; i < np; i += THREADS) denom += p.ws_l[base + i] * fast_exp2(p.ws_m[base + i] * mscale - mmax);
  denom = block_reduce(denom, false);
  const float inv = denom > 0.f ? 1.0f / denom : 0.f;
  const int slice = tid / HDT, d = tid % HDT;
  float o = 0.f;
  if (d < HD) {
#pragma unroll 4
    for (int i = slice; i < np; i += SLICES) {
      const float w = fast_exp2(p.ws_m[base + i] * mscale - mmax);
      if (V2FMT)
        o += to_float(static_cast<const T *>(p.tmp_out)[(base + i) * HD + d]) * (w * p.ws_l[base + i]);
      else
        o += p.ws_acc[(base + i) * HD + d] * w;
    }
  }
  s_o[slice][d] = o;
  __syncthreads();
  if (slice == 0 && d < HD) {
#pragma unroll
    for (int k = 1; k < SLICES; k++) o += s_o[k][d];
    op[d] = from_float<T>(o * inv);
  }
}

// The same for at most PARTS partitions: everything a thread needs is asked for at once -- the maxima, the sums and its
// element of every partition, also of those beyond this context's, which are left out of the sums -- instead of in four
// dependent steps.  (1 x 700 tokens: 9.0 -> 7.7 us with the launch in front; 1 x 2048: 9.4 -> 8.9.)
template <typename T, int HD, bool V2FMT, int PARTS, typename KEYS = AllKeys>
__global__ __launch_bounds__(HD <= 64 ? 64 : (HD <= 128 ? 128 : 256)) void paged_decode_reduce_few_kernel(DecodeParams p) {
  const int qh = blockIdx.x, seq = blockIdx.y, d = threadIdx.x;
  const int64_t base = ((int64_t)seq * p.Hq + qh) * p.num_parts;
  const float mscale = V2FMT ? kLog2e : 1.0f;
  const int len = p.context_lens[seq];
  float m[PARTS], l[PARTS], a[PARTS];
#pragma unroll
  for (int i = 0; i < PARTS; i++) {
    m[i] = l[i] = a[i] = 0.f;
    if (i < p.num_parts) {
      m[i] = p.ws_m[base + i];
      l[i] = p.ws_l[base + i];
      if (d < HD)
        a[i] = V2FMT ? to_float(static_cast<const T *>(p.tmp_out)[(base + i) * HD + d]) : p.ws_acc[(base + i) * HD + d];
    }
  }
  const int ctx = min(len, p.max_ctx);
  const int nblk = (ctx + kBlockSize - 1) / kBlockSize - (KEYS::window ? 2 * SeenKeys(p, ctx).skip : 0);
  const int np = (nblk + p.part_blocks - 1) / p.part_blocks;  // partitions that ran
  float mmax = -INFINITY;
#pragma unroll
  for (int i = 0; i < PARTS; i++)
    if (i < np) mmax = fmaxf(mmax, m[i] * mscale);
  float denom = 0.f, o = 0.f;
#pragma unroll
  for (int i = 0; i < PARTS; i++)
    if (i < np) {
      const float w = fast_exp2(m[i] * mscale - mmax), wl = w * l[i];
      denom += wl;
      o += a[i] * (V2FMT ? wl : w);
    }
  const float inv = denom > 0.f ? 1.0f / denom : 0.f;
  if (d < HD) static_cast<T *>(p.out)[seq * p.out_stride + (int64_t)qh * HD + d] = from_float<T>(o * inv);
}

template <typename T, int HD, bool V2FMT, int BS, typename KEYS = AllKeys>
void launch_decode(const DecodeParams &p, int64_t S, hipStream_t stream) {
  const int64_t n_wg = (int64_t)p.num_parts * p.Hkv * p.col_groups * S;
  HA_CHECK(n_wg <= 0x7fffffff, "paged_attention: too many workgroups");
  dim3 grid((unsigned)n_wg);
  if constexpr (!V2FMT && HD <= 128) {
    if (p.waves == 8) {
      paged_decode_kernel<T, HD, V2FMT, BS, 8, KEYS><<<grid, 512, 0, stream>>>(p);
      check_launch("paged_attention");
      return;
    }
  }
  paged_decode_kernel<T, HD, V2FMT, BS, 4, KEYS><<<grid, 256, 0, stream>>>(p);
  check_launch("paged_attention");
  if (p.num_parts > 1) {
    constexpr int kThreads = HD <= 64 ? 64 : (HD <= 128 ? 128 : 256);
    const dim3 rows((unsigned)p.Hq, (unsigned)S);
    if (p.num_parts <= 8)
      paged_decode_reduce_few_kernel<T, HD, V2FMT, 8, KEYS><<<rows, kThreads, 0, stream>>>(p);
    else if (p.num_parts <= 16)
      paged_decode_reduce_few_kernel<T, HD, V2FMT, 16, KEYS><<<rows, kThreads, 0, stream>>>(p);
    else
      paged_decode_reduce_kernel<T, HD, V2FMT, 512, KEYS><<<rows, 512, 0, stream>>>(p);
    check_launch("paged_attention reduce");
  }
}

template <typename T, int HD, int BS, typename KEYS = AllKeys>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void paged_decode_flat_kernel(DecodeParams p) {
  __shared__ FlatLds<HD> lds;
  decode_flat<T, HD, BS, KEYS>(p, blockIdx.x, lds);
}

template <typename T, int HD>
__global__ __launch_bounds__(128) void paged_decode_flat_reduce_kernel(DecodeParams p) {
  decode_flat_merge<T, HD>(p, blockIdx.x, blockIdx.y);
}

template <typename T, int HD, typename KEYS = AllKeys>
void launch_decode_flat(DecodeParams p, const DecodePlan &pl, int block_size, char *ws, hipStream_t stream) {
  flat_scratch_set(p, pl.flat_scratch, pl.flat_wgs, HD, ws);
  // the three instances differ in their address arithmetic only: what the device holds of one it holds of all
  switch (block_size) {
    case 8: paged_decode_flat_kernel<T, HD, 8, KEYS><<<dim3((unsigned)pl.flat_wgs), 256, 0, stream>>>(p); break;
    case 32: paged_decode_flat_kernel<T, HD, 32, KEYS><<<dim3((unsigned)pl.flat_wgs), 256, 0, stream>>>(p); break;
    default: paged_decode_flat_kernel<T, HD, kBlockSize, KEYS><<<dim3((unsigned)pl.flat_wgs), 256, 0, stream>>>(p); break;
  }
  check_launch("paged_attention");
  paged_decode_flat_reduce_kernel<T, HD><<<dim3((unsigned)p.Hq, (unsigned)p.num_seqs), HD <= 64 ? 64 : 128, 0, stream>>>(p);
  check_launch("paged_attention reduce");
}

}  // namespace
}  // namespace hipattn
