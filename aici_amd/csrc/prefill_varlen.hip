// Varlen (packed, ragged) flash-attention forward for gfx950.  Replaces the
// reference's mha_varlen_fwd (rllm/tch-cuda/kernels/flash_attn/flash_api.cpp:
// 447-655 and flash_fwd_kernel.h:590-1136) with a design laid out for CDNA4.
// Two kernels here share the mathematics (a third, for GQA launches of many workgroups, is in prefill_r3.hip):
//
//  * prefill_varlen_w8_kernel (head sizes up to 128, causal or unmasked): 8 wavefronts own 256 query rows, two
//    per SIMD, over 64-key tiles.  From rows of k / v, and from the paged cache where a block image can go
//    into LDS as it is, the tiles are copied global -> LDS without staging registers into five LDS stages and
//    the two wavefronts of a SIMD alternate between a block of MFMAs and a block of softmax; where images
//    cannot be copied as they are (head sizes below 32, or on request) the tiles of the paged cache are staged
//    through registers in one software-pipelined loop per wavefront over three stages.  Described at its
//    definition.
//  * prefill_varlen_kernel (head sizes up to 256, sliding windows): a workgroup
//    of 4 wavefronts owns 128 or 256 query rows of one (sequence, query head);
//    each wavefront keeps QT tiles of 32 query rows, their Q operands and their
//    fp32 output accumulators in registers; K and V tiles of 64 keys are staged
//    through LDS in double buffers; V stays row-major in LDS and the transposed
//    A operand of the second product comes from ds_read_b64_tr_b16.
//
// Common to both:
//  * both products run on v_mfma_f32_32x32x16 in the transposed orientation:
//    S^T = K.Q^T puts one query per lane column, so the softmax row maximum and
//    sum are in-lane loops plus a single cross-lane exchange, and the
//    accumulator layout of S^T is already the B-operand layout of
//    O^T = V^T.P^T (no shuffles between the two products);
//  * GQA: query head h reads kv head h / (Hq/Hkv); heads of one group are
//    scheduled onto the same XCD so the K/V tiles they share stay in that
//    XCD's L2;
//  * causal masking is bottom-right aligned (key j visible to query i iff
//    j <= i + Lk - Lq, flash_attn/softmax.h:159-160); tiles past the diagonal
//    are skipped, only tiles crossing it or the end of the keys are masked.
//
// Numerics follow the reference kernel: fp32 scores and accumulators, softmax
// in base 2 with scale*log2(e) folded in, un-normalised probabilities rounded
// to the input dtype as the second product's operand, division by the fp32 sum
// of the unrounded probabilities at the end.  One deliberate difference: the
// row maximum used as the exponent's reference is only moved when a row
// outgrows it by more than 2^8, which saves rescaling the accumulators on
// nearly every tile; probabilities then range up to 256 instead of 1, so the
// largest one is no longer exactly 1.0 and carries the operand's rounding
// error (2^-9 relative in bf16, 2^-12 in fp16); the normaliser is given the
// same rounding for each half-tile's largest term so that it cancels where it
// matters, on rows that one key dominates.
#include "prefill_w8.h"

namespace hipattn {

namespace {

// Row strides of the LDS tiles in elements.  K is read as 16 B per lane with
// 16 consecutive rows per access phase, V as 64 B runs of 4 consecutive rows;
// the paddings make those phases hit distinct banks.
template <int HDP>
struct Tile {
  static constexpr int KSTR = HDP + 8;
  static constexpr int VSTR = (HDP % 64 == 32) ? HDP : HDP + 32;
  static constexpr int K_ELEMS = BN * KSTR;
  static constexpr int V_ELEMS = BN * VSTR;
  static constexpr int VTSTR = BN + 8;  // paged form: V^T rows (head-element-major), 64 keys + 16 B
  static constexpr int VT_ELEMS = HDP * VTSTR;
  static constexpr int STAGE_ELEMS = K_ELEMS + (V_ELEMS > VT_ELEMS ? V_ELEMS : VT_ELEMS);
  static constexpr size_t LDS_BYTES = 2 * (size_t)STAGE_ELEMS * 2;
};

typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;

// PAGED: K and V are the paged caches, read through the block table (p.block_tables, p.context_lens); tiles
// are staged in the caches' own order -- 16-byte runs of K go to the rows they belong to, 16-byte runs of V (8
// tokens of one head element) to rows of a V^T tile, whose operands plain 8-byte LDS reads deliver.
// SINKS (paged, causal, win_left >= 0): the first p.sinks keys of a sequence are seen beside the window; tiles are numbered without the
// gap between them, as in prefill_varlen_w8_kernel.
template <typename T, int HDP, int QT, bool PAGED = false, bool SINKS = false>
__global__ __launch_bounds__(256) void prefill_varlen_kernel(PrefillParams p) {
  static_assert(PAGED || !SINKS, "sinks: the paged form alone");
  typedef typename Vec8<T>::type vec8;
  typedef Tile<HDP> TL;
  constexpr int KSTEPS = HDP / 16;  // contraction steps of S^T = K.Q^T
  constexpr int NDT = HDP / 32;     // 32-row tiles of O^T
  constexpr int CPR = HDP / 8;      // 16-byte chunks per tile row
  constexpr int NLOAD = CPR / 4;    // chunks per thread per tile (BN*CPR/256)
  constexpr int BM = 4 * QT * 32;

  extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
  T *smem = reinterpret_cast<T *>(smem_raw);

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int g = lane >> 5;   // k-group of 32x32x16 operands
  const int c = lane & 31;   // operand row / result column

  // Linear workgroup id -> (query block, sequence, head).  Heavy (late) query
  // blocks first; heads interleaved so that one GQA group shares an XCD.
  int id = blockIdx.x;
  const int slot = id % p.Hq;
  id /= p.Hq;
  RowBlock blk = {0, 0, 0, 0};
  const bool listed = SINKS && p.row_blocks > 0;
  if constexpr (SINKS)
    if (listed) {
      blk = row_block_of(p.cu_q, p.context_lens, p.win_left / 2, p.batch, BM, p.n_qblocks, id);
      if (blk.block < 0) return;
    }
  const int b = listed ? blk.seq : id % p.batch;
  const int qb = listed ? blk.block : p.n_qblocks - 1 - id / p.batch;
  const int h = (slot % p.Hkv) * p.G + slot / p.Hkv;
  const int kvh = h / p.G;

  const int q_begin = listed ? blk.begin : p.cu_q[b];
  const int Lq = listed ? blk.rows : p.cu_q[b + 1] - q_begin;
  const int k_begin = PAGED ? 0 : p.cu_k[b];
  int Lk = PAGED ? p.context_lens[b] : p.cu_k[b + 1] - k_begin;
  if (!PAGED && p.seqused_k) Lk = min(Lk, p.seqused_k[b]);
  const int wg_row0 = qb * BM;
  if (wg_row0 >= Lq) return;
  int off = Lk - Lq;  // bottom-right alignment of the mask
  const int wg_last_row = min(wg_row0 + BM, Lq) - 1;
  const bool bound_hi = p.win_right >= 0, bound_lo = p.win_left >= 0;
  int kmax = bound_hi ? min((int64_t)Lk, (int64_t)wg_last_row + off + p.win_right + 1) : Lk;
  if (kmax < 0) kmax = 0;
  int n_tiles = (kmax + BN - 1) / BN;
  // SINKS: tile t is the context's tile t, from gap_tile on tile t + skip; Lk, off and keys are counted that way, and keys from p.sinks to
  // seen_from are seen by no row of the workgroup.
  int gap_tile = 0, skip = 0, seen_from = 0;
  if constexpr (SINKS) {
    seen_from = max(wg_row0 + off - p.win_left, 0);
    gap_tile = (min(p.sinks, seen_from) + BN - 1) / BN;
    skip = max(seen_from / BN - gap_tile, 0);
    n_tiles -= skip;
    Lk -= skip * BN;
    off -= skip * BN;
    seen_from -= skip * BN;
  }
  // first tile that any row of the workgroup can see
  const int first_tile = SINKS ? 0 : bound_lo ? (int)max((int64_t)0, ((int64_t)wg_row0 + off - p.win_left)) / BN : 0;

  const int wave_row0 = wg_row0 + wave * (QT * 32);
  const int wave_last_row = wave_row0 + QT * 32 - 1;

  const T *qp = static_cast<const T *>(p.q) + (int64_t)q_begin * p.q_row + (int64_t)h * p.q_head;
  const T *kp = static_cast<const T *>(p.k) + (PAGED ? (int64_t)kvh * p.kc_head : (int64_t)k_begin * p.k_row + (int64_t)kvh * p.k_head);
  const T *vp = static_cast<const T *>(p.v) + (PAGED ? (int64_t)kvh * p.vc_head : (int64_t)k_begin * p.v_row + (int64_t)kvh * p.v_head);
  const int d_chunks = p.d / 8;

  // Q operands: lane (g, c) of tile qt holds q[row][16ks + 8g .. +8].
  vec8 qreg[QT][KSTEPS];
#pragma unroll
  for (int qt = 0; qt < QT; qt++) {
    const int row = wave_row0 + qt * 32 + c;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ks++) {
      u32x4_t raw = {0u, 0u, 0u, 0u};
      const int ch = 2 * ks + g;
      if (row < Lq && ch < d_chunks) raw = *reinterpret_cast<const u32x4_t *>(qp + (int64_t)row * p.q_row + ch * 8);
      qreg[qt][ks] = bit_cast<vec8>(raw);
    }
  }

  f32x16_t acc[QT][NDT];
#pragma unroll
  for (int qt = 0; qt < QT; qt++)
#pragma unroll
    for (int dt = 0; dt < NDT; dt++)
#pragma unroll
      for (int i = 0; i < 16; i++) acc[qt][dt][i] = 0.f;
  float m_run[QT], l_run[QT];
#pragma unroll
  for (int qt = 0; qt < QT; qt++) {
    m_run[qt] = -INFINITY;
    l_run[qt] = 0.f;
  }

  // Tile staging: thread t moves chunk (t + 256 i) of the tile.
  u32x4_t kst[NLOAD], vst[NLOAD];
  int staged_k0 = 0;  // first key of the tile held in the staging registers (paged form)
  const int32_t *table_row = PAGED ? p.block_tables + (int64_t)b * p.table_stride : nullptr;
  auto load_tile = [&](int tile) {
    const int k0 = tile * BN;
    if constexpr (PAGED) {
      // Units in the caches' own order, so that consecutive threads read consecutive 16-byte runs: K unit
      // (block r, chunk, token), V unit (block r, head element, half of the block's tokens).  Blocks past the
      // context re-read its last one (their keys are masked, their V runs cleared before they reach LDS).
      staged_k0 = k0;
      const int past = SINKS && tile >= gap_tile ? skip * BN : 0;  // keys of the gap in front of this tile
      if (p.block_log2 != 4) {
        // Caches of 8- or 32-token blocks: the same units -- a 16-byte run of K is (chunk, token) and one of V
        // (head element, 8 tokens) at any block size -- each finding its own block: the id comes from the
        // table row per unit, and the block's pitch takes the place of the 16.
        const int bl = p.block_log2, bs = 1 << bl;
        const int last_col = max(min((Lk - 1 + past) >> bl, p.table_cols - 1), 0);
        auto block_of = [&](int pos) -> int64_t {
          const int id = table_row[min((pos + past) >> bl, last_col)];
          return id < 0 ? 0 : (id >= p.num_blocks ? p.num_blocks - 1 : (int64_t)id);
        };
        constexpr int K_PER_16 = CPR * 16, V_PER_16 = HDP * 2;
#pragma unroll
        for (int i = 0; i < NLOAD; i++) {
          const int u = tid + 256 * i;
          {
            const int r = u / K_PER_16, rem = u % K_PER_16;
            const int ch = min(rem / 16, d_chunks - 1), pos = k0 + r * 16 + rem % 16;
            kst[i] = *reinterpret_cast<const u32x4_t *>(kp + block_of(pos) * p.kc_block + ((ch << bl) + (pos & (bs - 1))) * 8);
          }
          {
            const int r = u / V_PER_16, rem = u % V_PER_16;
            const int drow = min(rem / 2, p.d - 1), pos = k0 + r * 16 + (rem % 2) * 8;
            vst[i] = *reinterpret_cast<const u32x4_t *>(vp + block_of(pos) * p.vc_block + (drow << bl) + (pos & (bs - 1)));
          }
        }
        return;
      }
      const int last_col = max(min((Lk - 1 + past) >> 4, p.table_cols - 1), 0);
      int64_t blk[4];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int id = table_row[min(((k0 + past) >> 4) + r, last_col)];
        blk[r] = id < 0 ? 0 : (id >= p.num_blocks ? p.num_blocks - 1 : (int64_t)id);
      }
      constexpr int K_PER_BLOCK = CPR * 16, V_PER_BLOCK = HDP * 2;
#pragma unroll
      for (int i = 0; i < NLOAD; i++) {
        const int u = tid + 256 * i;
        {
          const int r = u / K_PER_BLOCK, rem = u % K_PER_BLOCK;
          const int ch = min(rem / 16, d_chunks - 1), tok = rem % 16;
          kst[i] = *reinterpret_cast<const u32x4_t *>(kp + blk[r] * p.kc_block + (ch * 16 + tok) * 8);
        }
        {
          const int r = u / V_PER_BLOCK, rem = u % V_PER_BLOCK;
          const int drow = min(rem / 2, p.d - 1), half = rem % 2;
          vst[i] = *reinterpret_cast<const u32x4_t *>(vp + blk[r] * p.vc_block + drow * 16 + half * 8);
        }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < NLOAD; i++) {
      const int idx = tid + 256 * i;
      const int row = idx / CPR, ch = idx % CPR;
      const int key = k0 + row;
      kst[i] = u32x4_t{0u, 0u, 0u, 0u};
      vst[i] = u32x4_t{0u, 0u, 0u, 0u};
      if (key < Lk && ch < d_chunks) {
        kst[i] = *reinterpret_cast<const u32x4_t *>(kp + (int64_t)key * p.k_row + ch * 8);
        vst[i] = *reinterpret_cast<const u32x4_t *>(vp + (int64_t)key * p.v_row + ch * 8);
      }
    }
  };
  auto store_tile = [&](int stage) {
    T *ks = smem + stage * TL::STAGE_ELEMS;
    T *vs = ks + TL::K_ELEMS;
    if constexpr (PAGED) {
      constexpr int K_PER_BLOCK = CPR * 16, V_PER_BLOCK = HDP * 2;
#pragma unroll
      for (int i = 0; i < NLOAD; i++) {
        const int u = tid + 256 * i;
        {
          const int r = u / K_PER_BLOCK, rem = u % K_PER_BLOCK;
          // (chunks past d carry a copy of the last real one: they meet the zeros of Q)
          *reinterpret_cast<u32x4_t *>(ks + (r * 16 + rem % 16) * TL::KSTR + (rem / 16) * 8) = kst[i];
        }
        {
          const int r = u / V_PER_BLOCK, rem = u % V_PER_BLOCK;
          const int drow = rem / 2, half = rem % 2;
          u32x4_t o = vst[i];
          // Cache tokens past the context hold whatever was there before (possibly NaN, which a zero
          // probability would not neutralise): clear them.
          if (staged_k0 + BN > Lk) {
            const int alive = Lk - (staged_k0 + r * 16 + half * 8);  // keys of this run inside the context
#pragma unroll
            for (int w = 0; w < 4; w++) {
              const int a2 = alive - 2 * w;
              o[w] &= a2 <= 0 ? 0u : (a2 == 1 ? 0xffffu : 0xffffffffu);
            }
          }
          if (SINKS && staged_k0 < seen_from && staged_k0 + BN > p.sinks) {  // ... and those between the sinks and the window
#pragma unroll
            for (int w = 0; w < 4; w++) {
              const int t = staged_k0 + r * 16 + half * 8 + 2 * w;
              o[w] &= (t >= p.sinks && t < seen_from ? 0u : 0xffffu) | (t + 1 >= p.sinks && t + 1 < seen_from ? 0u : 0xffff0000u);
            }
          }
          *reinterpret_cast<u32x4_t *>(vs + drow * TL::VTSTR + r * 16 + half * 8) = o;
        }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < NLOAD; i++) {
      const int idx = tid + 256 * i;
      const int row = idx / CPR, ch = idx % CPR;
      *reinterpret_cast<u32x4_t *>(ks + row * TL::KSTR + ch * 8) = kst[i];
      *reinterpret_cast<u32x4_t *>(vs + row * TL::VSTR + ch * 8) = vst[i];
    }
  };

  if (n_tiles > first_tile) {
    load_tile(first_tile);
    store_tile(first_tile & 1);
    if (n_tiles > first_tile + 1) load_tile(first_tile + 1);
  }
  __syncthreads();

  // Per-lane LDS offsets (elements).
  const int k_lane_off = c * TL::KSTR + g * 8;
  const int rh = (lane >> 4) & 1, li = lane & 15;
  const int v_lane_off = (4 * g + (li >> 2)) * TL::VSTR + 16 * rh + 4 * (li & 3);

  for (int j = first_tile; j < n_tiles; j++) {
    const int cur = j & 1;
    if (j + 1 < n_tiles) store_tile(cur ^ 1);
    if (j + 2 < n_tiles) load_tile(j + 2);

    const int k0 = j * BN;
    // Wave-level view of this tile: skip it if it lies entirely outside the
    // window of every row this wave owns.
    const bool unseen = (wave_row0 >= Lq) || (bound_hi && k0 > (int64_t)wave_last_row + off + p.win_right) ||
                      (bound_lo && k0 + BN - 1 < (int64_t)wave_row0 + off - p.win_left && (!SINKS || k0 >= p.sinks));
    if (!unseen) {
      const T *ks_base = smem + cur * TL::STAGE_ELEMS;
      const T *vs_base = ks_base + TL::K_ELEMS;
      const bool need_mask = (k0 + BN > Lk) || (bound_hi && k0 + BN - 1 > (int64_t)wave_row0 + off + p.win_right) ||
                             (bound_lo && k0 < (int64_t)wave_last_row + off - p.win_left);

      // S^T = K . Q^T for the 32 keys of half-tile hf: rows = keys, one query per lane column.
      auto qk = [&](int hf, f32x16_t(&s)[QT]) {
        const f32x16_t zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ks++) {
          const vec8 a = *reinterpret_cast<const vec8 *>(ks_base + k_lane_off + hf * 32 * TL::KSTR + ks * 16);
#pragma unroll
          for (int qt = 0; qt < QT; qt++) s[qt] = Mfma32<T>::run(a, qreg[qt][ks], ks == 0 ? zero : s[qt]);
        }
      };
      // Mask, running maximum with lazy rescaling, exponentials; leaves the B operands of the
      // second product in pk.  The reference maximum m_ref (log2 domain) only moves when a
      // row's maximum exceeds it by more than kRescaleThreshold, so probabilities stay below
      // 2^kRescaleThreshold and the accumulators are rarely touched by the vector ALU.
      auto softmax = [&](int hf, f32x16_t(&s)[QT], vec8(&pk)[QT][2]) {
#pragma unroll
        for (int qt = 0; qt < QT; qt++) {
          if (need_mask) {
            const int row = wave_row0 + qt * 32 + c;
            const int limit = bound_hi ? (int)min((int64_t)Lk - 1, (int64_t)row + off + p.win_right) : Lk - 1;
            const int first = bound_lo ? (int)max((int64_t)0, (int64_t)row + off - p.win_left) : 0;
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const int key = k0 + hf * 32 + (i >> 2) * 8 + g * 4 + (i & 3);
              if (key > limit || (key < first && (!SINKS || key >= p.sinks))) s[qt][i] = -INFINITY;
            }
          }
          float mx = s[qt][0];
#pragma unroll
          for (int i = 1; i < 16; i++) mx = fmaxf(mx, s[qt][i]);
          mx = max_across_halves(mx) * p.scale_log2;
          const bool grow = mx > m_run[qt] + p.rescale_thr;
          if (__builtin_expect(__any(grow), 0)) {
            const float m_new = grow ? mx : m_run[qt];
            // exp2(-inf - finite) = 0 on a row's first keys; rows that do not grow keep 1
            // (their m_run may still be -inf, and -inf - -inf is not a number).
            const float alpha = grow ? fast_exp2(m_run[qt] - m_new) : 1.0f;
            l_run[qt] *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; dt++) {
              // Pin the accumulator tile to the accumulation registers at this point, so the
              // copies the multiply needs are made here, inside the rarely taken branch,
              // and not hoisted into every iteration.
              asm volatile("" : "+a"(acc[qt][dt]));
              acc[qt][dt] *= alpha;
            }
            m_run[qt] = m_new;
          }
          const float msub = m_run[qt] == -INFINITY ? 0.f : m_run[qt];
          // The row's largest probability of this half-tile enters the second product
          // rounded to T; when one key dominates, that rounding is the whole error of the
          // row.  Put the same rounding into the normaliser (once per row: lane group 0).
          // It is exactly zero whenever the maximum is the reference itself (p = 1).
          const float pmax = fast_exp2(mx - msub);
          float psum = g == 0 ? to_float(from_float<T>(pmax)) - pmax : 0.f;
#pragma unroll
          for (int half = 0; half < 2; half++) {
            vec8 v;
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const float e = fast_exp2(s[qt][half * 8 + i] * p.scale_log2 - msub);
              psum += e;
              v[i] = from_float<T>(e);
            }
            pk[qt][half] = v;
          }
          l_run[qt] += psum;
        }
      };
      // O^T += V^T . P^T over the 32 keys of half-tile hf.
      auto pv = [&](int hf, vec8(&pk)[QT][2]) {
#pragma unroll
        for (int dt = 0; dt < NDT; dt++)
#pragma unroll
          for (int half = 0; half < 2; half++) {
            s16x4_t lo, hi;
            if constexpr (PAGED) {
              // V^T rows: head element dt * 32 + c, keys 4 g .. + 4 of the 16-key step and 8 further on
              const T *vptr = vs_base + (dt * 32 + c) * TL::VTSTR + hf * 32 + half * 16 + 4 * g;
              lo = *reinterpret_cast<const s16x4_t *>(vptr);
              hi = *reinterpret_cast<const s16x4_t *>(vptr + 8);
            } else {
              const T *vptr = vs_base + v_lane_off + (hf * 32 + half * 16) * TL::VSTR + dt * 32;
              lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vptr));
              hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vptr + 8 * TL::VSTR));
            }
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            const s16x8 av = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            const vec8 a = bit_cast<vec8>(av);
#pragma unroll
            for (int qt = 0; qt < QT; qt++) acc[qt][dt] = Mfma32<T>::run(a, pk[qt][half], acc[qt][dt]);
          }
      };

      f32x16_t s0[QT], s1[QT];
      vec8 p0[QT][2], p1[QT][2];
      qk(0, s0);
      softmax(0, s0, p0);
      pv(0, p0);
      qk(1, s1);
      softmax(1, s1, p1);
      pv(1, p1);
    }
    __syncthreads();
  }

  // ---- epilogue: normalise and store --------------------------------------
  T *op = static_cast<T *>(p.out) + (int64_t)q_begin * p.o_row + (int64_t)h * p.o_head;
  float *op32 = static_cast<float *>(p.out) + (int64_t)q_begin * p.o_row + (int64_t)h * p.o_head;
#pragma unroll
  for (int qt = 0; qt < QT; qt++) {
    const int row = wave_row0 + qt * 32 + c;
    const float l_tot = l_run[qt] + __shfl_xor(l_run[qt], 32, 64);
    if (row >= Lq) continue;
    const float inv = l_tot > 0.f ? 1.0f / l_tot : 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; dt++)
#pragma unroll
      for (int a = 0; a < 4; a++) {
        const int dcol = dt * 32 + a * 8 + g * 4;
        if (dcol < p.d && p.out_f32) {
          f32x4_t r;
#pragma unroll
          for (int i = 0; i < 4; i++) r[i] = acc[qt][dt][a * 4 + i] * inv;
          *reinterpret_cast<f32x4_t *>(op32 + (int64_t)row * p.o_row + dcol) = r;
        } else if (dcol < p.d) {
          T r[4];
#pragma unroll
          for (int i = 0; i < 4; i++) r[i] = from_float<T>(acc[qt][dt][a * 4 + i] * inv);
          *reinterpret_cast<u32x2_t *>(op + (int64_t)row * p.o_row + dcol) = *reinterpret_cast<u32x2_t *>(r);
        }
      }
    if (p.lse != nullptr && g == 0 && row < p.lse_pitch) {
      // Natural-log sum-exp of the scaled scores; +inf for a row without keys
      // (flash_fwd_kernel.h:629-668).
      const float lse = l_tot > 0.f ? (m_run[qt] + __builtin_amdgcn_logf(l_tot)) * kLn2 : INFINITY;
      p.lse[((int64_t)b * p.Hq + h) * p.lse_pitch + row] = lse;
    }
  }
}

// hl: log2 of the query heads per workgroup.
template <typename T, int HDP, int MODE, int NW>
void launch_prefill_nw(PrefillParams p, int hl, hipStream_t stream) {
  static bool attr_set = false;  // benign race: setting twice is harmless
  auto kernel = prefill_varlen_w8_kernel<T, HDP, MODE, PrefillAlone, NW>;
  constexpr size_t lds_bytes = MODE == W8_PAGED ? TileW8<HDP>::LDS_BYTES : (size_t)w8_stages(HDP, NW) * 2 * BN * HDP * 2;
  if (!attr_set) {
    HA_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)lds_bytes));
    attr_set = true;
  }
  p.wg_heads_log2 = hl;
  const int bm = (NW * 32) >> hl;
  p.n_qblocks = (p.max_q + bm - 1) / bm;
  const int64_t n_wg = (int64_t)p.n_qblocks * p.batch * (p.Hq >> hl);
  HA_CHECK(n_wg <= 0x7fffffff, "mha_varlen_fwd: too many workgroups");
  kernel<<<dim3((unsigned)n_wg), NW * 64, lds_bytes, stream>>>(p);
  check_launch("mha_varlen_fwd");
}

// Whether a launch takes workgroups of four wavefronts: a matter of time alone, the bits are those of eight.  The sizes are those that both
// entry points know -- workgroups of eight (wgs) and keys of a sequence, about -- so that rows and paged cache choose alike.  Two or three
// workgroups of four on a compute unit hide their set-up and wind-down behind one another (about 8 us of a workgroup of eight, which has its
// compute unit to itself); two wavefronts of one workgroup that alternate between the pipes need less time per key.  us, eight / four, rows
// of k / v (the paged cache within 5 % of the same ratios), by sequences x lengths:
//                     16 q / 2 kv x 64   32 / 32 x 80    32 / 8 x 128    32 / 32 x 128
//   64 x 30..300        33 / 25           114 / 65         84 / 67         121 / 93
//   24 x 40..700        37 / 31            96 / 72         88 / 79         104 / 92
//   32 x 512            54 / 42           127 / 99        132 / 117        139 / 147
//   32 x 1024          144 / 114          346 / 329       365 / 373        417 / 419
//   16 x 2048          214 / 196          533 / 526       583 / 621        653 / 683
//   4 x 512           13.8 / 12.3        20.2 / 20.2     18.8 / 19.9      21.3 / 22.2
//   2 x 2048            39 / 44            65 / 76
//   2 x 4096            91 / 109          222 / 231       266 / 277        277 / 289
//   1 x 300           10.0 / 9.1         11.3 / 11.0     14.0 / 12.2      12.5 / 12.0
//   32 x 20..100 + 500 17.0 / 17.7         69 / 55         43 / 44          79 / 62
//   8 x 512 + 2048      53 / 59           131 / 148
// Over 170 such sizes of each of nine kinds of heads, from both places, these lines cost 0.8 % on average against the better form of each (0.5 %
// at head sizes above 96), all four 1.2 % (1.8), all eight 11 % (7).
bool four_wavefronts_pay(const PrefillParams &p, int hdp, int heads) {
  const int64_t wgs = (p.total_q / (256 / heads) + p.batch / 2) * (p.Hq / heads);
  const int64_t keys = p.max_k > p.max_q ? p.max_k : p.total_q / p.batch;
  // Three workgroups to a compute unit.  Long contexts whose workgroups of eight are one round over 256 compute units (with two or three
  // sequences up to two rounds: a sequence's heavy row blocks then meet the next one's on the same compute units) stay with eight.
  if (hdp <= 96) return !(p.batch > 1 && keys >= 1000 && wgs > 250 && wgs <= (p.batch <= 3 ? 560 : 320));
  // Two: where eight leave compute units without work, and where there are more of them and contexts are short.
  return keys <= (wgs <= 220 ? 1900 : 800);
}

template <typename T, int HDP, int MODE = W8_ROWS>
void launch_prefill_w8(const PrefillParams &p, hipStream_t stream) {
  // Heads per workgroup (prefill_heads_log2): a workgroup then covers 64 rows of each of four heads that share
  // their K / V tiles instead of 256 rows of one, and a sequence's last, partly filled row block idles fewer
  // wavefronts.  Same bits whatever the number.  Measured on MI355X in turns (32 q / 8 kv heads, d 128): 8 x 4096
  // tokens 1, 2, 4 and 8 heads within 0.6 % of each other; 32 sequences of 1..2048 tokens 463 / 441 / 435 / 433 us
  // from rows and 441 / 424 / 412 / 411 us from the paged cache; 64 sequences of 1..1024 tokens 392 / 367 / 361 us;
  // 128 x 256 tokens 232 / 218 / 221 us; GQA ratios 3 and 7 (one head, whatever the switch) unchanged.
  const int hl = prefill_heads_log2(p, 3);
  if constexpr (MODE == W8_PAGED) {
    launch_prefill_nw<T, HDP, MODE, 8>(p, hl, stream);
  } else {
    const int force = tuning().prefill_kernel, hl4 = hl < 2 ? hl : 2;
    if (force == 5 || (force != 1 && four_wavefronts_pay(p, HDP, 1 << hl4)))
      launch_prefill_nw<T, HDP, MODE, 4>(p, hl4, stream);
    else
      launch_prefill_nw<T, HDP, MODE, 8>(p, hl, stream);
  }
}

template <typename T, int HDP, int QT, bool PAGED = false, bool SINKS = false>
void launch_prefill(PrefillParams p, hipStream_t stream) {
  constexpr int BM = 4 * QT * 32;
  static bool attr_set = false;  // benign race: setting twice is harmless
  auto kernel = prefill_varlen_kernel<T, HDP, QT, PAGED, SINKS>;
  if (!attr_set) {
    HA_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)Tile<HDP>::LDS_BYTES));
    attr_set = true;
  }
  p.n_qblocks = (p.max_q + BM - 1) / BM;
  const int64_t listed = SINKS ? row_blocks_of(p.total_q, p.batch, BM, p.n_qblocks) : 0;
  const int64_t n_wg = (listed > 0 ? listed : (int64_t)p.n_qblocks * p.batch) * p.Hq;
  HA_CHECK(n_wg <= 0x7fffffff, "mha_varlen_fwd: too many workgroups");
  p.row_blocks = (int)listed;
  kernel<<<dim3((unsigned)n_wg), 256, Tile<HDP>::LDS_BYTES, stream>>>(p);
  check_launch("mha_varlen_fwd");
}

template <typename T, int HDP>
void pick_qt(const PrefillParams &p, int64_t total_q, hipStream_t stream) {
  // The eight-wavefront kernel (256-row workgroups) is at least as fast at every launch size measured -- 4
  // sequences of 128..512 tokens x 32 heads: 21.6 vs 23.3 us, 4 x 512: 25 vs 36 us, 2 x 2048: 85 vs 152 us; one
  // 128-token sequence: 17 us either way -- so the four-wavefront kernel is left with what the other does not
  // do: head sizes above 128, sliding windows, rows too far apart for 32-bit offsets.
  if constexpr (HDP <= 128) {
    const int force = tuning().prefill_kernel;  // 0: choose here; 1: eight wavefronts; 2 / 3: four wavefronts, 2 / 1 row tiles
    // the eight-wavefront kernel addresses a tile's 64 rows with unsigned 32-bit byte offsets
    // ... and a sequence's keys and values with unsigned 32-bit byte offsets from its first row
    const int64_t span = (int64_t)1 << 32;
    const bool fits = p.k_row >= 0 && p.v_row >= 0 && (p.total_k + 64) * p.k_row * (int64_t)sizeof(T) < span &&
                      (p.total_k + 64) * p.v_row * (int64_t)sizeof(T) < span;
    // it knows the causal mask and no mask; other windows go to the four-wavefront kernel
    const bool plain = p.win_left < 0 && p.win_right <= 0;
    if (plain && fits && (force == 0 || force == 1 || force == 5)) {
      launch_prefill_w8<T, HDP>(p, stream);
      return;
    }
    if (force == 2) {
      launch_prefill<T, HDP, 2>(p, stream);
      return;
    }
  }
  (void)total_q;
  launch_prefill<T, HDP, 1>(p, stream);
}

template <typename T>
void dispatch_hd(const PrefillParams &p, int64_t total_q, hipStream_t stream) {
  const int hdp = ((p.d + 31) / 32) * 32;
  switch (hdp) {
    case 32: pick_qt<T, 32>(p, total_q, stream); break;
    case 64: pick_qt<T, 64>(p, total_q, stream); break;
    case 96: pick_qt<T, 96>(p, total_q, stream); break;
    case 128: pick_qt<T, 128>(p, total_q, stream); break;
    case 160: pick_qt<T, 160>(p, total_q, stream); break;
    case 192: pick_qt<T, 192>(p, total_q, stream); break;
    case 224: pick_qt<T, 224>(p, total_q, stream); break;
    case 256: pick_qt<T, 256>(p, total_q, stream); break;
    default: fail("mha_varlen_fwd: head size %d not supported (must be <= 256)", p.d);
  }
}

template <typename T>
__global__ void zero_kernel(T *ptr, int64_t rows, int64_t heads, int64_t d, int64_t row_stride, int64_t head_stride) {
  const int64_t n = rows * heads * d;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / (heads * d), hh = (i / d) % heads, e = i % d;
    ptr[r * row_stride + hh * head_stride + e] = from_float<T>(0.f);
  }
}

void check_qkv(const hipattn_tensor *t, const char *name, int dtype, int d, bool or_f32 = false) {
  check_tensor(t, name, 3);
  HA_CHECK(t->dtype == dtype || (or_f32 && t->dtype == HIPATTN_F32), "mha_varlen_fwd: %s dtype differs from q", name);
  HA_CHECK(t->sizes[2] == d, "mha_varlen_fwd: %s head size %lld differs from q's %d", name, (long long)t->sizes[2], d);
  HA_CHECK(d <= 1 || t->strides[2] == 1, "mha_varlen_fwd: %s must have a contiguous last dimension", name);
  const int per16 = 16 / dtype_size(t->dtype);
  HA_CHECK(t->strides[0] % per16 == 0 && t->strides[1] % per16 == 0 && (reinterpret_cast<uintptr_t>(t->data) & 15) == 0,
           "mha_varlen_fwd: %s rows and heads must be 16-byte aligned", name);
  check_data(t, name);
}

void mha_varlen_fwd_impl(const hipattn_tensor *q, const hipattn_tensor *k, const hipattn_tensor *v,
                         const hipattn_tensor *cu_q, const hipattn_tensor *cu_k, const hipattn_tensor *seqused_k,
                         int max_q, int max_k, float p_dropout, float scale, bool zero_tensors, bool causal,
                         int win_left, int win_right, hipattn_tensor *out, hipattn_tensor *lse, void *stream_arg) {
  check_tensor(q, "q", 3);
  HA_CHECK(q->dtype == HIPATTN_F16 || q->dtype == HIPATTN_BF16,
           "mha_varlen_fwd: only fp16 and bf16 are supported, got %s", dtype_name(q->dtype));
  const int d = (int)q->sizes[2];
  const int Hq = (int)q->sizes[1];
  HA_CHECK(d % 8 == 0, "mha_varlen_fwd: head size must be a multiple of 8, got %d", d);
  HA_CHECK(d > 0 && d <= 256, "mha_varlen_fwd: head size must be in (0, 256], got %d", d);
  check_qkv(q, "q", q->dtype, d);
  check_qkv(k, "k", q->dtype, d);
  check_qkv(v, "v", q->dtype, d);
  check_qkv(out, "out", q->dtype, d, true);
  const int Hkv = (int)k->sizes[1];
  HA_CHECK(v->sizes[0] == k->sizes[0] && v->sizes[1] == Hkv, "mha_varlen_fwd: k and v shapes differ");
  HA_CHECK(Hkv > 0 && Hq % Hkv == 0, "mha_varlen_fwd: %d query heads not divisible by %d kv heads", Hq, Hkv);
  HA_CHECK(out->sizes[0] == q->sizes[0] && out->sizes[1] == Hq, "mha_varlen_fwd: out shape differs from q");
  check_tensor(cu_q, "cu_seqlens_q", 1);
  check_tensor(cu_k, "cu_seqlens_k", 1);
  HA_CHECK(cu_q->dtype == HIPATTN_I32 && cu_k->dtype == HIPATTN_I32, "mha_varlen_fwd: cu_seqlens must be int32");
  check_contiguous(cu_q, "cu_seqlens_q");
  check_contiguous(cu_k, "cu_seqlens_k");
  HA_CHECK(cu_q->sizes[0] >= 1 && cu_k->sizes[0] == cu_q->sizes[0],
           "mha_varlen_fwd: cu_seqlens_q and cu_seqlens_k must both hold batch+1 entries");
  const int batch = (int)cu_q->sizes[0] - 1;
  if (seqused_k) {
    check_tensor(seqused_k, "seqused_k", 1);
    HA_CHECK(seqused_k->dtype == HIPATTN_I32 && seqused_k->sizes[0] == batch, "mha_varlen_fwd: seqused_k must be int32 [batch]");
    check_contiguous(seqused_k, "seqused_k");
    check_data(seqused_k, "seqused_k");
  }
  HA_CHECK(p_dropout == 0.f, "mha_varlen_fwd: dropout is not supported (inference only)");
  HA_CHECK(scale > 0.f, "mha_varlen_fwd: softmax_scale must be positive");
  // flash_api.cpp:466, 113-120: causal is the window (-inf, 0]; one given bound leaves the other open.
  // rLLM itself only ever passes (-1, -1) (lib.rs:96-97).
  if (causal) win_right = 0;
  if (win_left < 0) win_left = -1;
  if (win_right < 0) win_right = -1;
  causal = win_left < 0 && win_right == 0;
  HA_CHECK(max_q >= 0 && max_k >= 0, "mha_varlen_fwd: negative max_seqlen");
  if (lse) {
    check_tensor(lse, "softmax_lse", 3);
    HA_CHECK(lse->dtype == HIPATTN_F32 && lse->sizes[0] == batch && lse->sizes[1] == Hq && lse->sizes[2] >= max_q,
             "mha_varlen_fwd: softmax_lse must be f32 [batch, Hq, >= max_seqlen_q]");
    check_contiguous(lse, "softmax_lse");
    check_data(lse, "softmax_lse");
  }
  hipStream_t stream = resolve_stream(stream_arg);
  const int64_t total_q = q->sizes[0];
  if (zero_tensors && total_q > 0 && Hq > 0) {
    if (out->dtype == HIPATTN_F32)
      zero_kernel<float><<<1024, 256, 0, stream>>>(static_cast<float *>(out->data), total_q, Hq, d, out->strides[0], out->strides[1]);
    else if (q->dtype == HIPATTN_F16)
      zero_kernel<half_t><<<1024, 256, 0, stream>>>(static_cast<half_t *>(out->data), total_q, Hq, d, out->strides[0], out->strides[1]);
    else
      zero_kernel<bf16_t><<<1024, 256, 0, stream>>>(static_cast<bf16_t *>(out->data), total_q, Hq, d, out->strides[0], out->strides[1]);
    if (lse && numel(lse) > 0)
      zero_kernel<float><<<256, 256, 0, stream>>>(static_cast<float *>(lse->data), 1, 1, numel(lse), 0, 0);
    check_launch("mha_varlen_fwd zero");
  }
  if (batch == 0 || total_q == 0 || Hq == 0 || max_q == 0) return;
  check_data(cu_q, "cu_seqlens_q");
  check_data(cu_k, "cu_seqlens_k");

  PrefillParams p;
  memset(&p, 0, sizeof p);
  p.q = q->data;
  p.k = k->data;
  p.v = v->data;
  p.out = out->data;
  p.lse = lse ? static_cast<float *>(lse->data) : nullptr;
  p.q_row = q->strides[0];
  p.q_head = q->strides[1];
  p.k_row = k->strides[0];
  p.k_head = k->strides[1];
  p.v_row = v->strides[0];
  p.v_head = v->strides[1];
  p.o_row = out->strides[0];
  p.o_head = out->strides[1];
  p.cu_q = static_cast<const int32_t *>(cu_q->data);
  p.cu_k = static_cast<const int32_t *>(cu_k->data);
  p.seqused_k = seqused_k ? static_cast<const int32_t *>(seqused_k->data) : nullptr;
  p.total_k = k->sizes[0];
  p.batch = batch;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.d = d;
  p.max_q = max_q;
  p.max_k = max_k;
  p.total_q = total_q;
  p.lse_pitch = lse ? (int)lse->sizes[2] : 0;
  p.scale_log2 = scale * kLog2e;
  p.causal = causal ? 1 : 0;
  p.win_left = win_left;
  p.win_right = win_right;
  p.out_f32 = out->dtype == HIPATTN_F32 ? 1 : 0;
  p.rescale_thr = (float)tuning().prefill_rescale_log2;
  const int force = tuning().prefill_kernel;
  if ((force == 4 || (force == 0 && prefer_prefill_r3(p))) && launch_prefill_r3(p, q->dtype, stream)) return;
  if (q->dtype == HIPATTN_F16) dispatch_hd<half_t>(p, total_q, stream);
  else dispatch_hd<bf16_t>(p, total_q, stream);
}

template <typename T>
void dispatch_staged_window(const PrefillParams &p, hipStream_t stream) {
  switch ((p.d + 31) / 32 * 32) {
    case 32: launch_prefill<T, 32, 1, true, true>(p, stream); break;
    case 64: launch_prefill<T, 64, 1, true, true>(p, stream); break;
    case 96: launch_prefill<T, 96, 1, true, true>(p, stream); break;
    case 128: launch_prefill<T, 128, 1, true, true>(p, stream); break;
    case 160: launch_prefill<T, 160, 1, true, true>(p, stream); break;
    case 192: launch_prefill<T, 192, 1, true, true>(p, stream); break;
    case 224: launch_prefill<T, 224, 1, true, true>(p, stream); break;
    case 256: launch_prefill<T, 256, 1, true, true>(p, stream); break;
    default: fail("mha_varlen_fwd_paged_window: head size %d not supported (at most 256)", p.d);
  }
}

// Varlen prefill whose keys and values are read from the paged cache through block tables: what
// rLLM composes from gather_cached_kv -> repeat_kv -> flash_attn_varlen (llm/mod.rs:181-238) without
// the two copies.  Eight-wavefront kernel for head sizes up to 128, four-wavefront kernel above.
template <typename T>
void dispatch_paged(const PrefillParams &p, hipStream_t stream) {
  const int hdp = ((p.d + 31) / 32) * 32;
  // The block images go into LDS as they are (16-byte aligned images); head sizes that fill their MFMA tiles
  // take the plain form, those from 40 up that do not take the form that clears what an image leaves
  // untouched, the rest is staged through registers, which pads it.  The tuning switch paged_prefill_dma = 0
  // forces the staged form.
  const bool dma = paged_prefill_copies_images(p);
  if (p.block_log2 != 4) {
    // 8- and 32-token blocks (rLLM runs 16): the four-wavefront kernel, whose staged tiles take any block size
    switch (hdp) {
      case 32: launch_prefill<T, 32, 1, true>(p, stream); break;
      case 64: launch_prefill<T, 64, 1, true>(p, stream); break;
      case 96: launch_prefill<T, 96, 1, true>(p, stream); break;
      case 128: launch_prefill<T, 128, 1, true>(p, stream); break;
      case 160: launch_prefill<T, 160, 1, true>(p, stream); break;
      case 192: launch_prefill<T, 192, 1, true>(p, stream); break;
      case 224: launch_prefill<T, 224, 1, true>(p, stream); break;
      case 256: launch_prefill<T, 256, 1, true>(p, stream); break;
      default: fail("mha_varlen_fwd_paged: head size %d not supported (at most 256)", p.d);
    }
    return;
  }
#define HA_W8P(H)                                                                  \
  if (dma && p.d == H) launch_prefill_w8<T, H, W8_PAGED_DMA>(p, stream);           \
  else if (dma && H >= 64) launch_prefill_w8<T, (H >= 64 ? H : 64), W8_PAGED_DMA_PART>(p, stream); \
  else launch_prefill_w8<T, H, W8_PAGED>(p, stream)
  switch (hdp) {
    case 32: HA_W8P(32); break;
    case 64: HA_W8P(64); break;
    case 96: HA_W8P(96); break;
    case 128: HA_W8P(128); break;
    // head sizes above 128: the four-wavefront kernel, tiles staged through registers
    case 160: launch_prefill<T, 160, 1, true>(p, stream); break;
    case 192: launch_prefill<T, 192, 1, true>(p, stream); break;
    case 224: launch_prefill<T, 224, 1, true>(p, stream); break;
    case 256: launch_prefill<T, 256, 1, true>(p, stream); break;
    default: fail("mha_varlen_fwd_paged: head size %d not supported (at most 256)", p.d);
  }
#undef HA_W8P
}

}  // namespace

bool paged_prefill_params(const PagedPrefillCall &c, hipattn_tensor *out, hipattn_tensor *lse, PrefillParams &p) {
  const char *op = c.op;
  const hipattn_tensor *q = c.q, *key_cache = c.key_cache, *value_cache = c.value_cache, *block_tables = c.block_tables, *cu_q = c.cu_q,
                       *context_lens = c.context_lens;
  const int max_q = c.max_q, max_k = c.max_k;
  const float scale = c.scale;
  const bool causal = c.causal;
  check_tensor(q, "q", 3);
  HA_CHECK(q->dtype == HIPATTN_F16 || q->dtype == HIPATTN_BF16, "%s: only fp16 and bf16 are supported, got %s", op,
           dtype_name(q->dtype));
  const int d = (int)q->sizes[2];
  const int Hq = (int)q->sizes[1];
  HA_CHECK(d % 8 == 0 && d > 0 && d <= 256, "%s: head size must be a multiple of 8 in (0, 256], got %d", op, d);
  check_qkv(q, "q", q->dtype, d);
  check_qkv(out, "out", q->dtype, d, true);
  HA_CHECK(out->sizes[0] == q->sizes[0] && out->sizes[1] == Hq, "%s: out shape differs from q", op);
  check_tensor(key_cache, "key_cache", 5);
  check_tensor(value_cache, "value_cache", 4);
  HA_CHECK(key_cache->dtype == q->dtype && value_cache->dtype == q->dtype, "%s: caches must have q's dtype", op);
  const int Hkv = (int)key_cache->sizes[1];
  HA_CHECK(Hkv > 0 && Hq % Hkv == 0, "%s: %d query heads not divisible by %d kv heads", op, Hq, Hkv);
  const int64_t bs = key_cache->sizes[3];  // the caches say what their block size is
  HA_CHECK(bs == 8 || bs == 16 || bs == 32, "%s: unsupported block size %lld (supported: 8, 16, 32)", op, (long long)bs);
  HA_CHECK(key_cache->sizes[2] * key_cache->sizes[4] == d && key_cache->sizes[4] == 8,
           "%s: key_cache shape does not match [nb, %d, %d/8, block size, 8]", op, Hkv, d);
  HA_CHECK(value_cache->sizes[0] == key_cache->sizes[0] && value_cache->sizes[1] == Hkv &&
               value_cache->sizes[2] == d && value_cache->sizes[3] == bs,
           "%s: value_cache shape does not match [nb, %d, %d, %lld]", op, Hkv, d, (long long)bs);
  HA_CHECK(key_cache->strides[4] == 1 && key_cache->strides[3] == 8 && key_cache->strides[2] == 8 * bs &&
               value_cache->strides[3] == 1 && value_cache->strides[2] == bs,
           "%s: cache inner dims must be contiguous", op);
  HA_CHECK(key_cache->strides[0] % 8 == 0 && key_cache->strides[1] % 8 == 0 && value_cache->strides[0] % 4 == 0 &&
               value_cache->strides[1] % 4 == 0 && (reinterpret_cast<uintptr_t>(key_cache->data) & 15) == 0 &&
               (reinterpret_cast<uintptr_t>(value_cache->data) & 15) == 0,
           "%s: caches must be 16-byte aligned", op);
  HA_CHECK(key_cache->sizes[0] > 0, "%s: the cache has no blocks", op);
  check_tensor(cu_q, "cu_seqlens_q", 1);
  check_tensor(context_lens, "context_lens", 1);
  check_tensor(block_tables, "block_tables", 2);
  HA_CHECK(cu_q->dtype == HIPATTN_I32 && context_lens->dtype == HIPATTN_I32 && block_tables->dtype == HIPATTN_I32,
           "%s: cu_seqlens_q, context_lens and block_tables must be int32", op);
  check_contiguous(cu_q, "cu_seqlens_q");
  check_contiguous(context_lens, "context_lens");
  HA_CHECK(cu_q->sizes[0] >= 1, "%s: cu_seqlens_q must hold batch+1 entries", op);
  const int batch = (int)cu_q->sizes[0] - 1;
  HA_CHECK(context_lens->sizes[0] == batch && block_tables->sizes[0] == batch,
           "%s: context_lens and block_tables need %d rows", op, batch);
  HA_CHECK(block_tables->sizes[1] <= 1 || block_tables->strides[1] == 1, "%s: block_tables rows must be contiguous", op);
  HA_CHECK(scale > 0.f, "%s: softmax_scale must be positive", op);
  HA_CHECK(max_q >= 0 && max_k >= 0, "%s: negative max_seqlen", op);
  HA_CHECK(((int64_t)max_k + bs - 1) / bs <= block_tables->sizes[1], "%s: max_seqlen_k %d needs more than the %lld block-table columns",
           op, max_k, (long long)block_tables->sizes[1]);
  if (lse) {
    check_tensor(lse, "softmax_lse", 3);
    HA_CHECK(lse->dtype == HIPATTN_F32 && lse->sizes[0] == batch && lse->sizes[1] == Hq && lse->sizes[2] >= max_q,
             "%s: softmax_lse must be f32 [batch, Hq, >= max_seqlen_q]", op);
    check_contiguous(lse, "softmax_lse");
    check_data(lse, "softmax_lse");
  }
  const int64_t total_q = q->sizes[0];
  if (batch == 0 || total_q == 0 || Hq == 0 || max_q == 0) return false;
  check_data(cu_q, "cu_seqlens_q");
  check_data(context_lens, "context_lens");
  check_data(block_tables, "block_tables");
  check_data(key_cache, "key_cache");
  check_data(value_cache, "value_cache");
  memset(&p, 0, sizeof p);
  p.q = q->data;
  p.k = key_cache->data;
  p.v = value_cache->data;
  p.out = out->data;
  p.lse = lse ? static_cast<float *>(lse->data) : nullptr;
  p.q_row = q->strides[0];
  p.q_head = q->strides[1];
  p.o_row = out->strides[0];
  p.o_head = out->strides[1];
  p.cu_q = static_cast<const int32_t *>(cu_q->data);
  p.batch = batch;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.d = d;
  p.max_q = max_q;
  p.max_k = max_k;
  p.total_q = total_q;
  p.lse_pitch = lse ? (int)lse->sizes[2] : 0;
  p.scale_log2 = scale * kLog2e;
  p.causal = causal ? 1 : 0;
  p.win_left = -1;
  p.win_right = causal ? 0 : -1;
  p.out_f32 = out->dtype == HIPATTN_F32 ? 1 : 0;
  p.rescale_thr = (float)tuning().prefill_rescale_log2;
  p.block_tables = static_cast<const int32_t *>(block_tables->data);
  p.context_lens = static_cast<const int32_t *>(context_lens->data);
  p.table_stride = block_tables->strides[0];
  p.table_cols = (int)block_tables->sizes[1];
  p.num_blocks = key_cache->sizes[0];
  p.kc_block = key_cache->strides[0];
  p.kc_head = key_cache->strides[1];
  p.vc_block = value_cache->strides[0];
  p.vc_head = value_cache->strides[1];
  p.block_log2 = bs == 8 ? 3 : (bs == 16 ? 4 : 5);
  return true;
}

void launch_staged_window(const PrefillParams &p, int dtype, hipStream_t stream) {
  if (dtype == HIPATTN_F16) dispatch_staged_window<half_t>(p, stream);
  else dispatch_staged_window<bf16_t>(p, stream);
}

bool paged_prefill_copies_images(const PrefillParams &p) {
  return p.block_log2 == 4 && p.vc_block % 8 == 0 && p.vc_head % 8 == 0 && tuning().paged_prefill_dma != 0;
}

namespace {

void mha_varlen_fwd_paged_impl(const hipattn_tensor *q, const hipattn_tensor *key_cache,
                               const hipattn_tensor *value_cache, const hipattn_tensor *block_tables,
                               const hipattn_tensor *cu_q, const hipattn_tensor *context_lens, int max_q, int max_k,
                               float scale, bool causal, hipattn_tensor *out, hipattn_tensor *lse, void *stream_arg) {
  PrefillParams p;
  if (!paged_prefill_params(PagedPrefillCall{q, key_cache, value_cache, block_tables, cu_q, context_lens, max_q, max_k, scale, causal}, out, lse, p))
    return;
  hipStream_t stream = resolve_stream(stream_arg);
  if (q->dtype == HIPATTN_F16) dispatch_paged<half_t>(p, stream);
  else dispatch_paged<bf16_t>(p, stream);
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" char *hipattn_mha_varlen_fwd_paged(const hipattn_tensor *q, const hipattn_tensor *key_cache,
                                              const hipattn_tensor *value_cache, const hipattn_tensor *block_tables,
                                              const hipattn_tensor *cu_seqlens_q, const hipattn_tensor *context_lens,
                                              int max_seqlen_q, int max_seqlen_k, float softmax_scale, bool is_causal,
                                              hipattn_tensor *out, hipattn_tensor *softmax_lse, void *stream) {
  HA_PROTECT(mha_varlen_fwd_paged_impl(q, key_cache, value_cache, block_tables, cu_seqlens_q, context_lens, max_seqlen_q,
                                       max_seqlen_k, softmax_scale, is_causal, out, softmax_lse, stream));
}

extern "C" char *hipattn_mha_varlen_fwd(const hipattn_tensor *q, const hipattn_tensor *k, const hipattn_tensor *v,
                                        const hipattn_tensor *cu_seqlens_q, const hipattn_tensor *cu_seqlens_k,
                                        const hipattn_tensor *seqused_k, int max_seqlen_q, int max_seqlen_k,
                                        float p_dropout, float softmax_scale, bool zero_tensors, bool is_causal,
                                        int window_size_left, int window_size_right, hipattn_tensor *out,
                                        hipattn_tensor *softmax_lse, void *stream) {
  HA_PROTECT(mha_varlen_fwd_impl(q, k, v, cu_seqlens_q, cu_seqlens_k, seqused_k, max_seqlen_q, max_seqlen_k, p_dropout,
                                 softmax_scale, zero_tensors, is_causal, window_size_left, window_size_right, out,
                                 softmax_lse, stream));
}
