// Attention of trees of drafted tokens over a paged cache: a sequence's n rows see the ctx - n keys in front of the tree and, of the tree's own
// keys (the last n of the context), those that their mask names.
//
//   out[i] = sum_t p[t] v[t] / sum_t p[t],  p[t] = 2^(log2(e) scale q[i].k[t] - m) where t < ctx - n or bit t - (ctx - n) of mask[i] is set, else 0
//
// The rows of a tree with the query heads of a kv group are columns of the decode kernel's products (paged_decode.h), 16 to a tile; a wavefront
// holds the cache bytes of 32 tokens in registers and takes them through up to NT tiles of columns, so that a tree of 16 NT / G rows reads its
// context once.  The 32-token pairs of a part of the context are dealt out to the wavefronts of a workgroup, the parts to workgroups; the
// wavefronts meet in LDS, the parts in a second launch.
//
// A tree is memory-bound in theory up to some 300 columns (its products per byte of the cache); the softmax and the masks make it so up to
// about 64.  Only pairs that reach into the tree look at the mask.
//
// Numerics are those of paged decode: scores and sums in fp32, probabilities rounded to the cache's type as operands of the second product,
// the normaliser not.
#include <algorithm>

#include "paged_decode.h"
#include "prefill_common.h"

namespace hipattn {

namespace {

constexpr int kTreeMostParts = 64;
constexpr size_t kTreeScratchBytes = (size_t)64 << 20;

struct TreeParams {
  DecodeParams cache;  // the caches, tables, context lengths and scale
  const void *q;
  void *out;
  int64_t q_row, q_head, o_row, o_head, total_q;
  const int32_t *cu_q;
  const unsigned long long *mask;
  int64_t mask_row;
  int words;  // of a row of the mask
  int batch, Hq, Hkv, G;
  int col_groups;  // workgroups that share the columns of a (sequence, kv head)
  int columns;     // that they have; rows beyond max_seqlen_q may have none
  int part_pairs, num_parts, max_pairs;
  float *part_acc, *part_ml;  // of part i of row r and head h, at (i * total_q + r) * Hq + h: d sums; maximum and sum
};

// Pairs of 16-token runs of a context; what max_seqlen_k does not allow for is left out, as there is no part for it.
__device__ __forceinline__ int tree_pairs(const TreeParams &p, int ctx) {
  return ctx > 0 ? min((int)(((int64_t)ctx + 31) / 32), p.max_pairs) : 0;
}

// Bits j .. j + 3 of a row's mask; bits in front of the tree are set, those behind it are not.
__device__ __forceinline__ unsigned tree_bits(const unsigned long long *row, int words, int n, int j) {
  unsigned bits = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int b = j + i;
    bool seen = b < 0;
    if (b >= 0 && b < n && (b >> 6) < words) seen = (row[b >> 6] >> (b & 63)) & 1;
    bits |= (unsigned)seen << i;
  }
  return bits;
}

template <typename T>
__device__ __forceinline__ bool not_finite(uint16_t e) {
  constexpr uint16_t top = sizeof(T) == 2 && __is_same(T, half_t) ? 0x7c00 : 0x7f80;
  return (e & top) == top;
}

template <typename T, int HD, int BS, int NT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void tree_attention_kernel(TreeParams p) {
  typedef typename Vec8<T>::type vec8;
  constexpr int NCH = HD / 8, NSTEP = (HD + 31) / 32, NDT = HD / 16;
  constexpr int IDS = 32 / BS, HELD = 64 / IDS;  // blocks of a pair; pairs whose blocks' numbers a wavefront's lanes hold
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), kg = lane >> 4, col = lane & 15;
  // Workgroup -> (part, sequence, column group, kv head), the kv head fastest: the column groups that read the same keys share an XCD's L2.
  int id = blockIdx.x;
  const int kvh = id % p.Hkv;
  id /= p.Hkv;
  const int cg = id % p.col_groups;
  id /= p.col_groups;
  const int seq = id % p.batch, part = id / p.batch;
  const int q_begin = p.cu_q[seq], n = min(p.cu_q[seq + 1], (int)p.total_q) - q_begin;
  const int c0 = cg * 16 * NT;
  if (q_begin < 0 || n <= 0 || c0 >= (int64_t)n * p.G) return;
  const int ctx = p.cache.context_lens[seq], front = ctx - n;
  const int pairs = tree_pairs(p, ctx), first = part * p.part_pairs;
  if (first >= pairs && part > 0) return;
  const int my_pairs = min(first + p.part_pairs, pairs) - first;
  const int32_t *table = p.cache.block_tables + seq * p.cache.max_blocks;
  const int tiles = min(NT, (int)(((int64_t)n * p.G - c0 + 15) / 16));  // with a column

  int row[NT], head[NT];
  bool ok[NT];
  vec8 qreg[NT][NSTEP];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int c = c0 + t * 16 + col;
    row[t] = c / p.G;
    head[t] = kvh * p.G + c - row[t] * p.G;
    ok[t] = row[t] < n;
    const T *qp = static_cast<const T *>(p.q) + (int64_t)(q_begin + row[t]) * p.q_row + head[t] * p.q_head;
#pragma unroll
    for (int s = 0; s < NSTEP; s++) {
      const int ch = 4 * s + kg;
      u32x4_t raw = {0u, 0u, 0u, 0u};
      if (ok[t] && ch < NCH) raw = *reinterpret_cast<const u32x4_t *>(qp + ch * 8);
      qreg[t][s] = bit_cast<vec8>(raw);
    }
  }
  const T *kbase = static_cast<const T *>(p.cache.kc) + (int64_t)kvh * p.cache.k_head_stride;
  const T *vbase = static_cast<const T *>(p.cache.vc) + (int64_t)kvh * p.cache.v_head_stride;
  float m_run[NT], l_run[NT];
  f32x4_t acc[NT][NDT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    m_run[t] = -INFINITY;
    l_run[t] = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; dt++) acc[t][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  for (int g0 = wave; g0 < my_pairs; g0 += WAVES * HELD) {
    // The blocks of this wavefront's next HELD pairs, IDS lanes to a pair.
    int ids = 0;
    {
      const int64_t pair = (int64_t)first + g0 + WAVES * (lane / IDS), column = pair * IDS + lane % IDS;
      if (column < p.cache.table_cols) ids = table[column];
    }
    for (int j = 0; j < HELD && g0 + j * WAVES < my_pairs; j++) {
      PairRegs<HD> r;
      {
        const int at = j * IDS;
        const int64_t i0 = __builtin_amdgcn_readlane(ids, at), i1 = IDS > 1 ? __builtin_amdgcn_readlane(ids, at + IDS / 2 - (IDS == 4)) : 0;
        const int64_t i2 = IDS > 2 ? __builtin_amdgcn_readlane(ids, at + 2) : 0, i3 = IDS > 2 ? __builtin_amdgcn_readlane(ids, at + 3) : 0;
        pair_load_bs<T, HD, BS, false>(p.cache, kbase, vbase, i0, i1, i2, i3, r);
      }
      const int tok = (first + g0 + j * WAVES) * 32, tok_a = tok + kg * 4, tok_b = tok_a + 16;  // this lane's tokens, four of each run
      const bool tail = tok + 32 > front;  // the pair reaches into the tree
      unsigned odd = 0;  // the tail's values of this lane's eight tokens that are not finite
      if (tail) {
        // What lies behind the context is anything, and a probability of zero does not undo it.
#pragma unroll
        for (int dt = 0; dt < NDT; dt++) {
          uint16_t *ea = reinterpret_cast<uint16_t *>(&r.vra[dt]), *eb = reinterpret_cast<uint16_t *>(&r.vrb[dt]);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            if (tok_a + i >= ctx) ea[i] = 0;
            if (tok_b + i >= ctx) eb[i] = 0;
            if (not_finite<T>(ea[i])) {
              odd |= 1u << i;
              ea[i] = 0;
            }
            if (not_finite<T>(eb[i])) {
              odd |= 16u << i;
              eb[i] = 0;
            }
          }
        }
      }
      const bool any_odd = tail && __any(odd != 0);
#pragma unroll
      for (int t = 0; t < NT; t++) {
        if (t >= tiles) continue;
        f32x4_t sa = {0.f, 0.f, 0.f, 0.f}, sb = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NSTEP; s++) {
          sa = Mfma16<T>::run(bit_cast<vec8>(r.kra[s]), qreg[t][s], sa);
          sb = Mfma16<T>::run(bit_cast<vec8>(r.krb[s]), qreg[t][s], sb);
        }
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          x[i] = sa[i] * p.cache.scale_log2;
          x[4 + i] = sb[i] * p.cache.scale_log2;
        }
        unsigned seen = 0xff;
        if (tail) {
          const unsigned long long *words = p.mask + (int64_t)(q_begin + (ok[t] ? row[t] : 0)) * p.mask_row;
          seen = tree_bits(words, p.words, n, tok_a - front) | tree_bits(words, p.words, n, tok_b - front) << 4;
#pragma unroll
          for (int i = 0; i < 8; i++)
            if (!(seen >> i & 1)) x[i] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m_new = fmaxf(m_run[t], mx), m_safe = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = fast_exp2(m_run[t] - m_safe);
        float psum = 0.f;
        vec8 pv;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float e = fast_exp2(x[i] - m_safe);
          psum += e;
          pv[i] = from_float<T>(e);
        }
        l_run[t] = l_run[t] * alpha + psum;
        m_run[t] = m_new;
        if (__any(alpha != 1.0f)) {
#pragma unroll
          for (int dt = 0; dt < NDT; dt++) acc[t][dt] *= alpha;
        }
#pragma unroll
        for (int dt = 0; dt < NDT; dt++) {
          const u32x4_t a = {r.vra[dt][0], r.vra[dt][1], r.vrb[dt][0], r.vrb[dt][1]};
          acc[t][dt] = Mfma16<T>::run(bit_cast<vec8>(a), pv, acc[t][dt]);
        }
        if (any_odd) {
          // Values of the tree that are not finite count for the rows that see them, and for no others: token after token.
          for (int u = 0; u < 32; u++) {
            const int from = (u & 15) >> 2, i = (u >> 4) * 4 + (u & 3);  // the lanes that hold it, and which of their eight it is
            const unsigned long long holders = __ballot(odd >> i & 1) >> (16 * from) & 0xffff;
            if (holders == 0) continue;
            float e = 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++)
              if (k == i) e = to_float<T>(pv[k]);
            e = __shfl(e, from * 16 + col, 64);
            const bool sees = __shfl((int)(seen >> i & 1), from * 16 + col, 64) != 0;
            const int token = tok + u;
            int64_t block = token / BS < p.cache.table_cols ? table[token / BS] : 0;
            block = block < 0 ? 0 : (block < p.cache.num_blocks ? block : p.cache.num_blocks - 1);
            const T *v = vbase + block * p.cache.v_block_stride + token % BS;
#pragma unroll
            for (int dt = 0; dt < NDT; dt++)
#pragma unroll
              for (int k = 0; k < 4; k++) {
                const T value = v[(dt * 16 + kg * 4 + k) * BS];
                if (sees && not_finite<T>(bit_cast<uint16_t>(value))) acc[t][dt][k] += e * to_float<T>(value);
              }
          }
        }
      }
    }
  }

  // The wavefronts' states, the upper half of them into the lower until one is left.
  constexpr int HALF = WAVES / 2;
  __shared__ f32x4_t s_acc[HALF][NT * NDT][64];
  __shared__ float s_ml[HALF][2][NT][64];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    l_run[t] += __shfl_xor(l_run[t], 16, 64);
    l_run[t] += __shfl_xor(l_run[t], 32, 64);
  }
#pragma unroll
  for (int half = HALF; half > 0; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int t = 0; t < NT; t++) {
        s_ml[wave - half][0][t][lane] = m_run[t];
        s_ml[wave - half][1][t][lane] = l_run[t];
#pragma unroll
        for (int dt = 0; dt < NDT; dt++) s_acc[wave - half][t * NDT + dt][lane] = acc[t][dt];
      }
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const float m = s_ml[wave][0][t][lane], l = s_ml[wave][1][t][lane], top = fmaxf(m_run[t], m), base = top == -INFINITY ? 0.f : top;
        const float mine = fast_exp2(m_run[t] - base), other = fast_exp2(m - base);
        m_run[t] = top;
        l_run[t] = l_run[t] * mine + l * other;
#pragma unroll
        for (int dt = 0; dt < NDT; dt++) acc[t][dt] = acc[t][dt] * mine + s_acc[wave][t * NDT + dt][lane] * other;
      }
    }
    __syncthreads();
  }
  if (wave > 0) return;
  const bool whole = pairs <= p.part_pairs;  // nothing to merge
#pragma unroll
  for (int t = 0; t < NT; t++) {
    if (!ok[t]) continue;
    if (whole) {
      const float inv = l_run[t] == 0.f ? 0.f : 1.0f / l_run[t];  // (a row that sees nothing is zero, one with a NaN is NaN)
      T *op = static_cast<T *>(p.out) + (int64_t)(q_begin + row[t]) * p.o_row + head[t] * p.o_head + kg * 4;
#pragma unroll
      for (int dt = 0; dt < NDT; dt++) {
        T o[4];
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = from_float<T>(acc[t][dt][i] * inv);
        *reinterpret_cast<u32x2_t *>(op + dt * 16) = *reinterpret_cast<u32x2_t *>(o);
      }
    } else {
      const int64_t at = ((int64_t)part * p.total_q + q_begin + row[t]) * p.Hq + head[t];
#pragma unroll
      for (int dt = 0; dt < NDT; dt++) *reinterpret_cast<f32x4_t *>(p.part_acc + at * HD + dt * 16 + kg * 4) = acc[t][dt];
      if (kg == 0) *reinterpret_cast<float2 *>(p.part_ml + 2 * at) = make_float2(m_run[t], l_run[t]);
    }
  }
}

// The merge: a thread for four elements of a (row, head).
template <typename T, int HD>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeParams p) {
  constexpr int QUADS = HD / 4;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x, rh = idx / QUADS;
  const int r = (int)(rh / p.Hq), h = (int)(rh % p.Hq), e = (int)(idx % QUADS) * 4;
  if (r >= p.total_q) return;
  // the sequence that holds row r: the first that ends behind it
  int lo = 0, hi = p.batch;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_q[mid + 1] > r) hi = mid;
    else lo = mid + 1;
  }
  if (lo == p.batch || r < p.cu_q[lo]) return;
  const int pairs = tree_pairs(p, p.cache.context_lens[lo]);
  if (pairs <= p.part_pairs || (int64_t)(r - p.cu_q[lo]) * p.G + h % p.G >= p.columns) return;  // written, or left out
  const int parts = (pairs + p.part_pairs - 1) / p.part_pairs;
  const int64_t step = p.total_q * p.Hq;
  float top = -INFINITY;
  for (int k = 0; k < parts; k++) top = fmaxf(top, p.part_ml[2 * (k * step + rh)]);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = 0; k < parts; k++) {
    const int64_t at = k * step + rh;
    const float2 ml = *reinterpret_cast<const float2 *>(p.part_ml + 2 * at);
    const f32x4_t a = *reinterpret_cast<const f32x4_t *>(p.part_acc + at * HD + e);
    const float w = fast_exp2(ml.x - base);
    sum += w * ml.y;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] += w * a[j];
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  T out[4];
#pragma unroll
  for (int j = 0; j < 4; j++) out[j] = from_float<T>(o[j] * inv);
  *reinterpret_cast<u32x2_t *>(static_cast<T *>(p.out) + (int64_t)r * p.o_row + (int64_t)h * p.o_head + e) = *reinterpret_cast<u32x2_t *>(out);
}

struct TreePlan {
  int tiles;  // NT
  int waves;
  int col_groups, part_pairs, num_parts, max_pairs;
};

// Columns to a wavefront: as many as the largest tree has, up to four tiles.  Parts: two workgroups to a compute unit.
TreePlan plan_tree(const PrefillParams &p, int most_parts) {
  TreePlan pl;
  const int64_t cols = (int64_t)std::min<int64_t>(p.max_q, p.total_q) * p.G;
  pl.tiles = p.d > 128 ? (cols <= 16 ? 1 : 2) : (cols <= 16 ? 1 : (cols <= 32 ? 2 : 4));
  pl.waves = pl.tiles == 4 || (p.d > 128 && pl.tiles == 2) ? 4 : 8;
  pl.col_groups = (int)((cols + 16 * pl.tiles - 1) / (16 * pl.tiles));
  const int64_t pairs = std::max<int64_t>(((int64_t)p.max_k + 31) / 32, 1);
  // (column groups that trees of these rows together can have)
  const int64_t groups = std::min<int64_t>((int64_t)pl.col_groups * p.batch, (p.total_q * p.G) / (16 * pl.tiles) + p.batch) * p.Hkv;
  int64_t parts = std::max<int64_t>((int64_t)2 * compute_units() * (8 / pl.waves) / std::max<int64_t>(groups, 1), 1);
  parts = std::min<int64_t>(std::min<int64_t>(parts, most_parts), (pairs + pl.waves - 1) / pl.waves);
  pl.max_pairs = (int)pairs;
  pl.part_pairs = (int)((pairs + parts - 1) / parts);
  pl.num_parts = (int)((pairs + pl.part_pairs - 1) / pl.part_pairs);
  return pl;
}

template <typename T, int HD, int BS>
void launch_tree_bs(const TreeParams &p, const TreePlan &pl, dim3 grid, hipStream_t stream) {
  if (pl.tiles == 1) tree_attention_kernel<T, HD, BS, 1, 8><<<grid, 512, 0, stream>>>(p);
  else if constexpr (HD > 128) tree_attention_kernel<T, HD, BS, 2, 4><<<grid, 256, 0, stream>>>(p);
  else if (pl.tiles == 2) tree_attention_kernel<T, HD, BS, 2, 8><<<grid, 512, 0, stream>>>(p);
  else tree_attention_kernel<T, HD, BS, 4, 4><<<grid, 256, 0, stream>>>(p);
}

template <typename T, int HD>
void launch_tree(const TreeParams &p, const TreePlan &pl, int block_size, hipStream_t stream) {
  const int64_t wgs = (int64_t)p.Hkv * p.col_groups * p.batch * p.num_parts, merges = (p.total_q * p.Hq * (HD / 4) + 255) / 256;
  HA_CHECK(wgs <= 0x7fffffff && merges <= 0x7fffffff, "paged_attention_tree: too many workgroups");
  const dim3 grid((unsigned)wgs);
  switch (block_size) {
    case 8: launch_tree_bs<T, HD, 8>(p, pl, grid, stream); break;
    case 32: launch_tree_bs<T, HD, 32>(p, pl, grid, stream); break;
    default: launch_tree_bs<T, HD, 16>(p, pl, grid, stream); break;
  }
  check_launch("paged_attention_tree");
  if (p.num_parts > 1) {
    tree_merge_kernel<T, HD><<<dim3((unsigned)merges), 256, 0, stream>>>(p);
    check_launch("paged_attention_tree (merge)");
  }
}

template <typename T>
void dispatch_tree(const TreeParams &p, const TreePlan &pl, int head_size, int block_size, hipStream_t stream) {
  switch (head_size) {
    case 64: launch_tree<T, 64>(p, pl, block_size, stream); break;
    case 80: launch_tree<T, 80>(p, pl, block_size, stream); break;
    case 96: launch_tree<T, 96>(p, pl, block_size, stream); break;
    case 112: launch_tree<T, 112>(p, pl, block_size, stream); break;
    case 128: launch_tree<T, 128>(p, pl, block_size, stream); break;
    case 256: launch_tree<T, 256>(p, pl, block_size, stream); break;
    default: fail("paged_attention_tree: head size %d not supported (supported: 64, 80, 96, 112, 128, 256)", head_size);
  }
}

size_t tree_piece_bytes(int64_t total_q, int heads, int d) { return (size_t)total_q * heads * (d + 2) * sizeof(float); }
// Parts that there is scratch memory for, at most; 1: none is asked of anybody.
int tree_held_parts(int64_t total_q, int heads, int d) {
  return (int)std::max<size_t>(std::min<size_t>(kTreeScratchBytes / std::max<size_t>(tree_piece_bytes(total_q, heads, d), 1), kTreeMostParts), 1);
}

void paged_attention_tree_impl(const hipattn_tensor *q, const hipattn_tensor *key_cache, const hipattn_tensor *value_cache,
                               const hipattn_tensor *block_tables, const hipattn_tensor *cu_q, const hipattn_tensor *context_lens, int max_q,
                               int max_k, float scale, const hipattn_tensor *mask, hipattn_tensor *out, const hipattn_tensor *workspace,
                               void *stream_arg) {
  const char *op = "paged_attention_tree";
  check_tensor(q, "q", 3);
  check_tensor(out, "out", 3);
  HA_CHECK(out->dtype == q->dtype, "%s: out is %s, q is %s", op, dtype_name(out->dtype), dtype_name(q->dtype));
  const int64_t d = q->sizes[2];
  HA_CHECK(d == 64 || d == 80 || d == 96 || d == 112 || d == 128 || d == 256,
           "%s: head size %lld not supported (supported: 64, 80, 96, 112, 128, 256)", op, (long long)d);
  check_tensor(mask, "tree_mask", 2);
  HA_CHECK(mask->dtype == HIPATTN_I64, "%s: tree_mask must be int64 words of 64 bits, got %s", op, dtype_name(mask->dtype));
  HA_CHECK(mask->sizes[0] == q->sizes[0], "%s: tree_mask has %lld rows, q has %lld", op, (long long)mask->sizes[0], (long long)q->sizes[0]);
  HA_CHECK(mask->sizes[1] <= 1 || mask->strides[1] == 1, "%s: tree_mask rows must be contiguous", op);
  if (workspace) {
    check_tensor(workspace, "workspace", 1);
    HA_CHECK(workspace->dtype == HIPATTN_U8, "%s: workspace must be u8", op);
    check_contiguous(workspace, "workspace");
  }
  PrefillParams pp;
  if (!paged_prefill_params(PagedPrefillCall{q, key_cache, value_cache, block_tables, cu_q, context_lens, max_q, max_k, scale, true, op}, out,
                            nullptr, pp))
    return;
  const int64_t most_rows = std::min<int64_t>(max_q, q->sizes[0]);
  HA_CHECK(mask->sizes[1] * 64 >= most_rows, "%s: tree_mask of %lld words a row does not hold %lld rows", op, (long long)mask->sizes[1],
           (long long)most_rows);
  check_data(mask, "tree_mask");
  HA_CHECK((reinterpret_cast<uintptr_t>(mask->data) & 7) == 0, "%s: tree_mask must be 8-byte aligned", op);
  HA_CHECK(pp.table_cols > 0, "%s: block_tables has no columns", op);
  const int possible = tree_held_parts(pp.total_q, pp.Hq, pp.d);
  char *given = nullptr;
  if (workspace && possible > 1) {
    const size_t need = possible * tree_piece_bytes(pp.total_q, pp.Hq, pp.d);
    HA_CHECK(workspace->data != nullptr && (reinterpret_cast<uintptr_t>(workspace->data) & 255) == 0, "%s: workspace must be 256-byte aligned",
             op);
    HA_CHECK((size_t)workspace->sizes[0] >= need, "%s: workspace of %lld bytes is too small, %zu are needed (hipattn_%s_workspace_size)", op,
             (long long)workspace->sizes[0], need, op);
    given = static_cast<char *>(workspace->data);
  }
  hipStream_t stream = resolve_stream(stream_arg);
  TreePlan pl = plan_tree(pp, stream == hipStreamPerThread && !given ? 1 : possible);
  HeldWorkspace ws;
  void *scratch = given;
  if (pl.num_parts > 1 && !given) {
    ws = try_library_workspace(WS_TREE_ATTENTION, kTreeScratchBytes, stream);
    scratch = ws.ptr;
    if (scratch == nullptr) pl = plan_tree(pp, 1);
  }
  TreeParams p;
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
  p.q = pp.q;
  p.out = pp.out;
  p.q_row = pp.q_row;
  p.q_head = pp.q_head;
  p.o_row = pp.o_row;
  p.o_head = pp.o_head;
  p.total_q = pp.total_q;
  p.cu_q = pp.cu_q;
  p.mask = static_cast<const unsigned long long *>(mask->data);
  p.mask_row = mask->strides[0];
  p.words = (int)std::min<int64_t>(mask->sizes[1], 1 << 24);
  p.batch = pp.batch;
  p.Hq = pp.Hq;
  p.Hkv = pp.Hkv;
  p.G = pp.G;
  p.col_groups = pl.col_groups;
  p.columns = pl.col_groups * 16 * pl.tiles;
  p.max_pairs = pl.max_pairs;
  p.part_pairs = pl.part_pairs;
  p.num_parts = pl.num_parts;
  p.part_acc = static_cast<float *>(scratch);
  p.part_ml = pl.num_parts > 1 ? p.part_acc + (size_t)pl.num_parts * pp.total_q * pp.Hq * pp.d : nullptr;
  if (q->dtype == HIPATTN_F16) dispatch_tree<half_t>(p, pl, pp.d, 1 << pp.block_log2, stream);
  else dispatch_tree<bf16_t>(p, pl, pp.d, 1 << pp.block_log2, stream);
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" char *hipattn_paged_attention_tree(const hipattn_tensor *q, const hipattn_tensor *key_cache, const hipattn_tensor *value_cache,
                                              const hipattn_tensor *block_tables, const hipattn_tensor *cu_seqlens_q,
                                              const hipattn_tensor *context_lens, int max_seqlen_q, int max_seqlen_k, float softmax_scale,
                                              const hipattn_tensor *tree_mask, hipattn_tensor *out, const hipattn_tensor *workspace,
                                              void *stream) {
  HA_PROTECT(paged_attention_tree_impl(q, key_cache, value_cache, block_tables, cu_seqlens_q, context_lens, max_seqlen_q, max_seqlen_k,
                                       softmax_scale, tree_mask, out, workspace, stream));
}

extern "C" char *hipattn_paged_attention_tree_workspace_size(int64_t total_q, int num_heads, int head_size, int64_t *bytes) {
  HA_PROTECT({
    const char *op = "paged_attention_tree_workspace_size";
    HA_CHECK(bytes != nullptr, "%s: bytes is NULL", op);
    HA_CHECK(total_q >= 0 && total_q <= 0x7fffffff && num_heads >= 0 && num_heads <= 1 << 20, "%s: a size is negative or too large", op);
    HA_CHECK(head_size >= 0 && head_size <= 256, "%s: head size %d not supported (at most 256)", op, head_size);
    const int parts = tree_held_parts(total_q, num_heads, head_size);
    *bytes = parts > 1 ? (int64_t)(parts * tree_piece_bytes(total_q, num_heads, head_size)) : 0;
  });
}
