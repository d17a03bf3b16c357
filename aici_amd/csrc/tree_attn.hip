// Attention of trees of drafted tokens over a paged cache: a sequence's n rows see the ctx - n keys in front of the tree and, of the tree's own
// keys (the last n of the context), those that their mask names.
//
//   out[i] = sum_t p[t] v[t] / sum_t p[t],  p[t] = 2^(log2(e) scale q[i].k[t] - m) where t < ctx - n or bit t - (ctx - n) of mask[i] is set, else 0
//
// The rows of a tree with the query heads of a kv group are columns of the decode kernel's products (paged_decode.h), 16 to a tile and two tiles to a
// wavefront (one with heads of 256): 32 tokens' keys and values in registers go through both.  Up to that many columns, where there is little work, and
// where values do not lie on 16-byte boundaries, a workgroup's eight wavefronts take pairs of runs of their own, straight from the cache
// (tree_few_kernel); else wavefronts with different columns read the same pairs from LDS, so that a context is read once for 128 columns
// (tree_many_kernel).  The parts of a long context go to several workgroups, whose results a second launch adds up.
//
// A tree is memory-bound in theory up to some 300 columns (its products per byte of the cache).  Only pairs that reach into the tree look at the mask.
//
// Numerics are those of paged decode: scores and sums in fp32, probabilities rounded to the cache's type as operands of the second product,
// the normaliser not.
#include <algorithm>

#include "paged_decode.h"
#include "prefill_common.h"
#include "prefill_parts.h"

// The copies set M0, and say so; the compiler reports that it is a reserved register.
#pragma clang diagnostic ignored "-Winline-asm"

namespace hipattn {

namespace {

constexpr int kTreeMostParts = 64;
constexpr size_t kTreeScratchBytes = (size_t)128 << 20;

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
  float inv_G;
  int max_rows;  // of a sequence that are looked at
  int part_pairs, num_parts, max_pairs;
  float *part_acc, *part_ml;  // of part i of row r and head h, at (i * total_q + r) * Hq + h: d sums; maximum and sum
};

// Pairs of 16-token runs of a context; what max_seqlen_k does not allow for is left out, as there is no part for it.
__device__ __forceinline__ int tree_pairs(const TreeParams &p, int ctx) {
  return ctx > 0 ? min((int)(((int64_t)ctx + 31) / 32), p.max_pairs) : 0;
}

// Bits j .. j + 63 of a row's mask; bits in front of the tree are set, those behind its n rows are not.  Two words are read whatever they are needed
// for: a condition in front of each makes every one of them a wait (us, 1 tree of 24 rows over 1500 keys, 32 / 8 x 128: 21.5 -> 19.2 with the merge below).
// Compiled, the two of a call still stand behind one condition, that there are rows left, and are waited for there, with all loads in front of them: once for
// each tile in a pair that reaches into the tree, twice where a lane's tokens are of both runs.
__device__ __forceinline__ unsigned long long tree_bits(const unsigned long long *row, int words, int n, int j) {
  const int w = j >> 6, s = j & 63, last = words - 1;
  unsigned long long lo = row[min(max(w, 0), last)], hi = row[min(max(w + 1, 0), last)];
  lo = w < 0 ? ~0ull : (w > last ? 0ull : lo);
  hi = w + 1 < 0 ? ~0ull : (w + 1 > last ? 0ull : hi);
  const unsigned long long bits = s == 0 ? lo : lo >> s | hi << (64 - s);
  const int left = n - j;  // up to the tree's last row
  return left <= 0 ? 0ull : (left < 64 ? bits & ((1ull << left) - 1) : bits);
}

template <typename T>
__device__ __forceinline__ bool not_finite(uint16_t e) {
  constexpr uint16_t top = sizeof(T) == 2 && __is_same(T, half_t) ? 0x7c00 : 0x7f80;
  return (e & top) == top;
}

// What a wavefront knows of its columns: 16 NT of them, from column c0 of the (sequence, kv head) on.
template <typename T, int HD, int NT>
struct TreeColumns {
  typedef typename Vec8<T>::type vec8;
  static constexpr int NSTEP = (HD + 31) / 32, NDT = HD / 16;
  int c0, n, kvh;
  vec8 q[NT][NSTEP];
  float m[NT], l[NT];  // running maximum and sum (l of this lane's tokens alone)
  f32x4_t acc[NT][NDT];

  // Row of the tree and query head of this lane's column of a tile (found anew where needed: they would cost the loop its registers).
  // (a column's number below 2^22: the product with 1 / G is off by less than the half that is added)
  __device__ __forceinline__ int column(int t) const { return c0 + t * 16 + (int)(threadIdx.x & 15); }
  __device__ __forceinline__ int row(const TreeParams &p, int t) const { return (int)(((float)column(t) + 0.5f) * p.inv_G); }
  __device__ __forceinline__ int head(const TreeParams &p, int t) const { return kvh * p.G + column(t) - row(p, t) * p.G; }

  __device__ __forceinline__ void begin(const TreeParams &p, int c0_, int kvh_, int q_begin, int n_) {
    constexpr int NCH = HD / 8;
    const int lane = threadIdx.x & 63, kg = lane >> 4;
    c0 = c0_;
    n = n_;
    kvh = kvh_;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const bool ok = row(p, t) < n;
      const T *qp = static_cast<const T *>(p.q) + (int64_t)(q_begin + row(p, t)) * p.q_row + head(p, t) * p.q_head;
#pragma unroll
      for (int s = 0; s < NSTEP; s++) {
        const int ch = 4 * s + kg;
        u32x4_t raw = {0u, 0u, 0u, 0u};
        if (ok && ch < NCH) raw = *reinterpret_cast<const u32x4_t *>(qp + ch * 8);
        q[t][s] = bit_cast<vec8>(raw);
      }
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int dt = 0; dt < NDT; dt++) acc[t][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
};

// A sequence of a launch.
struct TreeSeq {
  int q_begin, n, ctx, front;  // first row and rows; keys, and those in front of the tree
  const int32_t *table;
};

// Folds the pair of runs from token `tok` on into the columns' states.  The keys are in r; the values as well, or load_values puts them there.  A lane's
// eight tokens are 8 kg .. 8 kg + 7 of the pair (EIGHTS), or 4 kg .. 4 kg + 3 of each run.
// A column's reference maximum moves when a score outgrows it by more than 2^kRescale: until then there is nothing to exchange between lanes, and
// nothing to rescale.  (Probabilities up to 2^kRescale have the relative steps of those up to 1.)
// The tiles go through every step together: with a branch of their own each they wait for their own results (us, 64 trees of 16 to 32 rows over
// up to 15000 keys, 32 / 8 x 128: 585 -> 470).
constexpr float kRescale = 8.f;
template <typename T, int HD, int BS, int NT, bool EIGHTS, typename F>
__device__ __forceinline__ void tree_pair(const TreeParams &p, const TreeSeq &sq, int tok, PairRegs<HD> &r, const T *vbase,
                                          TreeColumns<T, HD, NT> &c, F load_values) {
  typedef typename Vec8<T>::type vec8;
  constexpr int NSTEP = (HD + 31) / 32, NDT = HD / 16;
  const int lane = threadIdx.x & 63, kg = lane >> 4, col = lane & 15;
  const int tok_a = tok + (EIGHTS ? 8 : 4) * kg, tok_b = tok_a + (EIGHTS ? 4 : 16);  // this lane's tokens, four from each on
  float x[NT][8];
  {
    f32x4_t sa[NT], sb[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) sa[t] = sb[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < NSTEP; s++)
#pragma unroll
      for (int t = 0; t < NT; t++) {
        sa[t] = Mfma16<T>::run(bit_cast<vec8>(r.kra[s]), c.q[t][s], sa[t]);
        sb[t] = Mfma16<T>::run(bit_cast<vec8>(r.krb[s]), c.q[t][s], sb[t]);
      }
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[t][i] = sa[t][i];
        x[t][4 + i] = sb[t][i];
      }
  }
  load_values(r);
  unsigned odd = 0;                       // the values of this lane's eight tokens that are not finite, of a pair that reaches into the tree
  unsigned long long seen = ~0ull;        // of the tiles' eight tokens, a byte each
  if (tok + 32 > sq.front) {
    // What lies behind the context is anything, and a probability of zero does not undo it.
#pragma unroll
    for (int dt = 0; dt < NDT; dt++) {
      uint16_t *ea = reinterpret_cast<uint16_t *>(&r.vra[dt]), *eb = reinterpret_cast<uint16_t *>(&r.vrb[dt]);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (tok_a + i >= sq.ctx) ea[i] = 0;
        if (tok_b + i >= sq.ctx) eb[i] = 0;
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
    seen = 0;
    unsigned of_tile[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const unsigned long long *words = p.mask + (int64_t)(sq.q_begin + min(c.row(p, t), sq.n - 1)) * p.mask_row;
      if constexpr (EIGHTS)
        of_tile[t] = (unsigned)tree_bits(words, p.words, sq.n, tok_a - sq.front) & 0xff;
      else
        of_tile[t] = ((unsigned)tree_bits(words, p.words, sq.n, tok_a - sq.front) & 15) | ((unsigned)tree_bits(words, p.words, sq.n, tok_b - sq.front) & 15) << 4;
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const unsigned bits = of_tile[t];
      seen |= (unsigned long long)bits << (8 * t);
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (!(bits >> i & 1)) x[t][i] = -INFINITY;
    }
  }
  const float scale = p.cache.scale_log2;
  float mx[NT];
  bool outgrown = false;
#pragma unroll
  for (int t = 0; t < NT; t++) {
    mx[t] = fmaxf(fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])), fmaxf(fmaxf(x[t][4], x[t][5]), fmaxf(x[t][6], x[t][7]))) * scale;
    outgrown |= mx[t] > c.m[t] + kRescale;
  }
  if (__any(outgrown)) {
#pragma unroll
    for (int t = 0; t < NT; t++) {
      mx[t] = fmaxf(mx[t], __shfl_xor(mx[t], 16, 64));
      mx[t] = fmaxf(mx[t], __shfl_xor(mx[t], 32, 64));
      const float m_new = fmaxf(c.m[t], mx[t]), alpha = fast_exp2(c.m[t] - (m_new == -INFINITY ? 0.f : m_new));
      c.l[t] *= alpha;
      c.m[t] = m_new;
#pragma unroll
      for (int dt = 0; dt < NDT; dt++) c.acc[t][dt] *= alpha;
    }
  }
  vec8 pv[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const float base = c.m[t] == -INFINITY ? 0.f : c.m[t];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float e = fast_exp2(__builtin_fmaf(x[t][i], scale, -base));
      c.l[t] += e;
      pv[t][i] = from_float<T>(e);
    }
  }
#pragma unroll
  for (int dt = 0; dt < NDT; dt++) {
    const u32x4_t a = {r.vra[dt][0], r.vra[dt][1], r.vrb[dt][0], r.vrb[dt][1]};
#pragma unroll
    for (int t = 0; t < NT; t++) c.acc[t][dt] = Mfma16<T>::run(bit_cast<vec8>(a), pv[t], c.acc[t][dt]);
  }
  if (__any(odd != 0)) {
    // Values of the tree that are not finite count for the rows that see them, and for no others: token after token.
    for (int u = 0; u < 32; u++) {
      // the lanes that hold it, and which of their eight it is
      const int from = EIGHTS ? u >> 3 : (u & 15) >> 2, i = EIGHTS ? u & 7 : (u >> 4) * 4 + (u & 3);
      const unsigned long long holders = __ballot(odd >> i & 1) >> (16 * from) & 0xffff;
      if (holders == 0) continue;
      const int token = tok + u;
      int64_t block = token / BS < p.cache.table_cols ? sq.table[token / BS] : 0;
      block = block < 0 ? 0 : (block < p.cache.num_blocks ? block : p.cache.num_blocks - 1);
      const T *v = vbase + block * p.cache.v_block_stride + token % BS;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float e = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (k == i) e = to_float<T>(pv[t][k]);
        e = __shfl(e, from * 16 + col, 64);
        const bool sees = __shfl((int)(seen >> (8 * t + i) & 1), from * 16 + col, 64) != 0;
#pragma unroll
        for (int dt = 0; dt < NDT; dt++)
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const T value = v[(dt * 16 + kg * 4 + k) * BS];
            if (sees && not_finite<T>(bit_cast<uint16_t>(value))) c.acc[t][dt][k] += e * to_float<T>(value);
          }
      }
    }
  }
}

// LDS in which groups of wavefronts with the same columns meet: KG groups of CW.
template <int HD, int NT>
__host__ __device__ constexpr int tree_meet_bytes(int cw, int groups) {
  return groups / 2 * cw * NT * (HD / 16 + 1) * 1024;
}

// The states of the groups, the upper half of them into the lower until one is left; then the outputs, or the part's.
template <typename T, int HD, int NT, int CW, int KG>
__device__ __forceinline__ void tree_finish(const TreeParams &p, const TreeSeq &sq, int part, bool whole, TreeColumns<T, HD, NT> &c, char *lds) {
  constexpr int NDT = HD / 16;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), kg = lane >> 4, cw = wave % CW, group = wave / CW;
#pragma unroll
  for (int t = 0; t < NT; t++) {
    c.l[t] += __shfl_xor(c.l[t], 16, 64);
    c.l[t] += __shfl_xor(c.l[t], 32, 64);
  }
#pragma unroll
  for (int half = KG / 2; half > 0; half /= 2) {
    f32x4_t *place = reinterpret_cast<f32x4_t *>(lds) + (group % half * CW + cw) * NT * (NDT + 1) * 64 + lane;
    __syncthreads();
    if (group >= half && group < 2 * half) {
#pragma unroll
      for (int t = 0; t < NT; t++) {
        place[t * (NDT + 1) * 64] = f32x4_t{c.m[t], c.l[t], 0.f, 0.f};
#pragma unroll
        for (int dt = 0; dt < NDT; dt++) place[(t * (NDT + 1) + 1 + dt) * 64] = c.acc[t][dt];
      }
    }
    __syncthreads();
    if (group < half) {
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const f32x4_t ml = place[t * (NDT + 1) * 64];
        const float top = fmaxf(c.m[t], ml[0]), base = top == -INFINITY ? 0.f : top;
        const float mine = fast_exp2(c.m[t] - base), other = fast_exp2(ml[0] - base);
        c.m[t] = top;
        c.l[t] = c.l[t] * mine + ml[1] * other;
#pragma unroll
        for (int dt = 0; dt < NDT; dt++) c.acc[t][dt] = c.acc[t][dt] * mine + place[(t * (NDT + 1) + 1 + dt) * 64] * other;
      }
    }
  }
  if (group > 0) return;
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int row = c.row(p, t), head = c.head(p, t);
    if (row >= min(sq.n, p.max_rows)) continue;
    if (whole) {
      const float inv = c.l[t] == 0.f ? 0.f : 1.0f / c.l[t];  // (a row that sees nothing is zero, one with a NaN is NaN)
      T *op = static_cast<T *>(p.out) + (int64_t)(sq.q_begin + row) * p.o_row + head * p.o_head + kg * 4;
#pragma unroll
      for (int dt = 0; dt < NDT; dt++) {
        T o[4];
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = from_float<T>(c.acc[t][dt][i] * inv);
        *reinterpret_cast<u32x2_t *>(op + dt * 16) = *reinterpret_cast<u32x2_t *>(o);
      }
    } else {
      const int64_t at = ((int64_t)part * p.total_q + sq.q_begin + row) * p.Hq + head;
#pragma unroll
      for (int dt = 0; dt < NDT; dt++) *reinterpret_cast<f32x4_t *>(p.part_acc + at * HD + dt * 16 + kg * 4) = c.acc[t][dt];
      if (kg == 0) *reinterpret_cast<float2 *>(p.part_ml + 2 * at) = make_float2(c.m[t], c.l[t]);
    }
  }
}

// A context's parts: as many as parts of part_pairs pairs would be, of one length.
struct TreeParts {
  int count, pairs;
  __device__ __forceinline__ TreeParts(const TreeParams &p, int all_pairs) {
    count = max((all_pairs + p.part_pairs - 1) / p.part_pairs, 1);
    pairs = (all_pairs + count - 1) / count;
    if (pairs > 0) count = (all_pairs + pairs - 1) / pairs;
  }
};

// A workgroup's place: sequence, part, column group and kv head, the kv head fastest and the column groups next, so that those that read the same
// keys share an XCD's L2.  Only what there is has a place, one sequence's behind the other's (a workgroup takes a compute unit's whole LDS, if
// only to end at once: 12 trees of 1 to 45 rows, 12 / 4 x 112, 44.4 us with places for the longest of all, 28.8 so), and those with the longest contexts come first, as a launch otherwise ends with
// the few that began one last (us, 64 trees of 16 to 32 rows over up to 15000 keys, 32 / 8 x 128: 470 as they come, 370 so).  By whole wavefronts,
// which ask for all sequences' lengths at once.  False: nothing to do.
struct TreePlace {
  int kvh, cg, part;
  int first, pairs, parts;  // the part's pairs of runs, and the parts of the context
};
constexpr int kTreeSorted = 256;  // sequences, at most, that are put in order
// (rows with columns: at most p.max_rows, whose columns fit 22 bits)
__device__ __forceinline__ int column_groups(const TreeParams &p, int columns, int n) { return (min(n, p.max_rows) * p.G + columns - 1) / columns; }
template <int COLUMNS>
__device__ __forceinline__ bool tree_place(const TreeParams &p, TreeSeq &sq, TreePlace &at) {
  const int lane = threadIdx.x & 63;
  at.kvh = blockIdx.x % p.Hkv;
  const int id = blockIdx.x / p.Hkv;
  // places of a sequence, 0 where its lengths are not those of rows of q
  auto places = [&](int begin, int end, int ctx) {
    const int n = min(end, (int)p.total_q) - begin;
    return begin < 0 || n <= 0 ? 0 : column_groups(p, COLUMNS, n) * TreeParts(p, tree_pairs(p, ctx)).count;
  };
  int seq = -1, local = 0, behind = 0;
  for (int s0 = 0; s0 < p.batch && seq < 0; s0 += 64) {
    const int mine = s0 + lane, s = min(mine, p.batch - 1), ctx = p.cache.context_lens[s], begin = p.cu_q[s], end = p.cu_q[s + 1];
    const int n = mine < p.batch ? places(begin, end, ctx) : 0;
    int before = 0;  // places of the sequences in front of it
    if (p.batch <= kTreeSorted) {
      for (int o0 = 0; o0 < p.batch; o0 += 64) {
        int o_ctx = ctx, o_n = n;
        if (o0 != s0) {
          const int o = min(o0 + lane, p.batch - 1);
          o_ctx = p.cache.context_lens[o];
          o_n = o0 + lane < p.batch ? places(p.cu_q[o], p.cu_q[o + 1], o_ctx) : 0;
        }
        const int others = min(64, p.batch - o0);
        for (int o = 0; o < others; o++) {
          const int theirs = __builtin_amdgcn_readlane(o_ctx, o), theirs_n = __builtin_amdgcn_readlane(o_n, o);
          before += theirs > ctx || (theirs == ctx && o0 + o < mine) ? theirs_n : 0;
        }
      }
    } else {
      int upto = n;
      for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(upto, o, 64);
        if (lane >= o) upto += t;
      }
      before = behind + upto - n;
      behind += __builtin_amdgcn_readlane(upto, 63);
    }
    const unsigned long long hit = __ballot(before <= id && id < before + n);
    if (hit == 0) continue;
    const int l = __builtin_ctzll(hit);
    seq = s0 + l;
    local = id - __builtin_amdgcn_readlane(before, l);
    sq.q_begin = __builtin_amdgcn_readlane(begin, l);
    sq.n = min(__builtin_amdgcn_readlane(end, l), (int)p.total_q) - sq.q_begin;
    sq.ctx = __builtin_amdgcn_readlane(ctx, l);
  }
  if (seq < 0) return false;
  sq.front = sq.ctx - sq.n;
  sq.table = p.cache.block_tables + seq * p.cache.max_blocks;
  const int all_pairs = tree_pairs(p, sq.ctx);
  const TreeParts parts(p, all_pairs);
  const int groups = column_groups(p, COLUMNS, sq.n);
  at.cg = local % groups;
  at.part = local / groups;
  at.parts = parts.count;
  at.first = at.part * parts.pairs;
  at.pairs = min(at.first + parts.pairs, all_pairs) - at.first;
  return true;
}

// Few columns: every wavefront has all of them and pairs of its own, the cache's bytes straight into registers.
template <typename T, int HD, int BS, int NT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void tree_few_kernel(TreeParams p) {
  constexpr int IDS = 32 / BS, HELD = 64 / IDS;  // blocks of a pair; pairs whose blocks' numbers a wavefront's lanes hold
  __shared__ __align__(16) char meet[tree_meet_bytes<HD, NT>(1, WAVES)];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  TreeSeq sq;
  TreePlace at;
  if (!tree_place<16 * NT>(p, sq, at)) return;
  const int c0 = at.cg * 16 * NT;
  TreeColumns<T, HD, NT> c;
  c.begin(p, c0, at.kvh, sq.q_begin, sq.n);
  const T *kbase = static_cast<const T *>(p.cache.kc) + (int64_t)at.kvh * p.cache.k_head_stride;
  const T *vbase = static_cast<const T *>(p.cache.vc) + (int64_t)at.kvh * p.cache.v_head_stride;
  for (int g0 = wave; g0 < at.pairs; g0 += WAVES * HELD) {
    // The blocks of this wavefront's next HELD pairs, IDS lanes to a pair.
    int ids = 0;
    {
      const int64_t pair = (int64_t)at.first + g0 + WAVES * (lane / IDS), column = pair * IDS + lane % IDS;
      if (column < p.cache.table_cols) ids = sq.table[column];
    }
    for (int j = 0; j < HELD && g0 + j * WAVES < at.pairs; j++) {
      PairRegs<HD> r;
      const int l = j * IDS;
      const int64_t i0 = __builtin_amdgcn_readlane(ids, l), i1 = IDS > 1 ? __builtin_amdgcn_readlane(ids, l + 1) : 0;
      const int64_t i2 = IDS > 2 ? __builtin_amdgcn_readlane(ids, l + 2) : 0, i3 = IDS > 2 ? __builtin_amdgcn_readlane(ids, l + 3) : 0;
      pair_load_bs<T, HD, BS, false>(p.cache, kbase, vbase, i0, i1, i2, i3, r);
      tree_pair<T, HD, BS, NT, false>(p, sq, (at.first + g0 + j * WAVES) * 32, r, vbase, c, [](PairRegs<HD> &) {});
    }
  }
  tree_finish<T, HD, NT, 1, WAVES>(p, sq, at.part, at.parts == 1, c, meet);
}

__device__ __forceinline__ void tree_copy_1k(uint32_t lds, const char *base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void tree_copy_1k_at(uint32_t lds, const char *at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(lds), "v"(at) : "memory", "m0");
}

// Many columns: CW wavefronts of 16 NT columns each read the same pairs from LDS, where they are copied to in rounds of P pairs, S of them in a ring; the
// 8 / CW groups of such wavefronts take pairs of their own of a round.  In LDS a run of 16 tokens of K lies about as in a 16-token block, [16-byte run
// of d][token], and one of V as well, [d][token], whatever the cache's block size: a lane's 16 bytes can come from anywhere.  The rows of the first
// product's tiles are chosen so that a lane's probabilities belong to eight tokens in a row, 16 bytes of V; for operand reads without bank
// conflicts the two halves of V's rows change places in every second eight of them, and tokens 4 to 7 of K with 0 to 3 (12 to 15 with 8 to 11) in
// the second run.
// Wavefront w copies images w, w + 8, .. of a round: K and V of both runs of its pairs.
template <int HD>
constexpr int tree_image_bytes() { return (HD * 32 + 1023) / 1024 * 1024; }
template <int HD, int P>
constexpr int tree_ring_rounds() {
  constexpr int fit = 144 * 1024 / (P * 4 * tree_image_bytes<HD>());
  return fit > 8 ? 8 : fit;
}

template <typename T, int HD, int BS, int NT, int CW, int P>
__global__ __launch_bounds__(512) void tree_many_kernel(TreeParams p) {
  constexpr int KG = 8 / CW, PW = P / KG, S = tree_ring_rounds<HD, P>(), IMG = tree_image_bytes<HD>(), IMAGES = P * 4 / 8, PIECES = IMG / 1024;
  constexpr int kCopies = IMAGES * PIECES;
  static_assert(P % KG == 0 && P * 4 % 8 == 0 && S >= 2, "rounds divide evenly");
  constexpr int kRing = S * P * 4 * IMG, kMeet = tree_meet_bytes<HD, NT>(CW, KG);
  __shared__ __align__(1024) char ring[kRing > kMeet ? kRing : kMeet];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), kg = lane >> 4, col = lane & 15;
  const int cw = wave % CW, group = wave / CW;
  TreeSeq sq;
  TreePlace at;
  if (!tree_place<16 * NT * CW>(p, sq, at)) return;
  const int c0 = (at.cg * CW + cw) * 16 * NT;
  const bool idle = c0 >= min(sq.n, p.max_rows) * p.G;  // without a column: the wavefront copies and no more
  const T *kbase = static_cast<const T *>(p.cache.kc) + (int64_t)at.kvh * p.cache.k_head_stride;
  const T *vbase = static_cast<const T *>(p.cache.vc) + (int64_t)at.kvh * p.cache.v_head_stride;
  const uint32_t ring_lds = uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)ring);
  const int rounds = (at.pairs + P - 1) / P;

  // Image i of this wavefront's is that of K (even) or V of run (wave + 8 i) / 2 % 2 of pair (wave + 8 i) / 4 of a round: always the same kind and run.
  static_assert(P <= 4, "a wavefront's images lie two pairs apart");
  const bool is_v = wave & 1;
  const int run_in_pair = wave >> 1 & 1;
  // Blocks of the next 64 rounds, a lane for each; with 8-token blocks those of both halves of the run.
  int ids[IMAGES][BS == 8 ? 2 : 1];
  auto fetch_ids = [&](int round0) {
#pragma unroll
    for (int i = 0; i < IMAGES; i++) {
      const int64_t pair = (int64_t)at.first + (int64_t)(round0 + lane) * P + (wave >> 2) + 2 * i, run = pair * 2 + run_in_pair;
#pragma unroll
      for (int h = 0; h < (BS == 8 ? 2 : 1); h++) {
        const int64_t column = BS == 8 ? 2 * run + h : (BS == 32 ? run / 2 : run);
        int id = column < p.cache.table_cols ? sq.table[column] : 0;
        ids[i][h] = id < 0 ? 0 : (id < p.cache.num_blocks ? id : (int)p.cache.num_blocks - 1);
      }
    }
  };
  // (used as soon as they are there, so that what uses them later does not wait for the copies in front of it every time)
  auto use_ids = [&]() {
#pragma unroll
    for (int i = 0; i < IMAGES; i++)
#pragma unroll
      for (int h = 0; h < (BS == 8 ? 2 : 1); h++) asm volatile("" : "+v"(ids[i][h]));
  };
  // A lane's place in a piece of an image, in bytes from the block's start; from piece to piece it moves on by as much.  Beyond the image, where it
  // does not fill its last piece: the image's last 16 bytes.
  constexpr int STEP = BS == 16 ? 1024 : (BS == 32 ? 2048 : 512);
  constexpr bool RAGGED = HD * 32 % 1024 != 0;
  // K: (run of d, token); V: (d, half of the tokens)
  auto token_of = [&](int r) { return (r & 15) ^ (run_in_pair ? 4 : 0); };
  auto half_of = [&](int r) { return (r & 1) ^ (r >> 4 & 1); };
  auto place_of = [&](int r) -> uint32_t {
    if (BS == 8) return is_v ? (r >> 1) * 16 : ((r >> 4) * 8 + (token_of(r) & 7)) * 16;
    const int wide = BS / 16, of_run = BS == 32 ? run_in_pair : 0;
    return is_v ? ((r >> 1) * 2 * wide + of_run * 2 + half_of(r)) * 16 : ((r >> 4) * 16 * wide + of_run * 16 + token_of(r)) * 16;
  };
  auto second = [&](int r) { return is_v ? half_of(r) != 0 : token_of(r) >= 8; };  // 8-token blocks: of the run's second block
  const int tail = min((PIECES - 1) * 64 + lane, HD * 2 - 1);
  const uint32_t off = place_of(lane), off_last = place_of(tail) - (PIECES - 1) * STEP;
  const bool upper = second(lane), upper_last = second(tail);
  const char *base = reinterpret_cast<const char *>(is_v ? vbase : kbase);
  const int64_t stride = (is_v ? p.cache.v_block_stride : p.cache.k_block_stride) * (int64_t)sizeof(T);
  auto ask = [&](int slot, int round) {
    if (round > 0 && (round & 63) == 0) {
      fetch_ids(round);
      use_ids();
    }
#pragma unroll
    for (int i = 0; i < IMAGES; i++) {
      const uint32_t to = ring_lds + ((slot * P + (wave >> 2) + 2 * i) * 4 + (wave & 3)) * IMG;
      const char *b0 = uniform_ptr(base + (int64_t)__builtin_amdgcn_readlane(ids[i][0], round & 63) * stride);
      if constexpr (BS == 8) {
        const char *b1 = uniform_ptr(base + (int64_t)__builtin_amdgcn_readlane(ids[i][1], round & 63) * stride);
#pragma unroll
        for (int k = 0; k < PIECES; k++) {
          const bool last = RAGGED && k == PIECES - 1;
          tree_copy_1k_at(to + k * 1024, ((last ? upper_last : upper) ? b1 : b0) + (last ? off_last : off) + k * STEP);
        }
      } else {
#pragma unroll
        for (int k = 0; k < PIECES; k++) tree_copy_1k(to + k * 1024, b0 + k * STEP, RAGGED && k == PIECES - 1 ? off_last : off);
      }
    }
  };
  TreeColumns<T, HD, NT> c;
  fetch_ids(0);
  c.begin(p, c0, at.kvh, sq.q_begin, sq.n);
  use_ids();
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int s = 0; s < (HD + 31) / 32; s++) asm volatile("" : "+v"(c.q[t][s]));  // (as above)
#pragma unroll
  for (int j = 0; j < S - 1; j++)
    if (j < rounds) ask(j, j);
  int slot = 0;
  for (int round = 0; round < rounds; round++) {
    // This wavefront's copies of the round have landed, and behind the barrier everybody's; the barrier also says that the round before has been
    // read, so its place takes the copies of the round S - 1 further on.
    if (round + S - 2 < rounds) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * kCopies) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    if (round + S - 1 < rounds) ask(slot == 0 ? S - 1 : slot - 1, round + S - 1);
    const char *images = ring + slot * P * 4 * IMG;
    slot = slot == S - 1 ? 0 : slot + 1;
    if (idle) continue;
#pragma unroll
    for (int j = 0; j < PW; j++) {
      const int u = group * PW + j, pair = round * P + u;
      if (pair >= at.pairs) break;
      const char *im = images + u * 4 * IMG;
      PairRegs<HD> r;
      // rows of the first product: tokens 8 (row / 4) + row % 4 of the pair, and four further on
      const int place_a = (8 * (col >> 2 & 1) + (col & 3)) ^ (col >= 8 ? 4 : 0);
      const char *keys = im + (col >> 3) * 2 * IMG;
#pragma unroll
      for (int s = 0; s < (HD + 31) / 32; s++) {
        const int ch = 4 * s + kg;
        r.kra[s] = r.krb[s] = u32x4_t{0u, 0u, 0u, 0u};
        if (HD / 8 % 4 == 0 || ch < HD / 8) {
          r.kra[s] = *reinterpret_cast<const u32x4_t *>(keys + (ch * 16 + place_a) * 16);
          r.krb[s] = *reinterpret_cast<const u32x4_t *>(keys + (ch * 16 + (place_a ^ 4)) * 16);
        }
      }
      tree_pair<T, HD, BS, NT, true>(p, sq, (at.first + pair) * 32, r, vbase, c, [&](PairRegs<HD> &r) {
#pragma unroll
        for (int dt = 0; dt < HD / 16; dt++) {
          const u32x4_t v = *reinterpret_cast<const u32x4_t *>(im + (1 + (kg >> 1) * 2) * IMG + (dt * 16 + col) * 32 + (((kg & 1) ^ (col >> 3)) * 16));
          r.vra[dt] = u32x2_t{v[0], v[1]};
          r.vrb[dt] = u32x2_t{v[2], v[3]};
        }
      });
    }
  }
  tree_finish<T, HD, NT, CW, KG>(p, sq, at.part, at.parts == 1, c, ring);
}

// The merge: a thread for four elements of a (row, head), workgroups of 256 of a row; parts eight at a time, all of which are asked for at once.
template <typename T, int HD>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeParams p) {
  constexpr int QUADS = HD / 4, kAtOnce = 8;
  const int of_row = (p.Hq * QUADS + 255) / 256, r = blockIdx.x / of_row, i = blockIdx.x % of_row * 256 + threadIdx.x;
  const int h = i / QUADS, e = i % QUADS * 4;
  const int seq = sequence_of_row(p.cu_q, p.batch, r);
  if (seq < 0 || h >= p.Hq) return;
  const int parts = TreeParts(p, tree_pairs(p, p.cache.context_lens[seq])).count;
  if (parts == 1 || r - p.cu_q[seq] >= p.max_rows) return;  // written, or left out
  const int64_t step = p.total_q * p.Hq, rh = (int64_t)r * p.Hq + h;
  float top = -INFINITY, sum = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < parts; k0 += kAtOnce) {
    float2 ml[kAtOnce];
    f32x4_t a[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; k++) {
      const int64_t at = min(k0 + k, parts - 1) * step + rh;
      ml[k] = *reinterpret_cast<const float2 *>(p.part_ml + 2 * at);
      a[k] = *reinterpret_cast<const f32x4_t *>(p.part_acc + at * HD + e);
    }
    float most = top;
#pragma unroll
    for (int k = 0; k < kAtOnce; k++) most = fmaxf(most, ml[k].x);
    const float base = most == -INFINITY ? 0.f : most, before = fast_exp2(top - base);
    top = most;
    sum *= before;
    o *= before;
#pragma unroll
    for (int k = 0; k < kAtOnce; k++) {
      if (k0 + k >= parts) continue;
      const float w = fast_exp2(ml[k].x - base);
      sum += w * ml[k].y;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] += w * a[k][j];
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  T out[4];
#pragma unroll
  for (int j = 0; j < 4; j++) out[j] = from_float<T>(o[j] * inv);
  *reinterpret_cast<u32x2_t *>(static_cast<T *>(p.out) + (int64_t)r * p.o_row + (int64_t)h * p.o_head + e) = *reinterpret_cast<u32x2_t *>(out);
}

// How columns and keys are dealt out.
struct TreePlan {
  int tiles;  // of 16 columns to a wavefront
  int cw;     // wavefronts beside one another that share pairs in LDS, 4; 0: every wavefront pairs of its own
  int part_pairs, num_parts, max_pairs;
  int64_t groups;  // (sequence, column group, kv head), at most
};

TreePlan plan_tree(const PrefillParams &p, int most_parts) {
  TreePlan pl;
  const int64_t cols = (int64_t)std::min<int64_t>(p.max_q, p.total_q) * p.G;
  const int64_t pairs = std::max<int64_t>(((int64_t)p.max_k + 31) / 32, 1);
  // (column groups that trees of these rows together can have)
  const auto groups_of = [&](int wide) {
    return std::min<int64_t>((cols + wide - 1) / wide * p.batch, (p.total_q * p.G) / wide + p.batch) * p.Hkv;
  };
  pl.max_pairs = (int)pairs;
  // Little work, that a workgroup to a compute unit does in twelve rounds of its wavefronts: columns in groups of 16, each with the keys to itself, start
  // some 5 us sooner than those that share them.  us, so / with groups of 128: 1 tree of 24 rows over 1500 keys, 32 / 8 x 128 13.2 / 19.2, 8 of 12 over up
  // to 3000 25.9 / 34.3, 4 of 24 over up to 6000, 12 / 4 x 112 23.0 / 35.6; at sixteen rounds 12 of 1 to 45 over up to 4000, 12 / 4 x 112 28.3 / 26.0.
  const int64_t alone = compute_units() / groups_of(16);
  if (alone > 0 && pairs <= alone * 96) {
    pl.cw = 0;
    pl.tiles = 1;
    pl.groups = groups_of(16);
    const int64_t parts = std::min<int64_t>(std::min<int64_t>(alone, most_parts), (pairs + 7) / 8);
    pl.part_pairs = (int)((pairs + parts - 1) / parts);
    pl.num_parts = (int)((pairs + pl.part_pairs - 1) / pl.part_pairs);
    return pl;
  }
  // Values go into LDS in pieces of 16 bytes; where blocks or heads of the cache do not keep to such boundaries every wavefront reads its own, by 8 (us, 64
  // trees over 1000 to 15000 keys, 32 / 8 x 128, blocks apart by a multiple of 16 bytes / of 8: 8 rows 365 / 365, 24 rows, 96 columns, 380 / 571, as 32 columns
  // at a time read the keys).
  // Up to 32 columns as well, which the other form would do in less time over long contexts: us, own pairs / shared ones, 64 trees of 5, 6, 8 rows over 1000
  // to 15000 keys, 32 / 8 x 128 364 / 325, 365 / 326, 365 / 328; 16 of 8 124 / 113; 64 of 30 over 1000 to 8000, 32 / 32 x 80 543 / 525; 8 of 5 over 500
  // to 8000 43.6 / 43.6.
  const bool shares = p.vc_block % 8 == 0 && p.vc_head % 8 == 0;
  pl.cw = !shares || cols <= (p.d > 128 ? 16 : 32) ? 0 : 4;
  pl.tiles = p.d > 128 || cols <= 16 || (pl.cw > 0 && cols > 32 && cols <= 64) ? 1 : 2;
  const int64_t groups = groups_of(16 * pl.tiles * std::max(pl.cw, 1));
  // Parts for two workgroups to a compute unit, or one where there are few sequences, whose lengths differ less: what a workgroup takes before its first
  // keys are there is some 8 us.  us, for one / two / four / eight: 2 trees of 40 rows over up to 8000 keys, 32 / 8 x 128 38 / 49 / - / -; 12
  // trees of 1 to 45 rows over up to 4000 keys, 12 / 4 x 112 38 / 29 / 40 / 39; 8 of 64 over up to 8000, 32 / 32 x 80 87 / 88 / 93 / 108; 64 of 16 to 32
  // over up to 15000, 32 / 8 x 128 386 / 386 / 446 / 482.  No part of less than 8 pairs (1 of 24 over 1500, 32 / 8 x 128, of 2 / 4 / 8 / 16 pairs at least
  // 26.6 / 21.6 / 21.2 / 24.0).
  int64_t parts = std::max<int64_t>((int64_t)(p.batch <= 4 ? 1 : 2) * compute_units() / std::max<int64_t>(groups, 1), 1);
  parts = std::min<int64_t>(std::min<int64_t>(parts, most_parts), (pairs + 7) / 8);
  pl.part_pairs = (int)((pairs + parts - 1) / parts);
  pl.num_parts = (int)((pairs + pl.part_pairs - 1) / pl.part_pairs);
  pl.groups = groups;
  return pl;
}

template <typename T, int HD, int BS>
void launch_tree_bs(const TreeParams &p, const TreePlan &pl, dim3 grid, hipStream_t stream) {
  if (pl.cw == 0 && pl.tiles == 1) tree_few_kernel<T, HD, BS, 1, (HD > 128 ? 4 : 8)><<<grid, HD > 128 ? 256 : 512, 0, stream>>>(p);
  else if (pl.tiles == 1) tree_many_kernel<T, HD, BS, 1, 4, 2><<<grid, 512, 0, stream>>>(p);
  else if constexpr (HD <= 128) {
    if (pl.cw == 0) tree_few_kernel<T, HD, BS, 2, 8><<<grid, 512, 0, stream>>>(p);
    else tree_many_kernel<T, HD, BS, 2, 4, 2><<<grid, 512, 0, stream>>>(p);
  }
}

template <typename T, int HD>
void launch_tree(const TreeParams &p, const TreePlan &pl, int block_size, hipStream_t stream) {
  const int64_t wgs = pl.groups * p.num_parts, merges = p.total_q * ((p.Hq * (HD / 4) + 255) / 256);
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
  HA_CHECK(most_rows * pp.G < 1 << 22, "%s: trees of %lld rows of %d heads a kv group are too large", op, (long long)most_rows, pp.G);
  HA_CHECK(mask->sizes[1] * 64 >= most_rows, "%s: tree_mask of %lld words a row does not hold %lld rows", op, (long long)mask->sizes[1],
           (long long)most_rows);
  check_data(mask, "tree_mask");
  HA_CHECK((reinterpret_cast<uintptr_t>(mask->data) & 7) == 0, "%s: tree_mask must be 8-byte aligned", op);
  HA_CHECK(pp.table_cols > 0, "%s: block_tables has no columns", op);
  // A workgroup has all that it reads of q before it writes, and nobody else reads those heads of those rows.
  HA_CHECK((out->data == q->data && (pp.total_q == 1 || out->strides[0] == q->strides[0]) && (pp.Hq == 1 || out->strides[1] == q->strides[1])) ||
               !may_share(out, q),
           "%s: out lies over part of q", op);
  const struct {
    const hipattn_tensor *t;
    const char *name;
  } others[] = {{key_cache, "key_cache"}, {value_cache, "value_cache"}, {block_tables, "block_tables"}, {cu_q, "cu_seqlens_q"},
                {context_lens, "context_lens"}, {mask, "tree_mask"}};
  for (const auto &o : others) HA_CHECK(!may_share(out, o.t), "%s: out lies over %s", op, o.name);
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
  p.inv_G = 1.0f / (float)pp.G;
  p.max_rows = (int)most_rows;
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
