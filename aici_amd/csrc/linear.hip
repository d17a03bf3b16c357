// Linear layer for a handful of rows: y = x · Wᵀ (+ bias) (+ residual) with at most 128 rows of x -- the
// projections of a generation step (rllm/rllm-cuda/src/llm/llama.rs:81-83, 96, 135-143, 210 through
// `linear_no_bias`, llm/mod.rs:401-407; phi.rs:70-71, 99, 116-117 through `linear`, mod.rs:409-416), where every
// element of W is used once per row of x and the time goes into reading W from HBM exactly once.
//
// The kernels copy W and x global -> LDS (global_load_lds_dwordx4, no registers) into a ring of stages of 64 values
// of k: an instruction brings 128 whole bytes of eight rows, its runs of 16 bytes swizzled by the row's low bits so that the
// operands of v_mfma_f32_16x16x32 are read from LDS without bank conflicts.  What bounds them is how many whole
// cache lines are on their way: the same loop with W loaded straight into the operands (16 rows x 64 bytes per instruction, so
// every line asked for twice, and both copies of it held in the 32 KB L1) reached 5.1 TB/s on a 28672 x 4096 weight and one row of x,
// 4.0 with sixteen; this form 5.9 and 5.4, and with ranges of k that begin inside (StageOrder) 6.5 and 6.4 (library GEMM: 4.0 / 3.9).
//
//   linear_stream_kernel, up to 16 rows of x and a weight whose k is cut into ranges: a wavefront owns 16 rows of W and keeps a private
//   ring, its own copy of the rows of x in it, so nothing waits for anything but the wavefront's own copies; wavefronts that share
//   rows of W take different ranges of k and meet once, in LDS, at the end.
//   norm_linear_kernel, up to 4 rows with the RMS norm in front: the rows are held in LDS whole and normalised there, the ring is W's alone.
//   linear_tile_kernel, 17 to 128 rows, fewer where k is not cut: the copies of x are shared by the workgroup (one barrier per stage); ranges of k
//   go to workgroups of their own, which leave fp32 sums for a second launch to add up.
//
// The ranges of k are a function of the weight's shape alone, every range is summed front to back and the ranges are
// added up first to last: a row gets the same bits whichever kernel, launch shape and company it is computed in, and
// on every run (no atomics).  Front to back: from a stage of the range on that follows from the row of W, and round (StageOrder).
//
// Microseconds (bf16, copies of W in turns so that no cache holds it; library GEMM -> here):
//                       1 row          16 rows        32 rows        64 rows        128 rows
//   4096 x 4096         22.8 -> 7.7    20.8 -> 8.2    21.1 -> 11.3   21.1 -> 12.2   24.2 -> 16.1
//   6144 x 4096         20.8 -> 10.9   19.8 -> 12.7   19.8 -> 14.5   19.6 -> 16.6   25.3 -> 21.3
//   4096 x 14336        25.6 -> 19.2   25.8 -> 22.7   30.8 -> 24.9   38.9 -> 27.0   75.3 -> 31.4
//   28672 x 4096        58.8 -> 36.4   59.8 -> 36.8   51.2 -> 38.4   51.4 -> 39.2   53.9 -> 49.3
//     + silu_and_mul    62.9 -> 36.5   64.2 -> 36.5   56.8 -> 38.5   57.9 -> 39.4   61.0 -> 50.3
//   128256 x 4096       183 -> 152     186 -> 154     197 -> 161     209 -> 176     233 -> 219
// (one row of 28672 x 4096 is 6.5 TB/s, 128 rows are 4.8.  At that end every workgroup copies as many bytes of x into LDS as of W and
// has the compute unit to itself, its start and end open; the reads of x from LDS, eight times the bytes of W, are not what bounds it:
// a third fewer of them changed nothing.)
// Narrower weights keep these kernels' lead: 1024 x 4096 13.6 -> 6.4 with one row and 18.3 -> 12.7 with 128 against a kernel that cut them
// into up to 32 ranges and always added the ranges up in a second launch, 1024 x 14336 with 16 rows 22.0 -> 19.4.
//
// Rounding points: fp32 accumulation over k, + bias in fp32, rounded to T -- what a library GEMM with a bias epilogue
// does; then, if a residual is given, T(y + residual): the separate addition of llama.rs:166, 173, rounded again.
#include "cache_geom.h"
#include "common.h"
#include "device_types.h"
#include "workspace.h"

#include <type_traits>

// The copies set M0, and say so; the compiler reports that it is a reserved register.
#pragma clang diagnostic ignored "-Winline-asm"

namespace hipattn {
namespace {

constexpr int kLinMaxRows = 128;  // rows of x
constexpr int kLinMT = 8;         // 16-row tiles of x
constexpr int kLinStageK = 64;    // values of k per stage: 128 bytes of a row
constexpr int kLinStreamRows = 16;
constexpr int kLinHeldRows = 4;
// Of x and the norm's weight: two workgroups of four wavefronts per compute unit, where the ranges' sums take 4 KB (16 at most); one of eight
// (64 KB of ring, 8 of sums), which has the unit to itself (wide_workgroups).
constexpr int kLinHeldBytes = 40 * 1024;
constexpr int kHeldStages = 4;
constexpr int kLinMaxRanges = 8;  // ranges of k that the library itself chooses

// Behind the projection of q, k and v: the rotation of the query and key heads and the writes of keys and values to the cache.
struct QkvParams {
  const void *positions, *slots, *cos_sin;  // cos_sin: rows of head_size values, cosines first
  bool pos64, slot64;
  int64_t max_pos;
  int q_heads;
  void *key_cache, *value_cache;
  CacheGeom g;
};

struct LinearParams {
  const void *x, *w, *bias, *residual;
  void *out;
  float *partial;
  int M, N, K;
  int mtiles;  // ceil(M / 16)
  int64_t ldx, ldw, ldr, ldo;
  int splits, stages_per_split, total_stages;  // ranges of k
  // silu_and_mul behind the layer: W holds `half` gate rows and then as many up rows, the output has `half` columns
  int half;
  // with an RMS norm behind the layer: the sums go to the workspace as rows ([range][128 rows][N] fp32), and the
  // launch that adds them up also normalises the finished row
  int row_sums;
  int turned;     // ranges of k begin inside (StageOrder), the order that of a row's place in this many; 0: they do not
  int wide;       // rows of x or W more than 2^28 elements apart
  int tile_sums;  // the sums go to the workspace as tiles, and a second launch finishes them
  const void *norm_w;
  void *norm_out;
  int64_t ldn;
  float eps;
  int norm_in;  // the norm is that of the rows of x, in front of the layer
  QkvParams qkv;
};

template <typename T>
struct LinMfma;
template <>
struct LinMfma<half_t> {
  static __device__ __forceinline__ f32x4_t run(half8_t a, half8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct LinMfma<bf16_t> {
  static __device__ __forceinline__ f32x4_t run(bf16x8_t a, bf16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// v[r] = the fp32 sum for y[m][n + r], r = 0..3: bias, rounding, residual, one 8-byte store.
template <typename T>
__device__ __forceinline__ void linear_finish(const LinearParams &p, f32x4_t v, int m, int n) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  if (m >= p.M || n >= p.N) return;
  const T *bias = static_cast<const T *>(p.bias);
  const T *res = static_cast<const T *>(p.residual);
  vec4 b4 = vec4{(T)0.f, (T)0.f, (T)0.f, (T)0.f}, r4 = b4, o;
  if (bias != nullptr) b4 = *reinterpret_cast<const vec4 *>(bias + n);
  if (res != nullptr) r4 = *reinterpret_cast<const vec4 *>(res + (int64_t)m * p.ldr + n);
#pragma unroll
  for (int r = 0; r < 4; r++) {
    float f = v[r];
    if (bias != nullptr) f += to_float<T>(b4[r]);
    T y = from_float<T>(f);
    if (res != nullptr) y = add_t<T>(y, r4[r]);
    o[r] = y;
  }
  *reinterpret_cast<vec4 *>(static_cast<T *>(p.out) + (int64_t)m * p.ldo + n) = o;
}

// The same for a gated layer: gate and up sums of y[m][n + r], each rounded, then the arithmetic of silu_and_mul.
template <typename T>
__device__ __forceinline__ void linear_finish_gated(const LinearParams &p, f32x4_t gate, f32x4_t up, int m, int n) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  if (m >= p.M || n >= p.half) return;
  vec4 o;
#pragma unroll
  for (int r = 0; r < 4; r++) o[r] = mul_t<T>(silu_t<T>(from_float<T>(gate[r])), from_float<T>(up[r]));
  *reinterpret_cast<vec4 *>(static_cast<T *>(p.out) + (int64_t)m * p.ldo + n) = o;
}

// Rows of W of tile `tile` (16 of them): of a head that is rotated eight rows from its first half and the eight that they are rotated
// with, so that a wavefront's sums hold both; else sixteen in order.
struct QkvRows {
  int first, second;  // of eight rows each
  int head;
  bool rotated;
};
__device__ __forceinline__ QkvRows qkv_rows(const QkvParams &q, int tile) {
  const int hd = q.g.head_size, n = tile * 16, head = n / hd, r = (n - head * hd) / 2;
  QkvRows t;
  t.head = head;
  t.rotated = head < q.q_heads + q.g.num_heads;
  t.first = t.rotated ? head * hd + r : n;
  t.second = t.first + (t.rotated ? hd / 2 : 8);
  return t;
}

// Position and slot of row m: asked for in front of the weight's copies, needed behind them.
struct QkvToken {
  int64_t pos, slot;
};
__device__ __forceinline__ QkvToken qkv_token(const QkvParams &q, int m) {
  QkvToken t;
  t.pos = q.pos64 ? static_cast<const int64_t *>(q.positions)[m] : (int64_t)static_cast<const int32_t *>(q.positions)[m];
  t.slot = q.slot64 ? static_cast<const int64_t *>(q.slots)[m] : (int64_t)static_cast<const int32_t *>(q.slots)[m];
  return t;
}
template <typename T>
struct QkvTurn {  // cosines and sines of a lane's four elements
  typedef T vec4 __attribute__((ext_vector_type(4)));
  vec4 c, s;
  bool rotate;
};
template <typename T>
__device__ __forceinline__ QkvTurn<T> qkv_turn(const QkvParams &q, const QkvRows &rows, const QkvToken &tok, int kg) {
  using vec4 = typename QkvTurn<T>::vec4;
  const int hd = q.g.head_size;
  QkvTurn<T> t;
  t.rotate = rows.rotated && tok.pos >= 0 && tok.pos < q.max_pos;
  t.c = t.s = vec4{(T)0.f, (T)0.f, (T)0.f, (T)0.f};
  if (t.rotate) {
    const T *at = static_cast<const T *>(q.cos_sin) + tok.pos * hd + (rows.first - rows.head * hd) + 4 * (kg & 1);
    t.c = *reinterpret_cast<const vec4 *>(at);
    t.s = *reinterpret_cast<const vec4 *>(at + hd / 2);
  }
  return t;
}

// linear_finish for such a tile, with the arithmetic of rotary_cache_kernel on the rounded products, so its bits.  A launch of a few
// kilobytes less, for one more dependent load (the table's row) at the end of this one.  us, the projection and the launch behind it /
// together, weights cold: 6144 x 4096 (32 / 8 heads of 128) 1 row 15.3 / 11.6, 16 17.4 / 13.8, 32 19.7 / 16.4, 128 26.2 / 23.2; 7680 x
// 2560 (32 / 32 of 80) 14.0 / 9.5, 16.1 / 11.6, 19.9 / 15.7, 25.0 / 22.6; 12288 x 4096 27.7 / 22.4, 31.0 / 25.8, 32.5 / 28.4, 40.4 / 40.0.
// From 16384 rows of weight on the sums of more than 16 rows of x are finished in the tile kernel: not built for it.
template <typename T>
__device__ __forceinline__ void linear_finish_qkv(const LinearParams &p, f32x4_t v, int m, int kg, const QkvRows &rows, const QkvToken &tok,
                                                  const QkvTurn<T> &turn) {
  using vec4 = typename QkvTurn<T>::vec4;
  const QkvParams &q = p.qkv;
  const int hd = q.g.head_size;
  vec4 mine, o;
#pragma unroll
  for (int r = 0; r < 4; r++) mine[r] = from_float<T>(v[r]);
  const uint2 raw = bit_cast<uint2>(mine);
  const vec4 other = bit_cast<vec4>(make_uint2((uint32_t)__shfl_xor((int)raw.x, 32), (uint32_t)__shfl_xor((int)raw.y, 32)));
  const bool high = kg >= 2;
  o = mine;
  if (turn.rotate) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const T here = mul_t<T>(mine[r], turn.c[r]), there = mul_t<T>(other[r], turn.s[r]);
      o[r] = high ? add_t<T>(here, there) : sub_t<T>(here, there);
    }
  }
  const int n = (high ? rows.second : rows.first) + 4 * (kg & 1);
  if (m >= p.M || n >= p.N) return;
  *reinterpret_cast<vec4 *>(static_cast<T *>(p.out) + (int64_t)m * p.ldo + n) = o;
  if (rows.head < q.q_heads) return;
  int off;
  const int64_t blk = slot_block(tok.slot, q.g, off);
  if (blk < 0) return;
  const int i = n - rows.head * hd;  // element of the head
  if (rows.rotated) {
    T *kc = static_cast<T *>(q.key_cache) + blk * q.g.k_block_stride + (rows.head - q.q_heads) * q.g.k_head_stride;
    *reinterpret_cast<vec4 *>(kc + ((int64_t)(i / 8) * q.g.block_size + off) * 8 + (i & 7)) = o;
  } else {
    T *vc = static_cast<T *>(q.value_cache) + blk * q.g.v_block_stride + (rows.head - q.q_heads - q.g.num_heads) * q.g.v_head_stride;
#pragma unroll
    for (int r = 0; r < 4; r++) vc[(int64_t)(i + r) * q.g.block_size + off] = o[r];
  }
}

// The order in which a wavefront takes the stages of its ranges, one after the other: a range begins at a stage that follows from the
// rows of W, and wraps round.  Wavefronts that all walk their rows front to back ask for the same bytes of every row at a time, and
// where rows lie 8 KB apart those are a few of the memory's channels (see LinearPlan::turned).  kTurnRows rows of W share a place, and the
// two halves of the weight have the same ones (gate and up rows of an output share their copies of x): the order is that of the row,
// whatever the kernel and the launch.
constexpr int kTurnRows = 128;
struct StageOrder {
  int per_range, stages, turn;
  int at = 0, end = 0, left = 0, start;
  // n: a row of the tile
  __device__ __forceinline__ StageOrder(const LinearParams &p, int n, int stages_)
      : per_range(p.stages_per_split), stages(stages_), turn(p.turned ? n % p.turned / kTurnRows * 21 : 0), start(-p.stages_per_split) {}
  __device__ __forceinline__ int next() {
    if (left == 0) {
      start += per_range;
      left = min(per_range, stages - start);
      at = start + (int)((unsigned)turn % (unsigned)left);
      end = start + left;
    }
    const int st = at;
    at = at + 1 == end ? start : at + 1;
    left--;
    return st;
  }
};

template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <typename P>
__device__ __forceinline__ const P *uniform_base(const P *ptr) {
  const uint64_t v = reinterpret_cast<uint64_t>(ptr);
  return reinterpret_cast<const P *>(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32) |
                                     (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v));
}

// What a copy instruction brings of a stage: 128 bytes of each of eight rows (first .. first + 7; rows past `last` repeat
// it, and what is made of them is never stored).  One scalar base for the eight rows, a 32-bit offset per lane (WIDE, for rows further
// apart than that reaches: 64-bit, and the address in vector registers).
template <bool WIDE>
struct CopySource {
  const char *base;
  typename std::conditional<WIDE, int64_t, uint32_t>::type off;
};
template <typename T, bool WIDE>
__device__ __forceinline__ CopySource<WIDE> copy_source(const void *rows, int64_t ld, int first, int last, int stage0) {
  const int lane = threadIdx.x & 63, r = lane >> 3, q = (lane & 7) ^ r;  // run q of row r goes to this lane's place
  const int b = min(first, last);
  CopySource<WIDE> s;
  s.base = uniform_base(reinterpret_cast<const char *>(static_cast<const T *>(rows) + b * ld + (int64_t)stage0 * kLinStageK));
  const int rows_on = min(first + r, last) - b;
  if constexpr (WIDE)
    s.off = (int64_t)rows_on * ld * 2 + q * 16;
  else
    s.off = (uint32_t)rows_on * (uint32_t)(ld * 2) + q * 16;
  return s;
}

// 64 lanes x 16 bytes of stage st, global -> LDS: lane l's bytes go to lds + 16 l.  ONCE: with the read-once hint.
template <bool ONCE, bool WIDE>
__device__ __forceinline__ void copy_1k(uint32_t lds, const CopySource<WIDE> &s, int st) {
  const char *base = s.base + (int64_t)st * (kLinStageK * 2);
  if constexpr (WIDE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(base + s.off) : "memory", "m0");
  else if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(s.off), "s"(base) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(s.off), "s"(base) : "memory", "m0");
}

__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)p);
}

// A stage's rows lie 128 bytes apart; run q (16 bytes) of row r is kept at place q ^ (r & 7).
__device__ __forceinline__ const uint4 *staged_run(const char *rows, int r, int q) {
  return reinterpret_cast<const uint4 *>(rows + r * (kLinStageK * 2) + ((q ^ (r & 7)) * 16));
}

// The sums of a tile's ranges, first to last.
__device__ __forceinline__ f32x4_t add_ranges(const f32x4_t *src, int splits) {
  f32x4_t total = src[0];
  for (int i = 1; i < splits; i++) {
    const f32x4_t v = src[i * 64];
#pragma unroll
    for (int r = 0; r < 4; r++) total[r] += v[r];
  }
  return total;
}

// Up to 16 rows of x.  WAVES wavefronts; each owns 16 rows of W.  GATED: odd wavefronts take the up rows that
// belong to the gate rows of the wavefront before them.  QKV: rotation and cache writes behind it.
template <typename T, int S, int WAVES, bool GATED, bool QKV = false>
__global__ __launch_bounds__(WAVES * 64) void linear_stream_kernel(const LinearParams p) {
  using vec8 = typename Vec8<T>::type;
  constexpr int kParts = GATED ? 2 : 1;
  constexpr int kCopiesW = 2, kCopiesX = 2, kCopies = kCopiesW + kCopiesX;  // of 1 KB: eight rows each
  constexpr int kStageBytes = kCopies * 1024;
  __shared__ __align__(1024) char ring[WAVES * S * kStageBytes];
  __shared__ f32x4_t sums[kParts * kLinMaxRanges * 64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kg = lane >> 4;
  // wavefronts per tile of 16 rows, and the ranges of k each of them takes, one after the other
  const int per_tile = min(p.splits, WAVES / kParts);
  const int ranges = p.splits / per_tile;
  const int part = GATED ? wave & 1 : 0;
  const int tile = (wave / kParts) / per_tile, first_range = ((wave / kParts) % per_tile) * ranges;
  const int tiles = WAVES / kParts / per_tile;
  const int n_tile = (blockIdx.x * tiles + tile) * 16;
  const int n_end = GATED ? p.half : p.N;
  const int stage0 = first_range * p.stages_per_split;
  const int nst = max(0, min(ranges * p.stages_per_split, p.total_stages - stage0));

  QkvRows rows = {};
  QkvToken token = {};
  if constexpr (QKV) {
    rows = qkv_rows(p.qkv, blockIdx.x * tiles + tile);
    token = qkv_token(p.qkv, min(col, p.M - 1));
  }
  CopySource<false> wsrc[kCopiesW], xsrc[kCopiesX];
#pragma unroll
  for (int i = 0; i < kCopiesW; i++)
    wsrc[i] = copy_source<T, false>(p.w, p.ldw, QKV ? (i ? rows.second : rows.first) : part * p.half + n_tile + i * 8,
                                    part * p.half + n_end - 1, stage0);
#pragma unroll
  for (int i = 0; i < kCopiesX; i++) xsrc[i] = copy_source<T, false>(p.x, p.ldx, i * 8, p.M - 1, stage0);
  const char *mine = ring + wave * S * kStageBytes;
  const uint32_t mine_lds = lds_address(ring) + wave * S * kStageBytes;
  StageOrder order(p, n_tile, nst);
  auto ask = [&](int slot) {
    const int st = order.next();
    const uint32_t at = mine_lds + slot * kStageBytes;
#pragma unroll
    for (int i = 0; i < kCopiesX; i++) copy_1k<false, false>(at + (kCopiesW + i) * 1024, xsrc[i], st);
#pragma unroll
    for (int i = 0; i < kCopiesW; i++) copy_1k<true, false>(at + i * 1024, wsrc[i], st);
  };
  f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const bool meet = !QKV || p.splits > 1;
  f32x4_t *range_sums = sums + ((tile * kParts + part) * p.splits + first_range) * 64 + lane;
  int left = p.stages_per_split, range = 0;  // of the range in hand

#pragma unroll
  for (int j = 0; j < S; j++)
    if (j < nst) ask(j);
  for (int base = 0; base < nst; base += S) {
#pragma unroll
    for (int j = 0; j < S; j++) {
      const int st = base + j;
      if (st < nst) {
        // S stages are on their way, this one first; near the end fewer, and the wait is for all of them
        if (st + S - 1 < nst)
          wait_copies<(S - 1) * kCopies>();
        else
          wait_copies<0>();
        const char *stage = mine + j * kStageBytes;
        uint4 wf[2], xf[2];
#pragma unroll
        for (int s = 0; s < 2; s++) {
          wf[s] = *staged_run(stage, col, 4 * s + kg);
          xf[s] = *staged_run(stage + kCopiesW * 1024, col, 4 * s + kg);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage is in registers: its place can be filled again
        if (st + S < nst) ask(j);
#pragma unroll
        for (int s = 0; s < 2; s++) acc = LinMfma<T>::run(bit_cast<vec8>(wf[s]), bit_cast<vec8>(xf[s]), acc);
        if (ranges > 1 && --left == 0) {
          range_sums[range++ * 64] = acc;
          acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
          left = p.stages_per_split;
        }
      }
    }
  }
  QkvTurn<T> turn = {};
  // (a wavefront that finishes a tile finishes the workgroup's `wave`th, whichever it worked on)
  if constexpr (QKV) {
    if (meet) rows = qkv_rows(p.qkv, blockIdx.x * tiles + wave);
    if (!meet || wave < tiles) turn = qkv_turn<T>(p.qkv, rows, token, kg);
    if (!meet) {
      linear_finish_qkv<T>(p, acc, col, kg, rows, token, turn);
      return;
    }
  }
  for (; range < ranges; range++) {  // what is left of the last range; ranges past the end of k are zero
    range_sums[range * 64] = acc;
    acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  __syncthreads();
  if (wave < tiles) {
    const int n = (blockIdx.x * tiles + wave) * 16 + 4 * kg;
    f32x4_t total[kParts];
#pragma unroll
    for (int q = 0; q < kParts; q++) total[q] = add_ranges(sums + (wave * kParts + q) * p.splits * 64 + lane, p.splits);
    if constexpr (GATED)
      linear_finish_gated<T>(p, total[0], total[1], col, n);
    else if constexpr (QKV)
      linear_finish_qkv<T>(p, total[0], col, kg, rows, token, turn);
    else
      linear_finish<T>(p, total[0], col, n);
  }
}

// RMS norm of up to ROWS rows of x and the layer behind it.  The rows are held in LDS whole and normalised there, with the arithmetic
// and the order of additions of rms_norm_vec8_kernel, so with its bits, while the first stages of W are on their way: a launch of
// rms_norm less, whose time is all latency.  The rows' part repeats in every workgroup and costs about 1 us per row, so it ends at few
// rows.  LDS: ring | sums of ranges | rows of x | the norm's weight.
__host__ __device__ constexpr int held_pitch(int K) { return (K * 2 + 1023) / 1024 * 1024; }
template <typename T, int S, int ROWS, int WAVES, bool GATED, bool QKV>
__global__ __launch_bounds__(WAVES * 64) void norm_linear_kernel(const LinearParams p) {
  using vec8 = typename Vec8<T>::type;
  constexpr int kParts = GATED ? 2 : 1;
  constexpr int kStageBytes = 2048;
  extern __shared__ __align__(1024) char lds[];
  __shared__ float part_sums[ROWS * 16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kg = lane >> 4;
  const int per_tile = min(p.splits, WAVES / kParts), ranges = p.splits / per_tile;
  const int part = GATED ? wave & 1 : 0;
  const int tile = (wave / kParts) / per_tile, first_range = ((wave / kParts) % per_tile) * ranges;
  const int tiles = WAVES / kParts / per_tile;
  const int n_tile = (blockIdx.x * tiles + tile) * 16;
  const int n_end = GATED ? p.half : p.N;
  const int stage0 = first_range * p.stages_per_split;
  const int nst = max(0, min(ranges * p.stages_per_split, p.total_stages - stage0));
  f32x4_t *sums = reinterpret_cast<f32x4_t *>(lds + WAVES * S * kStageBytes);
  const int pitch = held_pitch(p.K);
  char *xrows = lds + WAVES * S * kStageBytes + tiles * kParts * p.splits * 1024;
  char *normw = xrows + p.M * pitch;

  // rows of x (and the norm's weight behind them), 1 KB a piece: run q of row r goes to place q ^ (r & 7) of its row
  {
    const int per_row = pitch / 1024, pieces = (p.M + 1) * per_row, last = p.K / 8 - 1;
    const uint32_t at = lds_address(xrows);
    for (int i = wave; i < pieces; i += WAVES) {
      const int r = i / per_row, q0 = (i % per_row) * 64;
      CopySource<false> src;
      src.base = uniform_base(static_cast<const char *>(r == p.M ? p.norm_w : static_cast<const T *>(p.x) + r * p.ldx));
      src.off = (uint32_t)min(q0 + (lane ^ (r == p.M ? 0 : r & 7)), last) * 16;
      copy_1k<false, false>(at + i * 1024, src, 0);
    }
  }
  QkvRows rows = {};
  QkvToken token = {};
  if constexpr (QKV) {
    rows = qkv_rows(p.qkv, blockIdx.x * tiles + tile);
    token = qkv_token(p.qkv, min(col, p.M - 1));
  }
  CopySource<false> wsrc[2];
#pragma unroll
  for (int i = 0; i < 2; i++)
    wsrc[i] = copy_source<T, false>(p.w, p.ldw, QKV ? (i ? rows.second : rows.first) : part * p.half + n_tile + i * 8,
                                    part * p.half + n_end - 1, stage0);
  const char *mine = lds + wave * S * kStageBytes;
  const uint32_t mine_lds = lds_address(lds) + wave * S * kStageBytes;
  StageOrder order(p, n_tile, nst);
  auto ask = [&](int slot) {
    const int st = order.next();
#pragma unroll
    for (int i = 0; i < 2; i++) copy_1k<true, false>(mine_lds + slot * kStageBytes + i * 1024, wsrc[i], st);
  };
#pragma unroll
  for (int j = 0; j < S; j++)
    if (j < nst) ask(j);
  if (nst >= S)
    wait_copies<2 * S>();
  else
    wait_copies<0>();
  asm volatile("s_barrier" ::: "memory");
  {
    // rms_norm_vec8_kernel's thread t owns run t of a row: a wavefront here takes the place of one of its wavefronts at a time
    const int runs = p.K / 8, waves = (runs + 63) / 64;
    auto at = [&](int r, int q) { return reinterpret_cast<uint4 *>(xrows + r * pitch + (q ^ (r & 7)) * 16); };
    for (int w = wave; w < waves; w += WAVES) {
      const int q = w * 64 + lane;
      uint4 raw[ROWS];
      float ss[ROWS] = {};
#pragma unroll
      for (int r = 0; r < ROWS; r++) raw[r] = *at(min(r, p.M - 1), min(q, runs - 1));
#pragma unroll
      for (int r = 0; r < ROWS; r++) {
        const T *e = reinterpret_cast<const T *>(&raw[r]);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = to_float(e[j]);
#pragma unroll
        for (int j = 0; j < 8; j++) ss[r] += v[j] * v[j];
        ss[r] = wave_sum(q < runs ? ss[r] : 0.f);
        if (lane == 0) part_sums[r * 16 + w] = ss[r];
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    float inv[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; r++) inv[r] = rsqrtf(wave_sum(lane < waves ? part_sums[r * 16 + (lane & 15)] : 0.f) / (float)p.K + p.eps);
    for (int w = wave; w < waves; w += WAVES) {
      const int q = min(w * 64 + lane, runs - 1);
      uint4 raw[ROWS];
      const uint4 wr = *reinterpret_cast<const uint4 *>(normw + q * 16);
      const T *we = reinterpret_cast<const T *>(&wr);
#pragma unroll
      for (int r = 0; r < ROWS; r++) raw[r] = *at(min(r, p.M - 1), q);
#pragma unroll
      for (int r = 0; r < ROWS; r++) {
        const T *e = reinterpret_cast<const T *>(&raw[r]);
        uint4 o;
        T *oe = reinterpret_cast<T *>(&o);
#pragma unroll
        for (int j = 0; j < 8; j++) oe[j] = from_float<T>(to_float(from_float<T>(to_float(e[j]) * inv[r])) * to_float(we[j]));
        if (r < p.M && w * 64 + lane < runs) *at(r, q) = o;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
  const int xr = min(col, p.M - 1);
  const char *xrow = xrows + xr * pitch + stage0 * (kLinStageK * 2);
  StageOrder held(p, n_tile, nst);  // the stages as they come out of the ring
  f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
  f32x4_t *range_sums = sums + ((tile * kParts + part) * p.splits + first_range) * 64 + lane;
  int left = p.stages_per_split, range = 0;  // of the range in hand
  for (int base = 0; base < nst; base += S) {
#pragma unroll
    for (int j = 0; j < S; j++) {
      const int st = base + j;
      if (st < nst) {
        if (st + S - 1 < nst)
          wait_copies<(S - 1) * 2>();
        else
          wait_copies<0>();
        const char *stage = mine + j * kStageBytes;
        const char *xstage = xrow + held.next() * (kLinStageK * 2);
        uint4 wf[2], xf[2];
#pragma unroll
        for (int s = 0; s < 2; s++) {
          wf[s] = *staged_run(stage, col, 4 * s + kg);
          xf[s] = *reinterpret_cast<const uint4 *>(xstage + ((4 * s + kg) ^ (xr & 7)) * 16);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage is in registers: its place can be filled again
        if (st + S < nst) ask(j);
#pragma unroll
        for (int s = 0; s < 2; s++) acc = LinMfma<T>::run(bit_cast<vec8>(wf[s]), bit_cast<vec8>(xf[s]), acc);
        if (ranges > 1 && --left == 0) {
          range_sums[range++ * 64] = acc;
          acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
          left = p.stages_per_split;
        }
      }
    }
  }
  QkvTurn<T> turn = {};
  if constexpr (QKV) {
    if (p.splits > 1) rows = qkv_rows(p.qkv, blockIdx.x * tiles + wave);
    if (p.splits == 1 || wave < tiles) turn = qkv_turn<T>(p.qkv, rows, token, kg);
    if (p.splits == 1) {
      linear_finish_qkv<T>(p, acc, col, kg, rows, token, turn);
      return;
    }
  }
  if (!GATED && p.splits == 1) {
    linear_finish<T>(p, acc, col, n_tile + 4 * kg);
    return;
  }
  for (; range < ranges; range++) {  // what is left of the last range; ranges past the end of k are zero
    range_sums[range * 64] = acc;
    acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  __syncthreads();
  if (wave < tiles) {
    const int n = (blockIdx.x * tiles + wave) * 16 + 4 * kg;
    f32x4_t total[kParts];
#pragma unroll
    for (int q = 0; q < kParts; q++) total[q] = add_ranges(sums + (wave * kParts + q) * p.splits * 64 + lane, p.splits);
    if constexpr (GATED)
      linear_finish_gated<T>(p, total[0], total[1], col, n);
    else if constexpr (QKV)
      linear_finish_qkv<T>(p, total[0], col, kg, rows, token, turn);
    else
      linear_finish<T>(p, total[0], col, n);
  }
}

// Up to 16 MT rows of x: a workgroup owns 16 WAVES rows of W over one range of k.  GATED: the second half of the
// wavefronts takes the up rows that belong to the gate rows of the first.
template <typename T, int MT, int S, int WAVES, bool GATED, bool WIDE>
__global__ __launch_bounds__(WAVES * 64) void linear_tile_kernel(const LinearParams p) {
  using vec8 = typename Vec8<T>::type;
  // The read-once hint on W (stream kernel: always) measured 3 to 8 % faster here as well, except on the short ranges that the
  // 64-row workgroups serve with many rows of x (4096 x 4096, 128 rows: 15.6 us without, 17.0 with).
  constexpr bool kOnce = MT <= 2 || WAVES == 8;
  constexpr int kCopiesW = 2;                           // of 1 KB per stage: this wavefront's rows of W
  constexpr int kAllX = 2 * MT, kCopiesX = (kAllX + WAVES - 1) / WAVES;  // all copies of x, this wavefront's share
  constexpr int kCopies = kCopiesW + kCopiesX;
  constexpr int kStageBytes = (kCopiesW * WAVES + kAllX) * 1024;
  constexpr int kCols = WAVES * 16;
  constexpr int kPitch = kCols + 4;  // floats per row of finished sums in LDS
  static_assert(S * kStageBytes >= MT * 16 * kPitch * 4, "the sums reuse the ring");
  __shared__ __align__(1024) char ring[S * kStageBytes];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, kg = lane >> 4;
  const int part = GATED ? wave / (WAVES / 2) : 0;
  const int n_end = GATED ? p.half : p.N;
  const int n_group = blockIdx.x * (GATED ? kCols / 2 : kCols);
  const int n_tile = n_group + (GATED ? wave % (WAVES / 2) : wave) * 16;  // within the part
  const int split = blockIdx.y;
  const int stage0 = split * p.stages_per_split;
  const int nst = max(0, min(p.stages_per_split, p.total_stages - stage0));

  CopySource<WIDE> wsrc[kCopiesW], xsrc[kCopiesX];
#pragma unroll
  for (int i = 0; i < kCopiesW; i++)
    wsrc[i] = copy_source<T, WIDE>(p.w, p.ldw, part * p.half + n_tile + i * 8, part * p.half + n_end - 1, stage0);
  // Where the copies of x do not divide evenly some are made twice (the same bytes to the same place): every wavefront
  // counts the same number of copies per stage.
#pragma unroll
  for (int i = 0; i < kCopiesX; i++) xsrc[i] = copy_source<T, WIDE>(p.x, p.ldx, ((wave + i * WAVES) % kAllX) * 8, p.M - 1, stage0);
  const uint32_t ring_lds = lds_address(ring);
  StageOrder order(p, n_group, nst);
  auto ask = [&](int slot) {
    const int st = order.next();
    const uint32_t at = ring_lds + slot * kStageBytes;
#pragma unroll
    for (int i = 0; i < kCopiesX; i++)
      copy_1k<false, WIDE>(at + (kCopiesW * WAVES + (wave + i * WAVES) % kAllX) * 1024, xsrc[i], st);
#pragma unroll
    for (int i = 0; i < kCopiesW; i++) copy_1k<kOnce, WIDE>(at + (wave * kCopiesW + i) * 1024, wsrc[i], st);
  };
  f32x4_t acc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; mt++) acc[mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < S - 1; j++)
    if (j < nst) ask(j);
  for (int base = 0; base < nst; base += S) {
#pragma unroll
    for (int j = 0; j < S; j++) {
      const int st = base + j;
      if (st < nst) {
        // This wavefront's copies of the stage have landed, and behind the barrier everybody's; the barrier also says
        // that the stage before has been read, so its place takes the copies of the stage S - 1 further on.
        if (st + S - 2 < nst)
          wait_copies<(S - 2) * kCopies>();
        else
          wait_copies<0>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (st + S - 1 < nst) ask((j + S - 1) % S);
        const char *stage = ring + j * kStageBytes;
        const char *wrows = stage + wave * kCopiesW * 1024, *xrows = stage + kCopiesW * WAVES * 1024;
#pragma unroll
        for (int s = 0; s < 2; s++) {
          const uint4 wf = *staged_run(wrows, col, 4 * s + kg);
          uint4 xf[MT];
#pragma unroll
          for (int mt = 0; mt < MT; mt++) xf[mt] = *staged_run(xrows, mt * 16 + col, 4 * s + kg);
#pragma unroll
          for (int mt = 0; mt < MT; mt++) acc[mt] = LinMfma<T>::run(bit_cast<vec8>(wf), bit_cast<vec8>(xf[mt]), acc[mt]);
        }
      }
    }
  }

  if (p.row_sums) {
    // rows of fp32 sums, one 16-byte piece per lane and tile (four lanes make 64 contiguous bytes of a row)
    const int n = n_tile + 4 * kg;
    if (n < p.N) {
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
        if (mt < p.mtiles)
          *reinterpret_cast<f32x4_t *>(p.partial + ((int64_t)split * kLinMaxRows + mt * 16 + col) * p.N + n) = acc[mt];
    }
  } else if (p.tile_sums) {
    if (n_tile < n_end) {
      const int nt = (part * p.half + n_tile) / 16;
      f32x4_t *dst = reinterpret_cast<f32x4_t *>(p.partial) + ((int64_t)(split * (p.N / 16) + nt) * kLinMT) * 64 + lane;
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
        if (mt < p.mtiles) dst[mt * 64] = acc[mt];
    }
  } else {
    // Turned through LDS so that the stores are whole stretches of a row (kCols outputs): straight from the accumulators
    // they are 32 bytes per row and instruction, which cost 25 of 240 us on a 128256 x 4096 weight with 128 rows.
    float *tile = reinterpret_cast<float *>(ring);
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
      *reinterpret_cast<f32x4_t *>(tile + (mt * 16 + col) * kPitch + wave * 16 + 4 * kg) = acc[mt];
    __syncthreads();
    constexpr int kQuads = (GATED ? kCols / 2 : kCols) / 4;
    for (int i = tid; i < p.M * kQuads; i += WAVES * 64) {
      const int m = i / kQuads, c = (i % kQuads) * 4;
      const f32x4_t v = *reinterpret_cast<const f32x4_t *>(tile + m * kPitch + c);
      if constexpr (GATED)
        linear_finish_gated<T>(p, v, *reinterpret_cast<const f32x4_t *>(tile + m * kPitch + kCols / 2 + c), m, n_group + c);
      else
        linear_finish<T>(p, v, m, n_group + c);
    }
  }
}

// Adds up the ranges' sums, the first range first, and finishes the tile: one thread per (16 rows of W, row tile, lane).
// QKV: a lane's sums are those of the rows that linear_finish_qkv wants there, from two tiles.
template <typename T, bool GATED, bool QKV>
__global__ __launch_bounds__(256) void linear_reduce_kernel(const LinearParams p) {
  const int ntiles = p.N / 16;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int lane = (int)(idx & 63);
  const int mt = (int)((idx >> 6) % p.mtiles);
  const int64_t nt = (idx >> 6) / p.mtiles;
  if (nt >= (GATED ? p.half / 16 : ntiles)) return;
  const int64_t stride = (int64_t)ntiles * kLinMT * 64;
  auto add_up = [&](int64_t tile, int from) {
    const f32x4_t *src = reinterpret_cast<const f32x4_t *>(p.partial) + (tile * kLinMT + mt) * 64 + from;
    f32x4_t s = src[0];
    for (int i = 1; i < p.splits; i++) {
      const f32x4_t v = src[i * stride];
#pragma unroll
      for (int r = 0; r < 4; r++) s[r] += v[r];
    }
    return s;
  };
  const int m = mt * 16 + (lane & 15), n = (int)nt * 16 + 4 * (lane >> 4);
  if constexpr (QKV) {
    const int kg = lane >> 4;
    const QkvRows rows = qkv_rows(p.qkv, (int)nt);
    const QkvToken token = qkv_token(p.qkv, min(m, p.M - 1));
    const int at = (kg < 2 ? rows.first : rows.second) + 4 * (kg & 1);
    const f32x4_t sum = add_up(at / 16, (lane & 15) + (at & 15) / 4 * 16);
    linear_finish_qkv<T>(p, sum, m, kg, rows, token, qkv_turn<T>(p.qkv, rows, token, kg));
  } else if constexpr (GATED)
    linear_finish_gated<T>(p, add_up(nt, lane), add_up(nt + p.half / 16, lane), m, n);
  else
    linear_finish<T>(p, add_up(nt, lane), m, n);
}

// Adds up the ranges' sums of one row of y, finishes the row (bias, rounding, residual: as linear_finish) and
// applies the RMS norm that follows the layer (llama.rs:165, 169, 207 behind 166, 173) in the same launch: one
// workgroup per row, a thread's eight columns stay in registers between the two.  The norm's arithmetic and the
// order of its additions are those of the stand-alone kernel (rms_norm_vec8_kernel: the same thread owns the same
// eight columns, the same block_sum), so the two routes give the same bits.
template <typename T>
__global__ __launch_bounds__(1024) void linear_reduce_norm_kernel(const LinearParams p) {
  __shared__ float smem[17];
  const int row = blockIdx.x;
  const int i = threadIdx.x * 8;
  const bool active = i < p.N;
  float v[8];
  float ss = 0.f;
  if (active) {
    const float *src = p.partial + (int64_t)row * p.N + i;
    const int64_t stride = (int64_t)kLinMaxRows * p.N;
    f32x4_t a = *reinterpret_cast<const f32x4_t *>(src), b = *reinterpret_cast<const f32x4_t *>(src + 4);
    for (int k = 1; k < p.splits; k++) {
      const f32x4_t a2 = *reinterpret_cast<const f32x4_t *>(src + k * stride);
      const f32x4_t b2 = *reinterpret_cast<const f32x4_t *>(src + k * stride + 4);
#pragma unroll
      for (int r = 0; r < 4; r++) {
        a[r] += a2[r];
        b[r] += b2[r];
      }
    }
    const T *bias = static_cast<const T *>(p.bias);
    const T *res = static_cast<const T *>(p.residual);
    uint4 braw = make_uint4(0, 0, 0, 0), rraw = braw, oraw;
    if (bias != nullptr) braw = *reinterpret_cast<const uint4 *>(bias + i);
    if (res != nullptr) rraw = *reinterpret_cast<const uint4 *>(res + (int64_t)row * p.ldr + i);
    const T *be = reinterpret_cast<const T *>(&braw);
    const T *re = reinterpret_cast<const T *>(&rraw);
    T *oe = reinterpret_cast<T *>(&oraw);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      float f = j < 4 ? a[j] : b[j - 4];
      if (bias != nullptr) f += to_float(be[j]);
      T y = from_float<T>(f);
      if (res != nullptr) y = add_t<T>(y, re[j]);
      oe[j] = y;
      v[j] = to_float(y);
    }
    *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + (int64_t)row * p.ldo + i) = oraw;
#pragma unroll
    for (int j = 0; j < 8; j++) ss += v[j] * v[j];
  }
  const float total = block_sum(ss, smem);
  const float inv = rsqrtf(total / (float)p.N + p.eps);
  if (active) {
    const uint4 wr = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.norm_w) + i);
    const T *we = reinterpret_cast<const T *>(&wr);
    uint4 o;
    T *oe = reinterpret_cast<T *>(&o);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const T normed = from_float<T>(v[j] * inv);
      oe[j] = from_float<T>(to_float(normed) * to_float(we[j]));
    }
    *reinterpret_cast<uint4 *>(static_cast<T *>(p.norm_out) + (int64_t)row * p.ldn + i) = o;
  }
}

struct LinearPlan {
  bool stream;  // the few-rows kernel
  int waves;    // tile kernel: wavefronts per workgroup
  int splits;   // ranges of k
  int stages_per_split;
  bool turned;  // ranges begin inside (StageOrder)
  size_t partial_bytes;  // fp32 sums of every range, [range][128 rows][N]; not used by the few-rows kernel
};

// Weights that are not cut and whose workgroups of 64 rows are more than one to a compute unit, but not two, while those of 128 rows are at most
// one: then every unit with work has the same.  us, 64 / 128 rows, 16 rows of x: 16384 x 4096 21.7 / 28.9; 18432 x 4096 33.7 / 29.2; 22016 x 4096
// gated 34.6 / 30.8; 28672 x 4096 gated 36.5 / 36.1, 32 rows 38.4 / 36.7; 32000 x 4096 40.4 / 40.5; 37888 x 3584 gated 46.4 / 56.0; 51200 x 2560
// 48.3 / 47.6.  With the norm in front, whose work on the
// rows of x repeats in every workgroup, 1 row: 28672 x 4096 gated 38.3 / 37.5, 22016 x 4096 33.6 / 30.7, 20480 x 2560 23.3 / 22.1; its ring of four
// stages for six: 37.5 / 38.8.
bool wide_workgroups(int N) { return N > 64 * 256 && N <= 128 * 256; }

// The ranges of k depend on the weight alone (see above).  As far as eight ranges allow: 1024 wavefronts' worth of (16 rows, range)
// pairs, four per compute unit, and no range longer than 2048 once k is cut at all -- 4096 x 4096 and 6144 x 4096 four, 4096 x
// 14336 eight, weights of 16384 rows and more none.
LinearPlan plan_linear(int M, int N, int K, bool few_only) {
  const Tuning &tn = tuning();
  LinearPlan pl;
  const int stages = K / kLinStageK;
  int splits = 1;
  while (splits < kLinMaxRanges && (int64_t)N * splits < 16384) splits *= 2;
  while (splits > 1 && splits < kLinMaxRanges && K / splits > 2048) splits *= 2;
  while (splits > stages) splits /= 2;
  // Where k is not cut, a workgroup's one copy of x: 28672 x 4096 gated, us, stream / tile kernel 1 row 38.4 / 36.4, 16 41.7 / 36.8; 51200 x 2560
  // 45.4 / 44.9, 52.7 / 48.3; 128256 x 4096 154.8 / 151.5, 156.2 / 153.4.  With ranges the tile kernel needs its second launch: 12288 x
  // 4096 19.3 / 21.1, 22.5 / 20.6.
  pl.stream = M <= kLinStreamRows && (few_only || splits > 1);
  if (tn.linear_splits > 0 && !few_only) splits = tn.linear_splits < stages ? tn.linear_splits : stages;
  if ((tn.linear_splits > 0 || tn.linear_waves > 0 || tn.linear_tiles > 0) && !few_only) pl.stream = false;
  pl.splits = splits;
  pl.stages_per_split = (stages + splits - 1) / splits;
  // Turned ranges, us (21 stages further per 128 rows of W: odd, so that consecutive places differ and all are used): 28672 x 4096
  // gated 1 / 32 / 128 rows 40.8 -> 38.0 (here 36.5 in the tile kernel), 42.9 -> 38.5, 53.9 -> 50.3, with the norm in front 42.5 -> 38.5;
  // 128256 x 4096 1 / 32 / 128 rows 162 -> 154, 189 -> 161, 250 -> 219; 16384 x 2048, 6144, 8192, 11008, 14336 15.0 -> 12.8, 40.4 ->
  // 32.1, 58.5 -> 39.3, 63.8 -> 54.7, 86.9 -> 68.7; in ranges 12288 x 4096 (2) 22.2 -> 19.4, 8192 x 8192 (4) 27.8 -> 21.9.  Nothing to gain where
  // rows are not so far apart or not by such powers of two (16384 x 1024, 3072, 5120, 20480 x 2560: +-1 %), where shorter ranges already
  // spread the wavefronts (4096 x 4096, 6144 x 4096, 4096 x 14336: +-1 %, with 128 rows 6144 x 4096 21.0 -> 21.6; 8192 x 28672, eight ranges,
  // 106 -> 108).
  pl.turned = N >= 8192 && N % (2 * kTurnRows) == 0 && splits <= 4 && (K % 2048 == 0 || K >= 6144);
  // Workgroups of 64 rows while the device holds all of them at once, one per compute unit, or where 32 rows of x leave the copies of x
  // cheap (37888 x 3584, 32 rows: 49.8 us against 60.2; 28672 x 4096, 64 rows: 49.2 against 40.0) and 128 rows are not one per unit; else of
  // 128 rows.
  pl.waves = ((int64_t)((N + 63) / 64) * splits <= 256 || (splits == 1 && M <= 32 && !wide_workgroups(N))) ? 4 : 8;
  if (tn.linear_tiles > 0) pl.waves = 4 * tn.linear_tiles;
  if (tn.linear_waves > 0) pl.waves = tn.linear_waves;
  pl.partial_bytes = (size_t)pl.splits * kLinMaxRows * N * sizeof(float);
  return pl;
}

// Stages of the ring: what fits half of the 160 KB of LDS (two workgroups per compute unit), or four where a stage takes more than 24 KB
// (us, five / four, 96 and 128 rows: 6144 x 4096 19.8 / 19.5, 20.9 / 20.2; 4096 x 14336 31.7 / 31.3, 34.0 / 33.6; 128256 x 4096 207.2 / 206.0,
// 217.8 / 217.1; three: 4096 x 4096 17.4 / 18.1).
template <int MT, int WAVES>
constexpr int ring_stages() {
  constexpr int kb = 2 * WAVES + 2 * MT;
  constexpr int s = kb <= 24 ? 80 / kb : 4;
  return s > 6 ? 6 : s;
}

// WIDE: MT and the workgroup are those of the largest call, which every smaller one fits.
template <typename T, int MT, bool GATED, bool WIDE = false>
void launch_tile(const LinearParams &p, const LinearPlan &pl, hipStream_t stream) {
  const int waves = WIDE ? 8 : pl.waves;
  const int n = GATED ? p.half : p.N, per_wg = waves * 16 / (GATED ? 2 : 1);
  const dim3 grid((n + per_wg - 1) / per_wg, pl.splits), block(waves * 64);
  if constexpr (!WIDE) {
    if (waves == 4) {
      hipLaunchKernelGGL((linear_tile_kernel<T, MT, ring_stages<MT, 4>(), 4, GATED, false>), grid, block, 0, stream, p);
      return;
    }
  }
  if constexpr (MT == 4 && !WIDE) {
    // one workgroup to a compute unit: five stages for three (28672 x 4096 gated, us, 33 / 64 rows of x 40.5 / 39.8 -> 39.1 / 38.8; 128256 x 4096, 64
    // rows 177 -> 182)
    if (p.splits == 1 && wide_workgroups(p.N)) {
      hipLaunchKernelGGL((linear_tile_kernel<T, MT, 5, 8, GATED, false>), grid, block, 0, stream, p);
      return;
    }
  }
  hipLaunchKernelGGL((linear_tile_kernel<T, MT, ring_stages<MT, 8>(), 8, GATED, WIDE>), grid, block, 0, stream, p);
}

template <typename T, int ROWS, int WAVES, bool GATED, bool QKV>
void launch_norm_linear_waves(const LinearParams &p, hipStream_t stream) {
  constexpr int S = kHeldStages;
  static bool attr_set = false;  // benign race: setting twice is harmless
  auto kernel = norm_linear_kernel<T, S, ROWS, WAVES, GATED, QKV>;
  if (!attr_set) {
    HA_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                               WAVES * S * 2048 + 16 * 1024 + kLinHeldBytes));
    attr_set = true;
  }
  const int parts = GATED ? 2 : 1, n = GATED ? p.half : p.N;
  const int per_tile = p.splits < WAVES / parts ? p.splits : WAVES / parts, tiles = WAVES / parts / per_tile;
  const int rows = 16 * tiles;
  const size_t bytes = WAVES * S * 2048 + tiles * parts * p.splits * 1024 + (size_t)(p.M + 1) * held_pitch(p.K);
  hipLaunchKernelGGL(kernel, dim3((n + rows - 1) / rows), dim3(WAVES * 64), bytes, stream, p);
  check_launch("rms_norm_linear");
}

template <typename T, int ROWS, bool GATED, bool QKV>
void launch_norm_linear(const LinearParams &p, hipStream_t stream) {
  if (p.splits == 1 && wide_workgroups(p.N))
    launch_norm_linear_waves<T, ROWS, 8, GATED, QKV>(p, stream);
  else
    launch_norm_linear_waves<T, ROWS, 4, GATED, QKV>(p, stream);
}

template <typename T, bool GATED, bool QKV = false>
void launch_linear(const LinearParams &p, const LinearPlan &pl, hipStream_t stream) {
  if (p.norm_in) {
    if (p.M == 1)
      launch_norm_linear<T, 1, GATED, QKV>(p, stream);
    else if (p.M == 2)
      launch_norm_linear<T, 2, GATED, QKV>(p, stream);
    else
      launch_norm_linear<T, kLinHeldRows, GATED, QKV>(p, stream);
    return;
  }
  if (pl.stream) {
    const int parts = GATED ? 2 : 1, n = GATED ? p.half : p.N;
    const int per_tile = p.splits < 4 / parts ? p.splits : 4 / parts;
    const int rows = 16 * (4 / parts / per_tile);
    hipLaunchKernelGGL((linear_stream_kernel<T, 3, 4, GATED, QKV>), dim3((n + rows - 1) / rows), dim3(256), 0, stream, p);
    check_launch("linear (few rows)");
    return;
  }
  if (p.wide)
    launch_tile<T, 8, GATED, true>(p, pl, stream);
  else if (p.M <= 16)
    launch_tile<T, 1, GATED>(p, pl, stream);
  else if (p.M <= 32)
    launch_tile<T, 2, GATED>(p, pl, stream);
  else if (p.M <= 64)
    launch_tile<T, 4, GATED>(p, pl, stream);
  else if (p.M <= 96)
    launch_tile<T, 6, GATED>(p, pl, stream);
  else
    launch_tile<T, 8, GATED>(p, pl, stream);
  check_launch("linear");
  if (p.row_sums) {
    int threads = (int)(((p.N / 8 + 63) / 64) * 64);
    if (threads > 1024) threads = 1024;  // (the entry point bounds N)
    hipLaunchKernelGGL((linear_reduce_norm_kernel<T>), dim3((unsigned)p.M), dim3((unsigned)threads), 0, stream, p);
    check_launch("linear (sum of the ranges + rms_norm)");
  } else if (p.tile_sums) {
    const int64_t threads = (int64_t)((GATED ? p.half : p.N) / 16) * p.mtiles * 64;
    hipLaunchKernelGGL((linear_reduce_kernel<T, GATED, QKV>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, p);
    check_launch("linear (sum of the ranges)");
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether rows of two 2-byte matrices may share memory.  Column ranges of one wider matrix lie between each other without.
bool rows_overlap(const hipattn_tensor *a, const hipattn_tensor *b) {
  struct Span {
    int64_t lo, hi;  // bytes, hi past the end
  };
  auto span = [](const hipattn_tensor *t) {
    const int64_t at = (int64_t)reinterpret_cast<uintptr_t>(t->data), reach = (t->sizes[0] - 1) * t->strides[0] * 2;
    return Span{at + (reach < 0 ? reach : 0), at + (reach > 0 ? reach : 0) + t->sizes[1] * 2};
  };
  const Span sa = span(a), sb = span(b);
  if (sa.hi <= sb.lo || sb.hi <= sa.lo) return false;
  const int64_t ld = a->strides[0] * 2, off = (int64_t)reinterpret_cast<uintptr_t>(b->data) - (int64_t)reinterpret_cast<uintptr_t>(a->data);
  if (ld <= 0 || a->strides[0] != b->strides[0]) return true;
  const int64_t within = ((off % ld) + ld) % ld;  // where b's columns start in a's rows
  return within < a->sizes[1] * 2 || within + b->sizes[1] * 2 > ld;
}

struct QkvOperands {
  const hipattn_tensor *positions, *cos_sin;
  hipattn_tensor *key_cache, *value_cache;
  const hipattn_tensor *slot_mapping;
};

QkvParams qkv_params(const QkvOperands &o, int64_t M, int64_t N, int dt) {
  const char *op = "qkv_linear";
  QkvParams q{};
  q.g = cache_geometry(o.key_cache, o.value_cache, op);
  check_index_tensor(o.positions, "positions", 1);
  check_index_tensor(o.slot_mapping, "slot_mapping", 1);
  check_tensor(o.cos_sin, "cos_sin_cache", 2);
  const int hd = q.g.head_size;
  HA_CHECK(o.key_cache->dtype == dt && o.cos_sin->dtype == dt, "%s: cos_sin_cache and the caches must be %s", op, dtype_name(dt));
  HA_CHECK(o.positions->sizes[0] == M && o.slot_mapping->sizes[0] == M, "%s: %lld positions and %lld slots for %lld rows", op,
           (long long)o.positions->sizes[0], (long long)o.slot_mapping->sizes[0], (long long)M);
  HA_CHECK(hd > 0 && hd % 16 == 0 && o.cos_sin->sizes[1] == hd, "%s: heads of %d, rotated over %lld; both must be the same multiple of 16", op, hd,
           (long long)o.cos_sin->sizes[1]);
  HA_CHECK(N % hd == 0 && N / hd > 2 * (int64_t)q.g.num_heads && q.g.num_heads > 0,
           "%s: %lld rows of weight are not query heads and %d key and value heads of %d", op, (long long)N, q.g.num_heads, hd);
  HA_CHECK(is_contiguous(o.cos_sin) && aligned16(o.cos_sin->data) && aligned16(o.key_cache->data) && q.g.k_block_stride % 8 == 0 &&
               q.g.k_head_stride % 8 == 0,
           "%s: rows of cos_sin_cache and of key_cache's heads must start on 16-byte boundaries", op);
  check_data(o.cos_sin, "cos_sin_cache");
  q.positions = o.positions->data;
  q.slots = o.slot_mapping->data;
  q.cos_sin = o.cos_sin->data;
  q.pos64 = o.positions->dtype == HIPATTN_I64;
  q.slot64 = o.slot_mapping->dtype == HIPATTN_I64;
  q.max_pos = o.cos_sin->sizes[0];
  q.q_heads = (int)(N / hd) - 2 * q.g.num_heads;
  q.key_cache = o.key_cache->data;
  q.value_cache = o.value_cache->data;
  return q;
}

// With `norm_out` the RMS norm of the finished rows (weight `norm_weight`, `eps`) is written there by the launch
// that adds up the ranges' sums; the workspace is then needed whatever the number of ranges.
void linear_impl(hipattn_tensor *out, const hipattn_tensor *x, const hipattn_tensor *weight, const hipattn_tensor *bias,
                 const hipattn_tensor *residual, const hipattn_tensor *workspace, void *stream_arg, int64_t *ws_query,
                 hipattn_tensor *norm_out = nullptr, const hipattn_tensor *norm_weight = nullptr, float eps = 0.f,
                 bool ws_query_with_norm = false, bool gated = false, bool norm_in = false, const QkvOperands *qkv = nullptr) {
  check_tensor(x, "x", 2);
  check_tensor(weight, "weight", 2);
  const int dt = x->dtype;
  HA_CHECK(dt == HIPATTN_F16 || dt == HIPATTN_BF16, "linear: x must be f16 or bf16, got %s", dtype_name(dt));
  HA_CHECK(weight->dtype == dt, "linear: weight is %s, x is %s", dtype_name(weight->dtype), dtype_name(dt));
  const int64_t M = x->sizes[0], K = x->sizes[1], N = weight->sizes[0];
  HA_CHECK(weight->sizes[1] == K, "linear: weight has %lld columns, x has %lld", (long long)weight->sizes[1], (long long)K);
  HA_CHECK(M <= kLinMaxRows, "linear: %lld rows of x; this kernel takes at most %d (use a library GEMM beyond that)",
           (long long)M, kLinMaxRows);
  HA_CHECK(K > 0 && K % 256 == 0, "linear: the inner size %lld must be a positive multiple of %d", (long long)K, 256);
  HA_CHECK(N % 16 == 0, "linear: the number of rows of weight (%lld) must be a multiple of 16", (long long)N);
  HA_CHECK(N < (1 << 24) && K < (1 << 24), "linear: sizes out of range");
  HA_CHECK(!gated || N % 32 == 0, "linear_silu_and_mul: gate and up rows (%lld together) must be multiples of 16 each", (long long)N);
  LinearPlan pl = plan_linear((int)M, (int)N, (int)K, norm_in || qkv != nullptr);
  const int64_t outputs = gated ? N / 2 : N;
  const bool with_norm = norm_out != nullptr || ws_query_with_norm;
  // the norm's launch takes rows of sums, however few the ranges
  if (pl.splits == 1 && !with_norm) pl.partial_bytes = 0;
  if (ws_query != nullptr) {  // whatever the rows of x: a buffer sized with one serves a step of 128
    *ws_query = (int64_t)pl.partial_bytes;
    return;
  }
  check_tensor(out, "out", 2);
  HA_CHECK(out->dtype == dt, "linear: out is %s, x is %s", dtype_name(out->dtype), dtype_name(dt));
  HA_CHECK(out->sizes[0] == M && out->sizes[1] == outputs, "linear: out is [%lld, %lld], expected [%lld, %lld]",
           (long long)out->sizes[0], (long long)out->sizes[1], (long long)M, (long long)outputs);
  if (M == 0 || N == 0) return;
  check_data(x, "x");
  check_data(weight, "weight");
  check_data(out, "out");
  HA_CHECK(x->strides[1] == 1 && weight->strides[1] == 1 && out->strides[1] == 1,
           "linear: the last dimension of x, weight and out must be contiguous");
  HA_CHECK(x->strides[0] % 8 == 0 && weight->strides[0] % 8 == 0 && aligned16(x->data) && aligned16(weight->data),
           "linear: rows of x and weight must start on 16-byte boundaries");
  HA_CHECK(out->strides[0] % 4 == 0 && (reinterpret_cast<uintptr_t>(out->data) & 7) == 0,
           "linear: rows of out must start on 8-byte boundaries");

  // Output rows over rows of x: both kernels write while other workgroups still read x, so every row of sums goes to the workspace
  // and a second launch finishes it.
  const bool overlap = rows_overlap(x, out);
  if (norm_in) {
    HA_CHECK(M <= kLinHeldRows && K <= 8192 && N < 65536 && (M + 1) * held_pitch((int)K) <= kLinHeldBytes,
             "rms_norm_linear: %lld rows of %lld and a weight of %lld rows; it takes at most %d rows of up to 8192, %d bytes with the norm's weight, and fewer than 65536 rows of weight",
             (long long)M, (long long)K, (long long)N, kLinHeldRows, kLinHeldBytes);
    HA_CHECK(!overlap, "rms_norm_linear: out lies over x");
    check_tensor(norm_weight, "norm_weight", 1);
    HA_CHECK(norm_weight->dtype == dt && norm_weight->sizes[0] == K && norm_weight->strides[0] == 1,
             "rms_norm_linear: norm_weight must be %lld contiguous %s", (long long)K, dtype_name(dt));
    check_data(norm_weight, "norm_weight");
    HA_CHECK(aligned16(norm_weight->data), "rms_norm_linear: norm_weight must start on a 16-byte boundary");
  }
  if (overlap) {
    pl.stream = false;
    pl.partial_bytes = (size_t)pl.splits * kLinMaxRows * N * sizeof(float);
  }

  LinearParams p{};
  p.x = x->data;
  p.w = weight->data;
  p.out = out->data;
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  p.mtiles = (int)((M + 15) / 16);
  p.ldx = M == 1 ? 0 : x->strides[0];
  p.ldw = weight->strides[0];
  // seven rows on must be within 32 bits of bytes, else one instance of the tile kernel serves all sizes (the last position of every
  // sequence of a [sequences, 65536, 4096] activation lies 2^28 elements apart)
  auto far = [](int64_t ld) { return ld < 0 || ld >= (1 << 28); };
  p.wide = far(p.ldx) || far(p.ldw);
  if (p.wide) pl.stream = false;
  if (norm_in) {
    HA_CHECK(pl.stream, "rms_norm_linear: rows of x or weight lie too far apart");
    p.norm_in = 1;
    p.norm_w = norm_weight->data;
    p.eps = eps;
  }
  p.ldo = out->strides[0];
  if (bias != nullptr) {
    check_tensor(bias, "bias", 1);
    HA_CHECK(bias->dtype == dt && bias->sizes[0] == N && bias->strides[0] == 1, "linear: bias must be %lld contiguous %s",
             (long long)N, dtype_name(dt));
    check_data(bias, "bias");
    p.bias = bias->data;
  }
  if (residual != nullptr) {
    check_tensor(residual, "residual", 2);
    HA_CHECK(residual->dtype == dt && residual->sizes[0] == M && residual->sizes[1] == N && residual->strides[1] == 1,
             "linear: residual must be [%lld, %lld] %s with a contiguous last dimension", (long long)M, (long long)N,
             dtype_name(dt));
    HA_CHECK(residual->strides[0] % 4 == 0 && (reinterpret_cast<uintptr_t>(residual->data) & 7) == 0,
             "linear: rows of residual must start on 8-byte boundaries");
    check_data(residual, "residual");
    p.residual = residual->data;
    p.ldr = residual->strides[0];
  }
  if (with_norm) {
    HA_CHECK(N % 8 == 0 && N <= 8192, "linear_rms_norm: the number of rows of weight (%lld) must be a multiple of 8, at most 8192",
             (long long)N);
    check_tensor(norm_out, "norm_out", 2);
    HA_CHECK(norm_weight != nullptr, "linear_rms_norm: norm_weight is NULL");
    check_tensor(norm_weight, "norm_weight", 1);
    HA_CHECK(norm_out->dtype == dt && norm_out->sizes[0] == M && norm_out->sizes[1] == N && norm_out->strides[1] == 1,
             "linear_rms_norm: norm_out must be [%lld, %lld] %s with a contiguous last dimension", (long long)M, (long long)N,
             dtype_name(dt));
    HA_CHECK(norm_weight->dtype == dt && norm_weight->sizes[0] == N && norm_weight->strides[0] == 1,
             "linear_rms_norm: norm_weight must be %lld contiguous %s", (long long)N, dtype_name(dt));
    check_data(norm_out, "norm_out");
    check_data(norm_weight, "norm_weight");
    HA_CHECK(out->strides[0] % 8 == 0 && norm_out->strides[0] % 8 == 0 && aligned16(out->data) && aligned16(norm_out->data) &&
                 aligned16(norm_weight->data) && (bias == nullptr || aligned16(bias->data)) &&
                 (residual == nullptr || (residual->strides[0] % 8 == 0 && aligned16(residual->data))),
             "linear_rms_norm: rows of out, norm_out and residual, and bias and norm_weight, must start on 16-byte boundaries");
    // The launch of rms_norm behind the few-rows kernel takes rows that lie end to end; other rows (a slice of a wider matrix) go the
    // way of larger batches, with the same bits.
    if (!is_contiguous(out) || !is_contiguous(norm_out)) pl.stream = false;
    p.row_sums = pl.stream ? 0 : 1;
    p.norm_w = norm_weight->data;
    p.norm_out = norm_out->data;
    p.ldn = norm_out->strides[0];
    p.eps = eps;
  }
  p.tile_sums = !pl.stream && !p.row_sums && (pl.splits > 1 || overlap);
  p.splits = pl.splits;
  p.turned = pl.turned ? (int)(N / 2) : 0;
  p.stages_per_split = pl.stages_per_split;
  p.total_stages = (int)(K / kLinStageK);
  p.half = gated ? (int)(N / 2) : 0;
  hipStream_t stream = resolve_stream(stream_arg);
  HeldWorkspace held;  // over all launches
  if (pl.partial_bytes > 0 && !pl.stream) {  // (the few-rows kernel leaves finished rows: a launch of rms_norm normalises them)
    if (workspace != nullptr) {
      check_tensor(workspace, "workspace", 1);
      HA_CHECK(workspace->dtype == HIPATTN_U8 && workspace->strides[0] == 1, "linear: workspace must be contiguous u8");
      HA_CHECK((size_t)workspace->sizes[0] >= pl.partial_bytes, "linear: workspace has %lld bytes, %zu are needed",
               (long long)workspace->sizes[0], pl.partial_bytes);
      HA_CHECK(aligned16(workspace->data), "linear: workspace must start on a 16-byte boundary");
      check_data(workspace, "workspace");
      p.partial = static_cast<float *>(workspace->data);
    } else {
      held = library_workspace(WS_LINEAR, pl.partial_bytes, stream);
      p.partial = static_cast<float *>(held.ptr);
    }
  }
  if (qkv != nullptr) {
    HA_CHECK(N < 65536 && (pl.stream || p.tile_sums),
             "qkv_linear: %lld rows of x and a weight of %lld rows; fewer than 65536 of weight, and than 16384 with more than %d rows of x", (long long)M,
             (long long)N, kLinStreamRows);
    p.qkv = qkv_params(*qkv, M, N, dt);
    if (p.turned != 0 && kTurnRows % p.qkv.g.head_size != 0) {
      // A row and the one that it is rotated with would have to share an order of k, and here they may have different ones (heads of 80, 96,
      // 256, ...): the calls themselves, with their bits.  us, an order without turns in one launch / the calls: 9216 x 2048 16 rows 12.5 /
      // 16.4, 12288 x 4096 16 and 64 rows 25.0 / 27.3, 29.6 / 31.2, 15360 x 8192 64 rows 64.7 / 57.0, 21504 x 8192 16 rows 80.5 / 63.4.
      held = HeldWorkspace{};  // (the call below takes it for itself)
      linear_impl(out, x, weight, nullptr, nullptr, nullptr, stream_arg, nullptr, nullptr, norm_weight, eps, false, false, norm_in);
      const int hd = p.qkv.g.head_size, Hkv = p.qkv.g.num_heads;
      auto columns = [&](int64_t first, int64_t heads) {
        hipattn_tensor t = *out;
        t.data = static_cast<char *>(out->data) + first * hd * 2;
        t.sizes[1] = heads * hd;
        return t;
      };
      hipattn_tensor q = columns(0, p.qkv.q_heads), k = columns(p.qkv.q_heads, Hkv), v = columns(p.qkv.q_heads + Hkv, Hkv);
      v.ndim = 3;
      v.sizes[1] = Hkv;
      v.sizes[2] = hd;
      v.strides[1] = hd;
      v.strides[2] = 1;
      raise(hipattn_rotary_embedding_and_cache(qkv->positions, &q, &k, &v, hd, qkv->cos_sin, true, qkv->key_cache, qkv->value_cache,
                                               qkv->slot_mapping, stream_arg));
      return;
    }
    dt == HIPATTN_BF16 ? launch_linear<bf16_t, false, true>(p, pl, stream) : launch_linear<half_t, false, true>(p, pl, stream);
    return;
  }
  if (dt == HIPATTN_BF16)
    gated ? launch_linear<bf16_t, true>(p, pl, stream) : launch_linear<bf16_t, false>(p, pl, stream);
  else
    gated ? launch_linear<half_t, true>(p, pl, stream) : launch_linear<half_t, false>(p, pl, stream);
  if (norm_out != nullptr && pl.stream) raise(hipattn_rms_norm(norm_out, out, norm_weight, eps, stream_arg));
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" char *hipattn_linear(hipattn_tensor *out, const hipattn_tensor *x, const hipattn_tensor *weight,
                                const hipattn_tensor *bias, const hipattn_tensor *residual,
                                const hipattn_tensor *workspace, void *stream) {
  HA_PROTECT(linear_impl(out, x, weight, bias, residual, workspace, stream, nullptr));
}

extern "C" char *hipattn_linear_silu_and_mul(hipattn_tensor *out, const hipattn_tensor *x, const hipattn_tensor *weight,
                                             const hipattn_tensor *workspace, void *stream) {
  HA_PROTECT(linear_impl(out, x, weight, nullptr, nullptr, workspace, stream, nullptr, nullptr, nullptr, 0.f, false, true));
}

extern "C" char *hipattn_rms_norm_linear(hipattn_tensor *out, const hipattn_tensor *x, const hipattn_tensor *norm_weight,
                                         float epsilon, const hipattn_tensor *weight, bool silu_and_mul, void *stream) {
  HA_PROTECT(linear_impl(out, x, weight, nullptr, nullptr, nullptr, stream, nullptr, nullptr, norm_weight, epsilon, false, silu_and_mul,
                         true));
}

extern "C" char *hipattn_qkv_linear(hipattn_tensor *out, const hipattn_tensor *x, const hipattn_tensor *norm_weight, float epsilon,
                                    const hipattn_tensor *weight, const hipattn_tensor *positions,
                                    const hipattn_tensor *cos_sin_cache, hipattn_tensor *key_cache, hipattn_tensor *value_cache,
                                    const hipattn_tensor *slot_mapping, void *stream) {
  HA_PROTECT({
    const QkvOperands qkv{positions, cos_sin_cache, key_cache, value_cache, slot_mapping};
    linear_impl(out, x, weight, nullptr, nullptr, nullptr, stream, nullptr, nullptr, norm_weight, epsilon, false, false,
                norm_weight != nullptr, &qkv);
  });
}

extern "C" char *hipattn_linear_workspace_size(const hipattn_tensor *x, const hipattn_tensor *weight, int64_t *bytes) {
  HA_PROTECT({
    HA_CHECK(bytes != nullptr, "linear_workspace_size: bytes is NULL");
    linear_impl(nullptr, x, weight, nullptr, nullptr, nullptr, nullptr, bytes);
  });
}

extern "C" char *hipattn_linear_rms_norm(hipattn_tensor *out, hipattn_tensor *norm_out, const hipattn_tensor *x,
                                         const hipattn_tensor *weight, const hipattn_tensor *bias,
                                         const hipattn_tensor *residual, const hipattn_tensor *norm_weight, float epsilon,
                                         const hipattn_tensor *workspace, void *stream) {
  HA_PROTECT({
    HA_CHECK(norm_out != nullptr, "linear_rms_norm: norm_out is NULL");
    linear_impl(out, x, weight, bias, residual, workspace, stream, nullptr, norm_out, norm_weight, epsilon);
  });
}

extern "C" char *hipattn_linear_rms_norm_workspace_size(const hipattn_tensor *x, const hipattn_tensor *weight,
                                                        int64_t *bytes) {
  HA_PROTECT({
    HA_CHECK(bytes != nullptr, "linear_rms_norm_workspace_size: bytes is NULL");
    linear_impl(nullptr, x, weight, nullptr, nullptr, nullptr, nullptr, bytes, nullptr, nullptr, 0.f, true);
  });
}
