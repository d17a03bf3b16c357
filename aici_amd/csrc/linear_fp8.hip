// Linear layer on a weight of 8-bit floating point (e4m3) with a scale for each 128 x 128 of it: y = x . Wᵀ (+ bias) (+ residual), any number
// of rows of x.  No counterpart in the reference, whose weights are those of hipattn_linear.
//
//   e[m, b] = the least integer with max |x[m, block b]| <= 448 2^e (at least -126);  q[m, k] = x[m, k] 2^-e rounded to e4m3, ties to even
//   y[m, n] = T( sum over blocks b of 2^e[m, b] ws[n / 128, b] (sum over k in b of q[m, k] w[n, k])  + bias[n] ) (+ residual[m, n], rounded again)
//   (the product of the two scales comes first, in fp32: it has to be a finite number, and a normal one for the sums to keep all their bits)
//
// The scales of x are powers of two, so that scaling is exact and what is rounded is x itself; the largest of a block lands in (224, 448], and e4m3
// has the same relative steps there as below.  Sums of a block are the matrix pipe's, the sum over blocks is one fp32 FMA per block.
//
// The matrix pipe adds the products of 8-bit numbers eight at a time, each cut at 2^-13 of the largest one's power of two (measured; seen also
// across lanes: fp32 from there on).  Against a row of 4096 random products that is some 2^-13 of the sum, a tenth of the rounding to bf16 and about
// that to fp16; products of 16-bit operands would keep all of it, at half the rate and with every byte of W unpacked first.
//
// A launch rounds the rows of x to 8 bits, with the blocks' scales beside them; the product's launch copies rows of W and x global -> LDS
// (128 bytes of a row at a time: a block of 128) into a ring, and takes v_mfma_f32_16x16x128 over them.  W is operand A, so that a lane's sums
// belong to one row of x and one scale serves all of them; which rows of W make a tile is chosen so that a lane's outputs lie end to end.
#include "common.h"
#include "device_types.h"
#include "workspace.h"

#include <type_traits>

// The copies set M0, and say so; the compiler reports that it is a reserved register.
#pragma clang diagnostic ignored "-Winline-asm"

namespace hipattn {
namespace {

constexpr int kMostSplits = 8;  // ranges of k
constexpr int kBlock = 128;  // columns (and rows of W) that share a scale; bytes of a row per stage

struct Fp8Params {
  const void *x, *bias, *residual;
  const uint8_t *w, *xq;  // xq [KB, M, 128]: a tile's rows end to end (us, 4096 x 28672 x 4096: 499 row by row, 488 so)
  const float *ws;
  float *xs;  // [KB, Mp]
  void *out;
  float *partial;  // [splits, M, N]
  int M, N, K, KB, Mp;
  int64_t ldx, ldw, ldws, ldr, ldo;
  int splits, stages_per_split;
  int tiles_m, tiles_n;
  int wide_out;  // rows of out (and residual, and bias) on 16-byte boundaries
};

// ------------------------------------------------------------------ rows of x to 8 bits

// Eight elements of a block of which 16 lanes in a row hold the others: in 8 bits, and the block's scale (NaN for a block with a NaN or an infinity).
template <typename T>
__device__ __forceinline__ uint2 round_run(const uint4 raw, float &scale) {
  const T *e = reinterpret_cast<const T *>(&raw);
  float v[8];
  unsigned most = 0;  // bits of the largest magnitude; infinities and NaN are larger than any number
#pragma unroll
  for (int j = 0; j < 8; j++) {
    v[j] = to_float(e[j]);
    most = max(most, bit_cast<unsigned>(v[j]) & 0x7fffffffu);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) most = max(most, (unsigned)__shfl_xor((int)most, o, 16));
  // the least power of two s with most <= 448 s = 1.75 * 2^8 s
  const int up = max((int)((most + 0x1fffffu) >> 23) - 8, 1);  // its exponent's bits
  const float down = bit_cast<float>((unsigned)(254 - up) << 23);
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * down, v[1] * down, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * down, v[3] * down, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * down, v[5] * down, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * down, v[7] * down, hi, true);
  scale = most >= 0x7f800000u ? bit_cast<float>(0x7fc00000u) : bit_cast<float>((unsigned)up << 23);
  return make_uint2((unsigned)lo, (unsigned)hi);
}

// A thread takes eight elements, 16 threads a block.
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const Fp8Params p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int b = (int)(i / 16 % p.KB), m = (int)(i / 16 / p.KB), k = b * kBlock + (int)(i % 16) * 8;
  if (m >= p.M) return;
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (k < p.K) raw = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.x) + (int64_t)m * p.ldx + k);
  float scale;
  const uint2 q = round_run<T>(raw, scale);
  *reinterpret_cast<uint2 *>(const_cast<uint8_t *>(p.xq) + ((int64_t)b * p.M + m) * kBlock + (i % 16) * 8) = q;
  if (i % 16 == 0) p.xs[(int64_t)b * p.Mp + m] = scale;
}

// ------------------------------------------------------------------ the product

template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)p);
}

__device__ __forceinline__ const char *uniform_base(const char *ptr) {
  const uint64_t v = reinterpret_cast<uint64_t>(ptr);
  return reinterpret_cast<const char *>(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32) |
                                        (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v));
}

// 64 lanes x 16 bytes, global -> LDS: lane l's bytes go to lds + 16 l.  ONCE: with the hint that they are read once.
template <bool ONCE = false>
__device__ __forceinline__ void copy_1k(uint32_t lds, const char *base, uint32_t off) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
// 64 lanes x 4 bytes.
__device__ __forceinline__ void copy_256(uint32_t lds, const char *base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(4))) float uniform_float;

__device__ __forceinline__ f32x4_t mfma_fp8(i32x8_t a, i32x8_t b) {
  const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, 0, 0, 0, 0, 0, 0);
}

// The runs of 16 bytes of a row lie in LDS in the order q ^ turn, so that the rows of a tile do not meet in the same banks.
__device__ __forceinline__ i32x8_t operand(const char *rows, int r, int turn, int kg) {
  const uint4 a = *reinterpret_cast<const uint4 *>(rows + r * kBlock + ((kg ^ turn) * 16));
  const uint4 b = *reinterpret_cast<const uint4 *>(rows + r * kBlock + (((4 + kg) ^ turn) * 16));
  return i32x8_t{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

// v: the sums of y[m][n .. n + 3].
template <typename T>
__device__ __forceinline__ void finish4(const Fp8Params &p, const f32x4_t v, int m, int n, T *o) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  const T *bias = static_cast<const T *>(p.bias), *res = static_cast<const T *>(p.residual);
  vec4 b4 = vec4{(T)0.f, (T)0.f, (T)0.f, (T)0.f}, r4 = b4;
  if (bias != nullptr) b4 = *reinterpret_cast<const vec4 *>(bias + n);
  if (res != nullptr) r4 = *reinterpret_cast<const vec4 *>(res + (int64_t)m * p.ldr + n);
#pragma unroll
  for (int r = 0; r < 4; r++) {
    float f = v[r];
    if (bias != nullptr) f += to_float<T>(b4[r]);
    o[r] = from_float<T>(f);
    if (res != nullptr) o[r] = add_t<T>(o[r], r4[r]);
  }
}

// The order in which the stages of a range of k are taken: from one on that follows from the rows of W, and round.  Workgroups that all walk their
// rows front to back ask for the same bytes of every row at a time, and where rows lie a power of two apart those are a few of the memory's
// channels.
__device__ __forceinline__ int turned(int st, int n, int stages) {
  const int t = st + (int)((unsigned)(n / kBlock * 21) % (unsigned)stages);
  return t < stages ? t : t - stages;
}

// Up to 16 rows of x.  A wavefront owns 16 rows of W over one range of k, with a ring of its own that only its own copies fill, so that it waits for
// nothing else; `per_tile` wavefronts of a workgroup share the rows and meet in LDS at the end.
// HELD: the few rows of x are copied into LDS whole, behind the first stages of W in the queue but in front of them in time, and rounded there: no
// launch for that.  Else the rounded rows go through the ring as well.
// LDS: ring | sums | rows of x | their scales.
constexpr int kHeldBytes = 32 * 1024;
__host__ __device__ constexpr int held_pitch(int K) { return (K * 2 + 1023) / 1024 * 1024; }
template <bool HELD>
constexpr int few_stage_bytes() { return HELD ? 2048 : 4096 + 256; }

template <typename T, int S, int WAVES, bool HELD>
__global__ __launch_bounds__(WAVES * 64) void fp8_few_kernel(const Fp8Params p) {
  constexpr int kStage = few_stage_bytes<HELD>(), kCopies = HELD ? 2 : 5;
  extern __shared__ __align__(1024) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, kg = lane >> 4;
  const int tile = wave / p.splits, range = wave % p.splits, tiles = WAVES / p.splits;
  const int n0 = (blockIdx.x * tiles + tile) * 16;
  const int stage0 = range * p.stages_per_split, nst = max(0, min(p.stages_per_split, p.KB - stage0));
  char *ring = lds + wave * S * kStage;
  f32x4_t *sums = reinterpret_cast<f32x4_t *>(lds + WAVES * S * kStage);
  char *rows = reinterpret_cast<char *>(sums + WAVES * 64);
  const int pitch = held_pitch(p.K), xr = min(col, p.M - 1);
  float *scales = reinterpret_cast<float *>(rows + p.M * pitch);  // [KB][M]

  if constexpr (HELD) {
    const int per_row = pitch / 1024, last = p.K / 8 - 1;
    const uint32_t to = lds_address(rows);
    for (int i = wave; i < p.M * per_row; i += WAVES) {
      const int r = i / per_row, run = i % per_row * 64 + lane;
      copy_1k(to + i * 1024, uniform_base(reinterpret_cast<const char *>(static_cast<const T *>(p.x) + r * p.ldx)), (uint32_t)min(run, last) * 16);
    }
  }
  const int row8 = lane >> 3, run = ((lane & 7) ^ row8) * 16;  // run q of row r lies at place q ^ (r & 7)
  const char *wbase[2], *xbase[2];
  uint32_t woff[2], xoff[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int first = min(n0 + i * 8, p.N - 1);
    wbase[i] = uniform_base(reinterpret_cast<const char *>(p.w) + (int64_t)first * p.ldw);
    woff[i] = (uint32_t)(min(n0 + i * 8 + row8, p.N - 1) - first) * (uint32_t)p.ldw;
    const int xfirst = min(i * 8, p.M - 1);
    xbase[i] = uniform_base(reinterpret_cast<const char *>(p.xq) + (int64_t)xfirst * kBlock);
    xoff[i] = (uint32_t)(min(i * 8 + row8, p.M - 1) - xfirst) * kBlock + run;
  }
  const uint32_t ring_lds = lds_address(ring);
  auto ask = [&](int slot, int st) {
    const int b = stage0 + turned(st, n0, nst);
    const uint32_t to = ring_lds + slot * kStage;
    if constexpr (!HELD) {
#pragma unroll
      for (int i = 0; i < 2; i++) copy_1k(to + 2048 + i * 1024, xbase[i] + (int64_t)b * p.M * kBlock, xoff[i]);
      copy_256(to + 4096, uniform_base(reinterpret_cast<const char *>(p.xs + (int64_t)b * p.Mp)), lane * 4);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) copy_1k<true>(to + i * 1024, wbase[i], woff[i] + (uint32_t)min(b * kBlock + run, p.K - 16));
  };
#pragma unroll
  for (int j = 0; j < S; j++)
    if (j < nst) ask(j, j);
  if constexpr (HELD) {
    if (nst >= S) wait_copies<S * kCopies>();
    else wait_copies<0>();
    asm volatile("s_barrier" ::: "memory");
    const int runs = p.KB * 16;  // of a row, up to the end of its last block
    for (int i = threadIdx.x; i < p.M * runs; i += WAVES * 64) {
      const int r = i / runs, q = i - r * runs;
      uint4 *at = reinterpret_cast<uint4 *>(rows + r * pitch + q * 16);
      const uint4 raw = q * 8 < p.K ? *at : make_uint4(0, 0, 0, 0);
      float scale;
      *reinterpret_cast<uint2 *>(at) = round_run<T>(raw, scale);  // eight bytes in the place of sixteen
      if (q % 16 == 0) scales[q / 16 * p.M + r] = scale;
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
  const uniform_float *ws = (const uniform_float *)uniform_base(
      reinterpret_cast<const char *>(p.ws + (int64_t)(min(n0, p.N - 1) / kBlock) * p.ldws + stage0));
  const char *xrow = rows + xr * pitch + kg * 32;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  static_assert(S % 2 == 0, "stages are taken two at a time");
  for (int base = 0; base < nst; base += S) {
#pragma unroll
    for (int j = 0; j < S; j += 2) {
      const int st = base + j;
      if (st >= nst) break;
      // S stages are on their way, these two first; near the end fewer, and the wait is for all of them
      if (st + S - 1 < nst) wait_copies<(S - 2) * kCopies>();
      else wait_copies<0>();
      // (of two, as a stage by itself is a chain of waits; what lies in the place behind the last one is not added)
      i32x8_t wf[2], xf[2];
      float sx[2], sw[2];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const char *stage = ring + (j + u) * kStage;
        const int at = turned(min(st + u, nst - 1), n0, nst), b = stage0 + at;
        sw[u] = ws[at];
        wf[u] = operand(stage, col, col & 7, kg);
        if constexpr (HELD) {
          const uint2 *x = reinterpret_cast<const uint2 *>(xrow + b * 256);
          const uint2 x0 = x[0], x1 = x[2], x2 = x[16], x3 = x[18];
          xf[u] = i32x8_t{(int)x0.x, (int)x0.y, (int)x1.x, (int)x1.y, (int)x2.x, (int)x2.y, (int)x3.x, (int)x3.y};
          sx[u] = scales[b * p.M + xr];
        } else {
          xf[u] = operand(stage + 2048, col, col & 7, kg);
          sx[u] = reinterpret_cast<const float *>(stage + 4096)[col];
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stages are in registers: their places can be filled again
#pragma unroll
      for (int u = 0; u < 2; u++)
        if (st + u + S < nst) ask(j + u, st + u + S);
      f32x4_t part[2];
#pragma unroll
      for (int u = 0; u < 2; u++) part[u] = mfma_fp8(wf[u], xf[u]);
      const float s0 = sx[0] * sw[0], s1 = sx[1] * sw[1];
#pragma unroll
      for (int i = 0; i < 4; i++) acc[i] = __builtin_fmaf(part[0][i], s0, acc[i]);
      if (st + 1 < nst) {
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = __builtin_fmaf(part[1][i], s1, acc[i]);
      }
    }
  }
  if (p.splits > 1) {
    sums[wave * 64 + lane] = acc;
    __syncthreads();
    if (range > 0) return;
    for (int i = 1; i < p.splits; i++) {
      const f32x4_t v = sums[(wave + i) * 64 + lane];
#pragma unroll
      for (int r = 0; r < 4; r++) acc[r] += v[r];
    }
  }
  const int n = n0 + kg * 4;
  if (col >= p.M || n >= p.N) return;
  __align__(8) T o[4];
  finish4<T>(p, acc, col, n, o);
  *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + (int64_t)col * p.ldo + n) = *reinterpret_cast<uint2 *>(o);
}

// KG groups of GN x GM wavefronts, each with WN x WM tiles of 16 rows of W x 16 rows of x; a group takes every KG-th stage of k, and their sums meet in
// LDS at the end.  S rounds of KG stages in the ring.  ONCE: no other workgroup reads the rows of W.
template <typename T, int WN, int WM, int GN, int GM, int KG, int S, bool ONCE>
__global__ __launch_bounds__(GN *GM *KG * 64) void fp8_tile_kernel(const Fp8Params p) {
  constexpr int WAVES = GN * GM * KG, BN = GN * WN * 16, BM = GM * WM * 16;
  constexpr int kAllW = KG * BN / 8, kCopiesW = (kAllW + WAVES - 1) / WAVES, kAllX = KG * BM / 8, kCopiesX = (kAllX + WAVES - 1) / WAVES;
  constexpr int kPieces = (BM + 63) / 64, kAllS = KG * kPieces, kCopiesS = (kAllS + WAVES - 1) / WAVES;  // of 64 scales
  constexpr int kCopies = kCopiesW + kCopiesX + kCopiesS;
  constexpr int kStageBytes = (BN + BM) * kBlock + kPieces * 256, kRoundBytes = KG * kStageBytes;
  constexpr int kMeetBytes = (KG - 1) * GN * GM * WN * WM * 1024;
  constexpr int kLds = S * kRoundBytes > kMeetBytes ? S * kRoundBytes : kMeetBytes;
  __shared__ __align__(1024) char ring[kLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, kg = lane >> 4;
  const int wn = wave % GN, wm = wave / GN % GM, group = wave / (GN * GM);
  // Tiles in strips of four of W by all of x, and of that list a contiguous part to each XCD, which shares an L2.
  const int tiles = p.tiles_m * p.tiles_n, per_xcd = (tiles + 7) / 8;
  const int at = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || at >= tiles) return;
  const int strip = at / (4 * p.tiles_m), in_strip = at - strip * 4 * p.tiles_m, width = min(4, p.tiles_n - strip * 4);
  const int n0 = (strip * 4 + in_strip % width) * BN, m0 = in_strip / width * BM;
  const int stage0 = blockIdx.y * p.stages_per_split, nst = max(0, min(p.stages_per_split, p.KB - stage0));
  const int rounds = (nst + KG - 1) / KG;

  // What a lane copies of eight rows: run q of row r to this lane's place.  Rows past the last repeat it; columns past the last of W, where x is zero,
  // repeat the row's last run; stages past the last repeat that.  Copies that do not divide evenly are made twice (the same bytes to the same place):
  // every wavefront counts the same number of them.
  const char *wbase[kCopiesW], *xbase[kCopiesX];
  uint32_t woff[kCopiesW], xoff[kCopiesX];
  int wrun[kCopiesW];
  const int row8 = lane >> 3;
#pragma unroll
  for (int i = 0; i < kCopiesW; i++) {
    const int r = (wave + i * WAVES) % kAllW % (BN / 8) * 8, in_tile = r + row8;  // row of the workgroup's
    const int in_wave = in_tile % (WN * 16), turn = (in_wave & 3) + 4 * (in_wave / (4 * WN) & 1);
    const int first = min(n0 + r, p.N - 1), rows_on = min(n0 + in_tile, p.N - 1) - first;
    wrun[i] = ((lane & 7) ^ turn) * 16;
    wbase[i] = uniform_base(reinterpret_cast<const char *>(p.w) + (int64_t)first * p.ldw);
    woff[i] = (uint32_t)rows_on * (uint32_t)p.ldw;
  }
#pragma unroll
  for (int i = 0; i < kCopiesX; i++) {
    const int r = (wave + i * WAVES) % kAllX % (BM / 8) * 8, in_tile = r + row8;
    const int first = min(m0 + r, p.M - 1), rows_on = min(m0 + in_tile, p.M - 1) - first;
    xbase[i] = uniform_base(reinterpret_cast<const char *>(p.xq) + (int64_t)first * kBlock);
    xoff[i] = (uint32_t)rows_on * kBlock + ((lane & 7) ^ (row8 & 7)) * 16;
  }
  const uint32_t ring_lds = lds_address(ring);
  const char *sbase = uniform_base(reinterpret_cast<const char *>(p.xs + m0));
  // The block of the u-th stage of a round (see `turned`; without its division here).  A strip's tiles of W that read the same rows of x at once read
  // the same blocks of them where there are many such rows (us, 4096 x 28672 x 4096: 523, 505 so; 600 rows: 107.6, 109.3, so not with few).
  const int turn = nst > 0 ? turned(0, p.tiles_m >= 4 ? strip * 4 * BN : n0, nst) : 0;
  auto block_of = [&](int round, int u) {
    const int t = min(round * KG + u, nst - 1) + turn;
    return stage0 + (t < nst ? t : t - nst);
  };
  // The c-th of a wavefront's copies of a round.
  auto ask = [&](int slot, int round, int c) {
    const uint32_t to = ring_lds + slot * kRoundBytes;
    if (c < kCopiesX) {
      const int i = (wave + c * WAVES) % kAllX, u = i / (BM / 8);
      copy_1k(to + u * kStageBytes + (BN + i % (BM / 8) * 8) * kBlock, xbase[c] + (int64_t)block_of(round, u) * p.M * kBlock, xoff[c]);
    } else if (c < kCopiesX + kCopiesW) {
      c -= kCopiesX;
      const int i = (wave + c * WAVES) % kAllW, u = i / (BN / 8);
      copy_1k<ONCE>(to + u * kStageBytes + i % (BN / 8) * 1024, wbase[c], woff[c] + (uint32_t)min(block_of(round, u) * kBlock + wrun[c], p.K - 16));
    } else {
      c -= kCopiesX + kCopiesW;
      const int i = (wave + c * WAVES) % kAllS, u = i / kPieces, piece = i % kPieces;
      copy_256(to + u * kStageBytes + (BN + BM) * kBlock + piece * 256, sbase + ((int64_t)block_of(round, u) * p.Mp + piece * 64) * 4, lane * 4);
    }
  };

  f32x4_t acc[WN][WM];
#pragma unroll
  for (int nt = 0; nt < WN; nt++)
#pragma unroll
    for (int mt = 0; mt < WM; mt++) acc[nt][mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // (through the scalar cache: a vector load would wait for the copies in front of it)
  const uniform_float *ws =
      (const uniform_float *)uniform_base(reinterpret_cast<const char *>(p.ws + (int64_t)(min(n0 + wn * WN * 16, p.N - 1) / kBlock) * p.ldws));
  float sw = nst > 0 ? ws[block_of(0, group)] : 0.f;
  const int turn_w = (col & 3) + 4 * (col >> 2 & 1);  // of this lane's row of every tile of W
#pragma unroll
  for (int j = 0; j < S - 1; j++) {
    if (j >= rounds) continue;
#pragma unroll
    for (int c = 0; c < kCopies; c++) ask(j, j, c);
  }
  int slot = 0;
  // (MORE: there is a round S - 1 further on to ask for; a loop of its own, as a condition around every copy keeps the products apart)
  auto take = [&](int st, auto more) {
    constexpr bool MORE = decltype(more)::value;
    // This wavefront's copies of the round have landed, and behind the barrier everybody's; the barrier also says that the round before has
    // been read, so its place takes the copies of the round S - 1 further on.
    if (MORE || st + S - 2 < rounds) wait_copies<(S - 2) * kCopies>();
    else wait_copies<0>();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const char *stage = ring + slot * kRoundBytes + group * kStageBytes;
    const int fill = slot == 0 ? S - 1 : slot - 1;
    slot = slot == S - 1 ? 0 : slot + 1;
    if (!MORE && KG > 1 && st * KG + group >= nst) return;  // (the last round)
    const char *wrows = stage + wn * WN * 16 * kBlock, *xrows = stage + BN * kBlock;
    const float *scales = reinterpret_cast<const float *>(stage + (BN + BM) * kBlock);
    const float sw_next = ws[block_of(st + 1, group)];  // (here: the next round's barrier waits for all of them)
    i32x8_t xf[WM];
    float s[WM];
#pragma unroll
    for (int mt = 0; mt < WM; mt++) {
      const int r = (wm * WM + mt) * 16 + col;
      xf[mt] = operand(xrows, r, col & 7, kg);
      s[mt] = scales[r];
    }
    // A tile's products go into the sums while the matrix pipe has the next tile's; the rows of W of the tile behind that are on their way.
    auto rows_of = [&](int nt) { return operand(wrows, (col >> 2) * (4 * WN) + nt * 4 + (col & 3), turn_w, kg); };
    i32x8_t wf = rows_of(0);
    f32x4_t part[WM];
#pragma unroll
    for (int nt = 0; nt <= WN; nt++) {
      const i32x8_t now = wf;
      if (nt + 1 < WN) wf = rows_of(nt + 1);
      if (nt == 1) {
#pragma unroll
        for (int mt = 0; mt < WM; mt++) s[mt] *= sw;
      }
#pragma unroll
      for (int mt = 0; mt < WM; mt++) {
        f32x4_t next = {0.f, 0.f, 0.f, 0.f};
        if (nt < WN) next = mfma_fp8(now, xf[mt]);
        if (nt > 0) {
#pragma unroll
          for (int i = 0; i < 4; i++) acc[nt - 1][mt][i] = __builtin_fmaf(part[mt][i], s[mt], acc[nt - 1][mt][i]);
        }
        part[mt] = next;
      }
      // The copies go out between the products, as the matrix pipe would wait for them if they were in front; behind the first of them where the
      // ring is short and they are needed in the next round.
      if constexpr (MORE) {
#pragma unroll
        for (int c = S > 2 ? kCopies * nt / (WN + 1) : 0; c < (S > 2 ? kCopies * (nt + 1) / (WN + 1) : (nt == 0 ? kCopies : 0)); c++)
          ask(fill, st + S - 1, c);
      }
      // (in this order: left to itself the compiler puts the additions in front, where they wait)
      if (nt + 1 < WN) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
      for (int mt = 0; mt < WM; mt++) {
        if (nt < WN) __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        if (nt > 0) __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    sw = sw_next;
  };
  int st = 0;
  for (; st + S - 1 < rounds; st++) take(st, std::true_type{});
  for (; st < rounds; st++) take(st, std::false_type{});
  if constexpr (KG > 1) {
    __syncthreads();
    f32x4_t *meet = reinterpret_cast<f32x4_t *>(ring) + (wave % (GN * GM)) * WN * WM * 64 + lane;
    constexpr int kGroup = GN * GM * WN * WM * 64;
    if (group > 0) {
#pragma unroll
      for (int nt = 0; nt < WN; nt++)
#pragma unroll
        for (int mt = 0; mt < WM; mt++) meet[(group - 1) * kGroup + (nt * WM + mt) * 64] = acc[nt][mt];
    }
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int g = 0; g < KG - 1; g++)
#pragma unroll
      for (int nt = 0; nt < WN; nt++)
#pragma unroll
        for (int mt = 0; mt < WM; mt++) {
          const f32x4_t v = meet[g * kGroup + (nt * WM + mt) * 64];
#pragma unroll
          for (int i = 0; i < 4; i++) acc[nt][mt][i] += v[i];
        }
  }

  // A lane has 4 WN outputs of a row, end to end.
  const int n = n0 + wn * WN * 16 + kg * 4 * WN;
#pragma unroll
  for (int mt = 0; mt < WM; mt++) {
    const int m = m0 + (wm * WM + mt) * 16 + col;
    if (m >= p.M) continue;
    if (p.splits > 1) {
      float *to = p.partial + ((int64_t)blockIdx.y * p.M + m) * p.N + n;
#pragma unroll
      for (int nt = 0; nt < WN; nt++)
        if (n + nt * 4 < p.N) *reinterpret_cast<f32x4_t *>(to + nt * 4) = acc[nt][mt];
      continue;
    }
    T *to = static_cast<T *>(p.out) + (int64_t)m * p.ldo + n;
    if constexpr (WN % 2 == 0) {
      if (p.wide_out) {
#pragma unroll
        for (int nt = 0; nt < WN; nt += 2) {
          if (n + nt * 4 >= p.N) continue;  // (N is a multiple of 16, so of the eight that lie here)
          __align__(16) T o[8];
          finish4<T>(p, acc[nt][mt], m, n + nt * 4, o);
          finish4<T>(p, acc[nt + 1][mt], m, n + nt * 4 + 4, o + 4);
          *reinterpret_cast<uint4 *>(to + nt * 4) = *reinterpret_cast<uint4 *>(o);
        }
        continue;
      }
    }
#pragma unroll
    for (int nt = 0; nt < WN; nt++) {
      if (n + nt * 4 >= p.N) continue;
      __align__(8) T o[4];
      finish4<T>(p, acc[nt][mt], m, n + nt * 4, o);
      *reinterpret_cast<uint2 *>(to + nt * 4) = *reinterpret_cast<uint2 *>(o);
    }
  }
}

// Adds up the ranges' sums, the first range first: a thread for four outputs.
template <typename T>
__global__ __launch_bounds__(256) void fp8_reduce_kernel(const Fp8Params p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int quads = p.N / 4, n = (int)(i % quads) * 4;
  const int64_t m = i / quads;
  if (m >= p.M) return;
  const float *from = p.partial + m * p.N + n;
  f32x4_t v[kMostSplits];  // (all asked for at once)
#pragma unroll
  for (int s = 0; s < kMostSplits; s++)
    if (s < p.splits) v[s] = *reinterpret_cast<const f32x4_t *>(from + (int64_t)s * p.M * p.N);
  f32x4_t sum = v[0];
#pragma unroll
  for (int s = 1; s < kMostSplits; s++)
    if (s < p.splits) {
#pragma unroll
      for (int r = 0; r < 4; r++) sum[r] += v[s][r];
    }
  __align__(8) T o[4];
  finish4<T>(p, sum, (int)m, n, o);
  *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + m * p.ldo + n) = *reinterpret_cast<uint2 *>(o);
}

// ------------------------------------------------------------------ choices

// The forms of the product: of few rows, and of tiles with the sizes of fp8_tile_kernel.
enum Fp8Form { FP8_HELD, FP8_FEW, FP8_TILES };
#define FP8_TILE_FORMS(X)          \
  X(0, 1, 2, 1, 1, 4, 4, true)     \
  X(1, 1, 2, 2, 1, 2, 4, true)     \
  X(2, 2, 2, 4, 1, 1, 4, true)     \
  X(3, 1, 4, 1, 1, 4, 3, true)     \
  X(4, 1, 4, 2, 1, 4, 3, true)     \
  X(5, 1, 4, 4, 1, 1, 4, true)     \
  X(6, 1, 4, 8, 1, 1, 4, true)     \
  X(7, 1, 4, 4, 2, 1, 4, true)     \
  X(8, 2, 4, 4, 2, 1, 3, true)     \
  X(9, 4, 4, 2, 2, 1, 2, false)    \
  X(10, 8, 4, 2, 4, 1, 2, false)
struct TileForm {
  int bn, bm;
};
constexpr TileForm kTileForms[] = {
#define X(i, WN, WM, GN, GM, KG, S, ONCE) {GN * WN * 16, GM * WM * 16},
    FP8_TILE_FORMS(X)
#undef X
};

struct Fp8Plan {
  Fp8Form form;
  int tile;  // of kTileForms
  int bn, bm, splits, stages_per_split;
  size_t xq_bytes, xs_bytes, bytes;  // rounded rows of x, their scales, everything
  int Mp;
};

// What bounds the tiles up to 128 rows is what a compute unit gets into LDS, some 30 to 40 bytes a nanosecond with 64 to 96 KB on their way:
// narrow tiles of W give every unit work, wide ones copy x less often.  us with the rows' launch, in rows of W per workgroup:
//   up to 32 rows   4096 x 4096 16: 10.2, 32: 11.2, 128: 17.9; 6144 x 4096 14.8, 12.1, 18.4; 4096 x 14336 20.5, 24.7, 49.7; 28672 x 4096 42.9, 29.4, 24.6
//   up to 64        4096 x 4096 16: 11.8, 32: 12.8, 64: 17.3, 128: 22.0; 6144 x 4096 18.9, 13.9, 17.8, 22.2; 28672 x 4096 50.7, 38.1, 27.6, 25.5
//   up to 128       6144 x 4096 64: 22.3, 128: 29.8; 28672 x 4096 46.2, 36.8
// Beyond 128 rows workgroups of 256 x 256, 2.1 us a stage (the choice below counts 2.25, from before the rounded rows lay block by block), of whose some 4100 cycles the matrix pipe is busy 2048 (us, 4096 x 28672 x 4096: 485; with no
// copies but the first stages' 402, which is what products, additions and reads of LDS take of each other; LDS 18 %, no bank conflicts; reading a stage's
// first rows among the last products of the one before, 482; refilling parts of a stage's place as soon as they have been read, with two more barriers,
// a third longer), or of 128 x 128, two to a compute unit, 1.2 a stage and 1.37 where there are two; ranges of k
// of workgroups of their own cost a launch and their sums' way through memory (4096 x 14336, 301 rows: one range 134, two 81, four 52).
// apart: out does not lie over x.
Fp8Plan plan_fp8(int64_t M, int N, int K, bool apart) {
  Fp8Plan pl;
  const int KB = (K + kBlock - 1) / kBlock;
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  if (M <= 16) {
    // Rows held in LDS cost the compute unit its second workgroup from three of 4096 on (us, 6144 x 4096, 4 rows: held 11.3, through the ring 9.2).
    // Every workgroup reads them while others write out, which is then no place over x.
    const bool held = apart && M <= 2 && M * held_pitch(K) <= kHeldBytes;
    pl.form = held ? FP8_HELD : FP8_FEW;
    // Wavefronts to a tile of 16 rows of W: until every compute unit has three, or four where a wavefront's chain of stages is long.  us, one row, 1 / 2
    // / 4 / 8: 4096 x 4096 10.3, 7.8, 6.7, 7.5; 6144 x 4096 10.5, 8.4, 8.6, 12.3; 4096 x 14336 26.4, 17.4, 14.9, 13.4; 28672 x 4096 20.6, 22.8, 25.2, 39.9.
    int per = 1;
    const int64_t tiles = (N + 15) / 16;
    while (per < 8 && KB / (2 * per) >= 2 && (tiles * per < 768 || (KB > 16 * per && tiles * per <= 1024))) per *= 2;
    pl.splits = per;
    pl.stages_per_split = (KB + per - 1) / per;
    pl.bn = pl.bm = 16;
    pl.tile = 0;
    pl.Mp = 64;
    pl.xq_bytes = held ? 0 : up((size_t)M * KB * kBlock);
    pl.xs_bytes = held ? 0 : up((size_t)KB * pl.Mp * 4);
    pl.bytes = pl.xq_bytes + pl.xs_bytes;
    return pl;
  }
  pl.form = FP8_TILES;
  int splits = 1;
  if (M <= 32) {
    pl.tile = N < 4800 ? 0 : (N < 16384 ? 1 : 2);
  } else if (M <= 64) {
    pl.tile = N < 4800 ? 3 : (N <= 8192 ? 4 : (N < 16384 ? 5 : 6));
  } else if (M <= 128) {
    pl.tile = N < 16384 ? 7 : 8;
    while (splits < kMostSplits && 2 * splits * ((N + 63) / 64) <= 256 && KB / (2 * splits) >= 8) splits *= 2;
  } else {
    const int64_t large = ((M + 255) / 256) * ((N + 255) / 256), small = ((M + 127) / 128) * ((N + 127) / 128);
    double us = (double)((large + 255) / 256) * 2.25 * KB;
    pl.tile = 10;
    for (int s = 1; s <= kMostSplits && (s == 1 || KB / s >= 4); s++) {
      const double t = (double)((small * s + 511) / 512) * ((KB + s - 1) / s) * (small * s <= 256 ? 1.2 : 1.37) +
                       (s > 1 ? 4 + (double)M * N * s * (8 / 3.5e6) : 0);
      if (t < us) {
        us = t;
        pl.tile = 9;
        splits = s;
      }
    }
  }
  pl.bn = kTileForms[pl.tile].bn;
  pl.bm = kTileForms[pl.tile].bm;
  pl.stages_per_split = (KB + splits - 1) / splits;
  pl.splits = (KB + pl.stages_per_split - 1) / pl.stages_per_split;
  pl.Mp = (int)((M + 255) / 256 * 256);
  pl.xq_bytes = up((size_t)M * KB * kBlock);
  pl.xs_bytes = up((size_t)KB * pl.Mp * 4);
  pl.bytes = pl.xq_bytes + pl.xs_bytes + (pl.splits > 1 ? up((size_t)pl.splits * M * N * 4) : 0);
  return pl;
}

template <typename T, int S, int WAVES, bool HELD>
void launch_few(const Fp8Params &p, hipStream_t stream) {
  auto kernel = fp8_few_kernel<T, S, WAVES, HELD>;
  constexpr size_t fixed = (size_t)WAVES * (S * few_stage_bytes<HELD>() + 1024);
  static bool attr_set = false;  // benign race: setting twice is harmless
  if (!attr_set) {
    HA_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    attr_set = true;
  }
  const int rows = 16 * (WAVES / p.splits);
  const size_t bytes = fixed + (HELD ? (size_t)p.M * (held_pitch(p.K) + p.KB * 4) : 0);
  kernel<<<dim3((unsigned)((p.N + rows - 1) / rows)), WAVES * 64, bytes, stream>>>(p);
  check_launch("linear_fp8 (few rows)");
}

template <typename T>
void launch_fp8(const Fp8Params &p, const Fp8Plan &pl, hipStream_t stream) {
  if (pl.form == FP8_HELD) {
    if (p.splits > 4) launch_few<T, 6, 8, true>(p, stream);
    else launch_few<T, 8, 4, true>(p, stream);
    return;
  }
  const int64_t threads = (int64_t)p.M * p.KB * 16;
  quantize_rows_kernel<T><<<dim3((unsigned)((threads + 255) / 256)), 256, 0, stream>>>(p);
  check_launch("linear_fp8 (rows)");
  if (pl.form == FP8_FEW) {
    if (p.splits > 4) launch_few<T, 4, 8, false>(p, stream);
    else launch_few<T, 4, 4, false>(p, stream);
    return;
  }
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  const dim3 grid((unsigned)((tiles + 7) / 8 * 8), (unsigned)p.splits);
  switch (pl.tile) {
#define X(i, WN, WM, GN, GM, KG, S, ONCE) \
  case i: fp8_tile_kernel<T, WN, WM, GN, GM, KG, S, ONCE><<<grid, GN * GM * KG * 64, 0, stream>>>(p); break;
    FP8_TILE_FORMS(X)
#undef X
  }
  check_launch("linear_fp8");
  if (p.splits > 1) {
    const int64_t quads = (int64_t)p.M * (p.N / 4);
    fp8_reduce_kernel<T><<<dim3((unsigned)((quads + 255) / 256)), 256, 0, stream>>>(p);
    check_launch("linear_fp8 (sum of the ranges)");
  }
}

bool at_multiple(const void *p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

void linear_fp8_impl(hipattn_tensor *out, const hipattn_tensor *x, const hipattn_tensor *weight, const hipattn_tensor *scale,
                     const hipattn_tensor *bias, const hipattn_tensor *residual, const hipattn_tensor *workspace, void *stream_arg,
                     int64_t *ws_query) {
  const char *op = "linear_fp8";
  check_tensor(x, "x", 2);
  check_tensor(weight, "weight", 2);
  const int dt = x->dtype;
  HA_CHECK(dt == HIPATTN_F16 || dt == HIPATTN_BF16, "%s: x must be f16 or bf16, got %s", op, dtype_name(dt));
  HA_CHECK(weight->dtype == HIPATTN_E4M3, "%s: weight must be e4m3, got %s", op, dtype_name(weight->dtype));
  const int64_t M = x->sizes[0], K = x->sizes[1], N = weight->sizes[0];
  HA_CHECK(weight->sizes[1] == K, "%s: weight has %lld columns, x has %lld", op, (long long)weight->sizes[1], (long long)K);
  HA_CHECK(K > 0 && K % 16 == 0 && N % 16 == 0, "%s: the inner size %lld must be a positive multiple of 16, the rows of weight %lld one of 16", op,
           (long long)K, (long long)N);
  HA_CHECK(N < (1 << 24) && K < (1 << 24) && M < (1 << 24), "%s: sizes out of range", op);
  if (ws_query != nullptr) {  // (of either place of out)
    *ws_query = M == 0 || N == 0 ? 0 : (int64_t)plan_fp8(M, (int)N, (int)K, false).bytes;
    return;
  }
  check_tensor(scale, "weight_scale", 2);
  check_tensor(out, "out", 2);
  HA_CHECK(out->dtype == dt, "%s: out is %s, x is %s", op, dtype_name(out->dtype), dtype_name(dt));
  HA_CHECK(out->sizes[0] == M && out->sizes[1] == N, "%s: out is [%lld, %lld], expected [%lld, %lld]", op, (long long)out->sizes[0],
           (long long)out->sizes[1], (long long)M, (long long)N);
  const int64_t NB = (N + kBlock - 1) / kBlock, KB = (K + kBlock - 1) / kBlock;
  HA_CHECK(scale->dtype == HIPATTN_F32 && scale->sizes[0] == NB && scale->sizes[1] == KB,
           "%s: weight_scale must be f32 [%lld, %lld], one for each 128 x 128 of weight", op, (long long)NB, (long long)KB);
  HA_CHECK(KB == 1 || scale->strides[1] == 1, "%s: rows of weight_scale must be contiguous", op);
  if (M == 0 || N == 0) return;
  check_data(x, "x");
  check_data(weight, "weight");
  check_data(scale, "weight_scale");
  check_data(out, "out");
  HA_CHECK(x->strides[1] == 1 && weight->strides[1] == 1 && out->strides[1] == 1,
           "%s: the last dimension of x, weight and out must be contiguous", op);
  HA_CHECK((M == 1 || x->strides[0] % 8 == 0) && weight->strides[0] % 16 == 0 && at_multiple(x->data, 16) && at_multiple(weight->data, 16),
           "%s: rows of x and weight must start on 16-byte boundaries", op);
  HA_CHECK((M == 1 || out->strides[0] % 4 == 0) && at_multiple(out->data, 8), "%s: rows of out must start on 8-byte boundaries", op);
  HA_CHECK(weight->strides[0] >= 0 && weight->strides[0] < (1 << 28), "%s: rows of weight lie too far apart", op);
  HA_CHECK(!may_share(out, weight), "%s: out lies over weight", op);
  HA_CHECK(!may_share(out, scale), "%s: out lies over weight_scale", op);
  const Fp8Plan pl = plan_fp8(M, (int)N, (int)K, !may_share(out, x));
  Fp8Params p{};
  if (bias != nullptr) {
    check_tensor(bias, "bias", 1);
    HA_CHECK(bias->dtype == dt && bias->sizes[0] == N && bias->strides[0] == 1 && at_multiple(bias->data, 8),
             "%s: bias must be %lld contiguous %s on an 8-byte boundary", op, (long long)N, dtype_name(dt));
    check_data(bias, "bias");
    HA_CHECK(!may_share(out, bias), "%s: out lies over bias", op);
    p.bias = bias->data;
  }
  if (residual != nullptr) {
    check_tensor(residual, "residual", 2);
    HA_CHECK(residual->dtype == dt && residual->sizes[0] == M && residual->sizes[1] == N && residual->strides[1] == 1,
             "%s: residual must be [%lld, %lld] %s with a contiguous last dimension", op, (long long)M, (long long)N, dtype_name(dt));
    HA_CHECK((M == 1 || residual->strides[0] % 4 == 0) && at_multiple(residual->data, 8), "%s: rows of residual must start on 8-byte boundaries",
             op);
    check_data(residual, "residual");
    HA_CHECK((out->data == residual->data && (M == 1 || out->strides[0] == residual->strides[0])) || !may_share(out, residual),
             "%s: out lies over part of residual", op);
    p.residual = residual->data;
    p.ldr = residual->strides[0];
  }
  p.x = x->data;
  p.w = static_cast<const uint8_t *>(weight->data);
  p.ws = static_cast<const float *>(scale->data);
  p.out = out->data;
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  p.KB = (int)KB;
  p.Mp = pl.Mp;
  p.ldx = M == 1 ? 0 : x->strides[0];
  p.ldw = weight->strides[0];
  p.ldws = scale->strides[0];
  p.ldo = M == 1 ? 0 : out->strides[0];
  if (M == 1) p.ldr = 0;
  p.splits = pl.splits;
  p.stages_per_split = pl.stages_per_split;
  p.tiles_m = (int)((M + pl.bm - 1) / pl.bm);
  p.tiles_n = (int)((N + pl.bn - 1) / pl.bn);
  p.wide_out = p.ldo % 8 == 0 && at_multiple(out->data, 16);
  HA_CHECK((int64_t)p.tiles_m * p.tiles_n < 0x7fffff00 / 8 && M * KB < (int64_t)0x7fffffff * 16, "%s: sizes out of range", op);
  hipStream_t stream = resolve_stream(stream_arg);
  HeldWorkspace held;  // over all launches
  char *store = nullptr;
  if (pl.bytes == 0) {
  } else if (workspace != nullptr) {
    check_tensor(workspace, "workspace", 1);
    HA_CHECK(workspace->dtype == HIPATTN_U8 && workspace->strides[0] == 1, "%s: workspace must be contiguous u8", op);
    HA_CHECK((size_t)workspace->sizes[0] >= pl.bytes, "%s: workspace has %lld bytes, %zu are needed", op, (long long)workspace->sizes[0], pl.bytes);
    HA_CHECK(workspace->data != nullptr && at_multiple(workspace->data, 256), "%s: workspace must be 256-byte aligned", op);
    store = static_cast<char *>(workspace->data);
  } else {
    held = library_workspace(WS_LINEAR_FP8, pl.bytes, stream);
    store = static_cast<char *>(held.ptr);
  }
  p.xq = reinterpret_cast<const uint8_t *>(store);
  p.xs = reinterpret_cast<float *>(store + pl.xq_bytes);
  p.partial = reinterpret_cast<float *>(store + pl.xq_bytes + pl.xs_bytes);
  if (dt == HIPATTN_BF16) launch_fp8<bf16_t>(p, pl, stream);
  else launch_fp8<half_t>(p, pl, stream);
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" char *hipattn_linear_fp8(hipattn_tensor *out, const hipattn_tensor *x, const hipattn_tensor *weight, const hipattn_tensor *weight_scale,
                                    const hipattn_tensor *bias, const hipattn_tensor *residual, const hipattn_tensor *workspace, void *stream) {
  HA_PROTECT(linear_fp8_impl(out, x, weight, weight_scale, bias, residual, workspace, stream, nullptr));
}

extern "C" char *hipattn_linear_fp8_workspace_size(const hipattn_tensor *x, const hipattn_tensor *weight, int64_t *bytes) {
  HA_PROTECT({
    HA_CHECK(bytes != nullptr, "linear_fp8_workspace_size: bytes is NULL");
    linear_fp8_impl(nullptr, x, weight, nullptr, nullptr, nullptr, nullptr, nullptr, bytes);
  });
}
