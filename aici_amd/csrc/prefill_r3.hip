// Varlen flash-attention forward for gfx950, the form that rotates three groups of wavefronts through the
// matrix pipe.  Replaces the reference's mha_varlen_fwd (rllm/tch-cuda/kernels/flash_attn/flash_api.cpp:
// 447-655 and flash_fwd_kernel.h:590-1136) for head sizes up to 128, causal or unmasked, K and V given as rows.
//
// A workgroup is twelve wavefronts of at most 168 registers, three per SIMD, in three groups of four (one
// wavefront of a group on each SIMD).  A wavefront owns 32 query rows and repeats three blocks per 32-key tile:
//   V1(t)  mask, row maximum, the (rare) rescaling of the accumulators;
//   V2(t)  the exponentials, row sums and roundings of P(t); then its share of the tile copies;
//   M(t)   the eight MFMAs of P(t).V(t) and the eight of S(t+1), one stream with its LDS operand reads.
// There is one workgroup barrier per tile, and each group meets it at a different place of its own sequence --
// group 0 behind V1, group 1 behind V2, group 2 behind M -- so between two barriers the three wavefronts of a
// SIMD run (V2 M V1), (M V1 V2) and (V1 V2 M): their M blocks follow one another.  What this is built on,
// measured on MI355X with one MFMA wavefront and up to two vector wavefronts on a SIMD: the MFMA wavefront
// keeps 32.5 cycles per v_mfma_f32_32x32x16 whatever runs beside it (and whichever wavefront is the older);
// two MFMA wavefronts take turns without loss; the vector wavefronts share what the MFMA issue leaves of the
// vector port (about 7 of every 32 cycles go to the issue of an MFMA).  So the matrix pipe is best fed by one
// wavefront at a time with dense blocks, and the vector port by the two others.
//
// The twelve wavefronts share the K and V tiles: with four query heads per kv head a workgroup covers four
// heads x 96 rows, otherwise one head x 384 rows.  Tiles are 32 keys: K as the two 16-token block images
// [16-byte run][token] of the paged cache's layout, V as the rows they are, both copied global -> LDS with
// global_load_lds_dwordx4 (no staging registers) into five places each.  The second product takes its operands
// from the V rows with the transposing LDS read.  Numerics and the orientation of the two products (S^T =
// K.Q^T, O^T = V^T.P^T on v_mfma_f32_32x32x16) are those of the other prefill kernels (prefill_varlen.hip).
//
// Against the eight-wavefront kernel (prefill_varlen.hip) on 8 x 4096 tokens, 32 q / 8 kv heads, d 128: a tile
// period of 2400 to 2700 cycles for three 32-key wavefront-tiles per SIMD (57 to 63 % of the matrix pipe inside
// the loop) against 3140 for two 64-key ones (65 %), and more cycles per workgroup outside the loop (the wait for
// Q at the first barrier; the launch of a 768-thread workgroup; the wind-down).  With the two kernels taking
// turns on a warm device this one is 1 % behind there and 2 to 8 % behind on shorter sequences; it is therefore
// kept as a kernel that a caller can ask for (prefill_kernel = 4), not one the library picks.
#include "prefill_common.h"

// The global -> LDS copies set M0 inside inline asm and name it in their clobber lists; M0 is a register
// the compiler reserves, and naming a reserved register there draws a warning per use.
#pragma clang diagnostic ignored "-Winline-asm"

namespace hipattn {

namespace {

constexpr int XBN = 32;  // keys per tile
constexpr int NW = 12;   // wavefronts per workgroup


template <typename T, int HDP>
__global__ __launch_bounds__(768) void prefill_varlen_r3_kernel(PrefillParams p) {
  typedef typename Vec8<T>::type vec8;
  constexpr int KSTEPS = HDP / 16;          // contraction steps of S^T = K.Q^T
  constexpr int NDT = HDP / 32;             // 32-row tiles of O^T
  constexpr int TILE_ELEMS = XBN * HDP;     // one K or one V tile
  constexpr int TILE_BYTES = TILE_ELEMS * (int)sizeof(T);
  constexpr int NBUF = 5;
  constexpr int V_REGION = NBUF * TILE_BYTES;  // V tiles lie behind the K tiles

  extern __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[];
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char *)smem_raw;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int wave_u = __builtin_amdgcn_readfirstlane(wave);
  const int g = lane >> 5;
  const int c = lane & 31;
  const int hl = p.wg_heads_log2;  // 0: one head x 384 rows; 2: four heads of a kv group x 96 rows
  const int BM = (32 * NW) >> hl;
  const int grp = wave_u >> 2;     // the group: which third of a period this wavefront has the matrix pipe in
  const int sub = wave_u & 3;      // its place in the group (the SIMD, as wavefronts are dealt)

  // Workgroups in launch order: query head fastest (the heads of a kv group land on one XCD and share its
  // L2), then the row blocks of a sequence, last rows -- the longest stretch of keys under the causal mask
  // -- first, then the sequence.
  int id = blockIdx.x;
  const int n_slots = p.Hq >> hl;
  const int slot = id % n_slots;
  id /= n_slots;
  const int b = id / p.n_qblocks;
  const int qb = p.n_qblocks - 1 - id % p.n_qblocks;
  const int head0 = ((slot % p.Hkv) * (p.G >> hl) + slot / p.Hkv) << hl;
  const int h = head0 + (hl == 0 ? 0 : sub);
  const int kvh = head0 / p.G;

  const int q_begin = p.cu_q[b];
  const int Lq = p.cu_q[b + 1] - q_begin;
  const int k_begin = p.cu_k[b];
  int Lk = p.cu_k[b + 1] - k_begin;
  if (p.seqused_k) Lk = min(Lk, p.seqused_k[b]);
  const int wg_row0 = qb * BM;
  if (wg_row0 >= Lq) return;
  const int off = Lk - Lq;  // bottom-right alignment of the causal mask
  const int wg_last_row = min(wg_row0 + BM, Lq) - 1;
  int kmax = p.causal ? min(Lk, wg_last_row + off + 1) : Lk;
  if (kmax < 0) kmax = 0;
  const int n_tiles = (kmax + XBN - 1) / XBN;
  // Under the causal mask a wavefront's work grows with its rows' place in the block.  With one head per
  // workgroup the three wavefronts of SIMD s take row groups (s, 7 - s, 8 + s): about the same sum everywhere.
  // With four heads a group is a row group and its wavefronts are the heads.
  const int row_group = hl != 0 ? grp : (grp == 0 ? sub : (grp == 1 ? 7 - sub : 8 + sub));
  const int wave_row0 = wg_row0 + row_group * 32;
  const int wave_last_row = wave_row0 + 31;

  const T *qp = static_cast<const T *>(p.q) + (int64_t)q_begin * p.q_row + (int64_t)h * p.q_head;
  const T *kp = static_cast<const T *>(p.k) + (int64_t)k_begin * p.k_row + (int64_t)kvh * p.k_head;
  const T *vp = static_cast<const T *>(p.v) + (int64_t)k_begin * p.v_row + (int64_t)kvh * p.v_head;
  const int d_chunks = p.d / 8;

  // Q operands: lane (g, c) holds q[row c][16 ks + 8 g .. + 8] for every contraction step ks.
  vec8 qreg[KSTEPS];
  {
    const int row = min(wave_row0 + c, Lq - 1);
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ks++) {
      u32x4_t raw = {0u, 0u, 0u, 0u};
      const int ch = 2 * ks + g;
      if (ch < d_chunks) raw = *reinterpret_cast<const u32x4_t *>(qp + (int64_t)row * p.q_row + ch * 8);
      qreg[ks] = bit_cast<vec8>(raw);
    }
  }

  // ---- tile copies, global -> LDS, 1 KiB per instruction (lane l's 16 bytes land at M0 + 16 l) ----
  // K: the tile as two 16-token block images [16-byte run][token][8 elements], the paged cache's own layout:
  // the first product's operand reads then need neither padding nor swizzle, and their addresses differ by
  // constants.  Piece q is runs [4 pi .. 4 pi + 4) x 16 tokens of block r = q / KPB, pi = q % KPB: lane l fetches
  // run 4 pi + l / 16 of token l % 16 -- 64 bytes of each of 16 rows per instruction, which costs twice the
  // time per byte of fetching whole rows; with twelve wavefronts to a tile that is the cheaper side.  Runs past d
  // fetch the last real one (they meet the zeros of Q), keys past Lk the last real key (masked).
  constexpr int KPB = HDP / 32;                // pieces per 16-token block
  constexpr int KNP = 2 * KPB;                 // pieces per tile
  constexpr int KNPW = (KNP + NW - 1) / NW;    // ... per wavefront
  const int kd_tok = lane & 15, kd_run = lane >> 4;
  const uint32_t kd_off = (uint32_t)(((int64_t)kd_tok * p.k_row + kd_run * 8) * (int64_t)sizeof(T));
  const uint32_t kd_off_last =
      (uint32_t)(((int64_t)kd_tok * p.k_row + (min(4 * (KPB - 1) + kd_run, d_chunks - 1) - 4 * (KPB - 1)) * 8) * (int64_t)sizeof(T));
  auto k_copy = [&](int tile) {
    const int k0 = tile * XBN;
#pragma unroll
    for (int i = 0; i < KNPW; i++) {
      const int q = wave_u + NW * i;
      if (q < KNP) {
        const int r = q / KPB, pi = q % KPB;
        uint32_t loff = pi == KPB - 1 ? kd_off_last : kd_off;
        int64_t first = (int64_t)(k0 + 16 * r) * p.k_row + 32 * pi;  // elements from kp; uniform
        if (k0 + XBN > Lk) {
          int l2 = lane;
          asm volatile("" : "+v"(l2));  // (derived here, not hoisted: the loop has no registers to keep it in)
          const int key = min(k0 + 16 * r + (l2 & 15), Lk - 1);
          loff = (uint32_t)(((int64_t)(key - k0) * p.k_row + (min(4 * pi + (l2 >> 4), d_chunks - 1) - 4 * pi) * 8) * (int64_t)sizeof(T));
          first = (int64_t)k0 * p.k_row + 32 * pi;
        }
        const T *src = uniform_ptr(kp + first);
        const unsigned dst = (unsigned)__builtin_amdgcn_readfirstlane(
            (int)(lds0 + (unsigned)((tile % NBUF) * TILE_BYTES + r * (HDP * 16) * (int)sizeof(T) + pi * 1024)));
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                     :
                     : "s"(dst), "v"(loff), "s"(src)
                     : "memory", "m0");
      }
    }
  };
  // V: the tile's rows as they are, [key][HDP elements], in pieces of 64 16-byte runs in row order.  For the
  // transposing reads to be free of bank conflicts -- one covers 64 bytes of each of 4 consecutive rows --
  // run c of row r lies at run c ^ vswz(r) of its row where the row pitch is a multiple of 256 bytes; a lane's
  // place in LDS is given by the instruction, so it fetches the run that belongs there.
  constexpr int CPRV = HDP / 8;         // runs per row
  constexpr int VNP = XBN * CPRV / 64;  // pieces per tile
  constexpr int VNPW = (VNP + NW - 1) / NW;   // ... per wavefront
  auto vswz = [](int r) -> int { return HDP == 128 ? (r & 3) << 2 : (HDP == 64 ? ((r >> 1) & 1) << 2 : 0); };
  uint32_t vd_off[VNPW];
#pragma unroll
  for (int i = 0; i < VNPW; i++) {
    const int u = (wave + NW * i) * 64 + lane;  // the lane's run of the tile, in LDS order
    const int r = u / CPRV, pc = u % CPRV;
    vd_off[i] = (uint32_t)(((int64_t)r * p.v_row + min(pc ^ vswz(r), d_chunks - 1) * 8) * (int64_t)sizeof(T));
  }
  auto v_copy = [&](int tile) {
    const int k0 = tile * XBN;
    const T *src = uniform_ptr(vp + (int64_t)k0 * p.v_row);
#pragma unroll
    for (int i = 0; i < VNPW; i++) {
      const int q = wave_u + NW * i;
      if (q < VNP) {
        uint32_t loff = vd_off[i];
        if (k0 + XBN > Lk) {
          int l2 = lane;
          asm volatile("" : "+v"(l2));
          const int u = q * 64 + l2;
          const int r = u / CPRV, pc = u % CPRV;
          loff = (uint32_t)(((int64_t)(min(k0 + r, Lk - 1) - k0) * p.v_row + min(pc ^ vswz(r), d_chunks - 1) * 8) * (int64_t)sizeof(T));
        }
        const unsigned dst = (unsigned)__builtin_amdgcn_readfirstlane(
            (int)(lds0 + (unsigned)(V_REGION + (tile % NBUF) * TILE_BYTES + q * 1024)));
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                     :
                     : "s"(dst), "v"(loff), "s"(src)
                     : "memory", "m0");
      }
    }
  };
  // ---- operand reads ----
  // K images: MFMA row m = [a1 a0 g' b1 b0] of lane c reads token [g' a0 b1 b0] of block a1, so that the 8
  // scores a lane holds for one P.V step belong to 8 consecutive keys.  Contraction step ks lies 512 bytes
  // (two runs) further on.
  const unsigned k_lane_addr =
      lds0 + (unsigned)(((c >> 4) * (HDP * 16) + g * 128 + (((c >> 2) & 1) * 8 + ((c >> 3) & 1) * 4 + (c & 3)) * 8) * (int)sizeof(T));
  // V rows: the transposing read hands lane (g, rh, li) head element 16 rh + li of the 4 keys whose rows its
  // 16-lane group addresses, so two reads, at rows 8 g + li / 4 and 4 further, make the 8 keys of an operand.
  // Output tile dt lies dt 64-byte groups further along the row, before the swizzle: with it (a power-of-two
  // row) the address of tile 0 with bits flipped, without it that many bytes further on.
  unsigned vtr_addr0;  // byte address in LDS of the lane's 8 bytes for output tile 0, tile place 0, step 0
  {
    const int li = lane & 15, rh = (lane >> 4) & 1, r = 8 * g + (li >> 2);
    vtr_addr0 = lds0 + V_REGION + (unsigned)((r * HDP + ((2 * rh + ((li & 3) >> 1)) ^ vswz(r)) * 8 + 4 * (li & 1)) * (int)sizeof(T));
  }

  f32x16_t acc[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; dt++)
#pragma unroll
    for (int i = 0; i < 16; i++) acc[dt][i] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  const f32x16_t zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};

  // The M block: O^T += V^T(tv).P^T, then S^T(tk) = K(tk).Q^T, as one stream of MFMAs whose LDS operand reads
  // run three MFMAs ahead, across the seam between the two products and -- the first three -- across the
  // barrier in front of the block (DO_PV / DO_S: which of the two products there is).  P.V step n = (16-key step n / NDT, output tile n % NDT): consecutive MFMAs go to different
  // accumulators.  All reads are inline asm (the transposing read's builtin takes no offset, and a register
  // per address is too many), so the waits for them are written here too: entry e of the stream is waited
  // for with the count of the reads sent after it, two per P.V operand, one per K operand.
  constexpr int PV_STEPS = NDT * 2;
  constexpr int DEPTH = 3;  // operand reads run this many MFMAs ahead (2 and 4 measure the same)
  constexpr int NSLOT = DEPTH + 1;
  // operands in flight: entry e lives in slot e % NSLOT (a P.V operand as the two halves its reads return)
  u32x2_t lo[NSLOT], hi[NSLOT];
  u32x4_t kk[NSLOT];
  unsigned va[NDT], kb = 0;  // this block's V and K tiles: the lane's byte addresses in LDS (V: per output tile)
  auto m_read = [&](int e) {
    if (e < PV_STEPS) {
      constexpr int ROW4 = 4 * HDP * (int)sizeof(T);
      const int n = e;
      asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%3\n\tds_read_b64_tr_b16 %1, %2 offset:%4"
                   : "=&v"(lo[e % NSLOT]), "=&v"(hi[e % NSLOT])
                   : "v"(va[n % NDT]), "n"((n / NDT) * 4 * ROW4), "n"((n / NDT) * 4 * ROW4 + ROW4)
                   : "memory");
    } else {
      const int ks = e - PV_STEPS;
      asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(kk[e % NSLOT]) : "v"(kb), "n"(ks * 512) : "memory");
    }
  };
  // The first three operand reads of a block whose stream starts at entry e0; a wavefront sends them ahead of
  // the barrier in front of its M block (the tiles have been in LDS for a third of a period by then).
  auto m_begin = [&](int e0, int e1, int tv, int tk) {
    const unsigned vb = vtr_addr0 + (unsigned)((tv % NBUF) * TILE_BYTES);
#pragma unroll
    for (int dt = 0; dt < NDT; dt++) va[dt] = (HDP & (HDP - 1)) == 0 ? vb ^ (unsigned)(dt << 6) : vb + (unsigned)(dt << 6);
    kb = k_lane_addr + (unsigned)((tk % NBUF) * TILE_BYTES);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // nothing else is counted from here on
#pragma unroll
    for (int e = e0; e < e0 + DEPTH && e < e1; e++) m_read(e);
  };
  auto m_block = [&](auto do_pv, auto do_s, f32x16_t &s, vec8(&pk)[2]) {
    constexpr bool DO_PV = decltype(do_pv)::value, DO_S = decltype(do_s)::value;
    constexpr int E0 = DO_PV ? 0 : PV_STEPS;                      // first and
    constexpr int E1 = DO_S ? PV_STEPS + KSTEPS : PV_STEPS;       // one past the last entry of the stream
    auto reads_of = [](int e) { return e >= E1 ? 0 : (e < PV_STEPS ? 2 : 1); };
#pragma unroll
    for (int e = E0; e < E1; e++) {
      if (e + DEPTH < E1) m_read(e + DEPTH);
      int later = 0;  // reads sent after those of entry e
#pragma unroll
      for (int i = 1; i <= DEPTH; i++) later += reads_of(e + i);
      switch (later) {
        case 10: asm volatile("s_waitcnt lgkmcnt(10)" ::: "memory"); break;
        case 9: asm volatile("s_waitcnt lgkmcnt(9)" ::: "memory"); break;
        case 8: asm volatile("s_waitcnt lgkmcnt(8)" ::: "memory"); break;
        case 7: asm volatile("s_waitcnt lgkmcnt(7)" ::: "memory"); break;
        case 6: asm volatile("s_waitcnt lgkmcnt(6)" ::: "memory"); break;
        case 5: asm volatile("s_waitcnt lgkmcnt(5)" ::: "memory"); break;
        case 4: asm volatile("s_waitcnt lgkmcnt(4)" ::: "memory"); break;
        case 3: asm volatile("s_waitcnt lgkmcnt(3)" ::: "memory"); break;
        case 2: asm volatile("s_waitcnt lgkmcnt(2)" ::: "memory"); break;
        case 1: asm volatile("s_waitcnt lgkmcnt(1)" ::: "memory"); break;
        default: asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); break;
      }
      __builtin_amdgcn_sched_barrier(0);
      if (e < PV_STEPS) {
        const u32x4_t av = {lo[e % NSLOT][0], lo[e % NSLOT][1], hi[e % NSLOT][0], hi[e % NSLOT][1]};
        acc[e % NDT] = Mfma32<T>::run(bit_cast<vec8>(av), pk[e / NDT], acc[e % NDT]);
      } else {
        const int ks = e - PV_STEPS;
        s = Mfma32<T>::run(bit_cast<vec8>(kk[e % NSLOT]), qreg[ks], ks == 0 ? zero : s);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // V1: mask, row maximum with a lazily moved reference, rescaling.  Leaves the reference to subtract (msub)
  // and the start of the row sum (psum0) for V2.
  float msub = 0.f, psum0 = 0.f;
  auto softmax_max = [&](int tile, f32x16_t &s) {
    const int k0 = tile * XBN;
    const bool need_mask = (k0 + XBN > Lk) || (p.causal && k0 + XBN - 1 > wave_row0 + off);
    if (need_mask) {
      const int row = wave_row0 + c;
      int limit = p.causal ? row + off : Lk - 1;
      limit = min(limit, Lk - 1);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int key = k0 + ((i >> 3) & 1) * 16 + g * 8 + ((i >> 2) & 1) * 4 + (i & 3);
        if (key > limit) s[i] = -INFINITY;
      }
    }
    float mx = fmaxf(s[0], s[1]);
#pragma unroll
    for (int i = 2; i < 16; i += 2) mx = max3(mx, s[i], s[i + 1]);
    mx = max_across_halves(mx) * p.scale_log2;
    const bool grow = mx > m_run + p.rescale_thr;
    if (__builtin_expect(__any(grow), 0)) {
      const float m_new = grow ? mx : m_run;
      // exp2(-inf - finite) = 0 on a row's first keys; rows that do not grow keep 1 (their reference may
      // still be -inf, and -inf - -inf is not a number).
      const float alpha = grow ? fast_exp2(m_run - m_new) : 1.0f;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; dt++) acc[dt] *= alpha;
      m_run = m_new;
    }
    msub = m_run == -INFINITY ? 0.f : m_run;
    // The tile's largest probability enters the second product rounded to T; when one key dominates, that
    // rounding is the whole error of the row.  The same rounding goes into the normaliser (once per row:
    // lane group 0).  It is exactly zero whenever the maximum is the reference itself (p = 1).
    const float pmax = fast_exp2(mx - msub);
    psum0 = g == 0 ? to_float(from_float<T>(pmax)) - pmax : 0.f;
  };
  // V2: exponentials, row sum; leaves the B operands of the second product in pk.
  auto softmax_exp = [&](f32x16_t &s, vec8(&pk)[2]) {
    float psum = psum0;
#pragma unroll
    for (int v = 0; v < 16; v++) {
      const float e = fast_exp2(s[v] * p.scale_log2 - msub);
      psum += e;
      pk[v / 8][v % 8] = from_float<T>(e);
    }
    l_run += psum;
  };
  // ---- prologue: tiles 0 to 3 ----
#pragma unroll
  for (int t0 = 0; t0 < 4; t0++)
    if (t0 < n_tiles) {
      k_copy(t0);
      v_copy(t0);
    }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  // The compiler counts the loads of Q as outstanding until it sees a use of their registers and would
  // otherwise wait for them, with vmcnt(0), in front of the first MFMA of every iteration -- and so for the
  // copies just sent.  An empty statement that takes and returns the registers puts that wait here.
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ks++) asm volatile("" : "+v"(qreg[ks]));
  __syncthreads();
  f32x16_t s;
  vec8 pk[2];

  // S(0), by every group at once.
  const int t_end = wave_row0 >= Lq ? 0 : (p.causal ? min(n_tiles, max(wave_last_row + off, -1) / XBN + 1) : n_tiles);  // live tiles: [0, t_end)
  if (t_end > 0) {
    m_begin(PV_STEPS, PV_STEPS + KSTEPS, 0, 0);
    m_block(std::false_type{}, std::true_type{}, s, pk);
  }

  // ---- the tile loop ----
  // Per tile t a wavefront runs V1(t), V2(t), M(t) = P(t).V(t) and S(t+1), and ONE workgroup barrier -- group 0
  // behind V1, group 1 behind V2, group 2 behind M.  Between two barriers group 0 therefore runs V2 M V1, group
  // 1 M V1 V2 and group 2 V1 V2 M: on every SIMD the three M blocks follow one another, and where they touch,
  // the matrix pipe goes from one wavefront to the next without a barrier in between (two wavefronts that both
  // want it simply take turns).  Call the time between barrier x and barrier x + 1 interval x.  In interval x
  // groups 0 and 1 run M(x), group 2 runs M(x + 1) (and group 1 sends the first reads of M(x + 1) ahead): the
  // tiles read are V(x), V(x + 1), K(x + 1), K(x + 2).  In interval x every wavefront waits for its pieces
  // sent in interval x - 1 and sends its pieces of tile x + 4, into the places of tile x - 1, last read in
  // interval x - 1; they are complete behind barrier x + 2, and K(x + 4) is first read in interval x + 2.
  auto copy_duty = [&](int x) {
    if (x >= 0) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wavefront's pieces sent an interval ago
      if (x + 4 < n_tiles) {
        k_copy(x + 4);
        v_copy(x + 4);
      }
    }
  };
  // A barrier that does not wait for this wavefront's LDS reads: the first operands of the M block are on
  // their way across it.  (No wavefront writes LDS except through the copies, which have their own wait.)
  auto barrier_reads_in_flight = [&]() { asm volatile("s_barrier" ::: "memory"); };
  const int duty_lag = grp == 0 ? 0 : 1;  // V2(t) of groups 1 and 2 lies in interval t - 1
  auto iteration = [&](auto with_s, int t) {
    constexpr bool WITH_S = decltype(with_s)::value;
    softmax_max(t, s);
    if (grp == 0) lds_barrier();
    softmax_exp(s, pk);
    copy_duty(t - duty_lag);
    m_begin(0, WITH_S ? PV_STEPS + KSTEPS : PV_STEPS, t, t + 1);
    if (grp == 1) barrier_reads_in_flight();
    m_block(std::true_type{}, with_s, s, pk);
    if (grp == 2) lds_barrier();
  };
  asm volatile(".p2align 6");
  for (int t = 0; t < t_end - 1; t++) iteration(std::true_type{}, t);
  if (t_end > 0) iteration(std::false_type{}, t_end - 1);  // the wavefront's last tile: no scores to follow
  for (int t = t_end; t < n_tiles; t++) {  // tiles past this wavefront's diagonal: its share of the copies only
    if (grp == 0) lds_barrier();
    copy_duty(t - duty_lag);
    if (grp != 0) lds_barrier();
  }

  // ---- epilogue: normalise and store ----
  // The accumulators hold O^T: a lane has 4 consecutive head elements of one row per register quad.
  const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  const float inv = l_tot > 0.f ? 1.0f / l_tot : 0.f;
  int tid_e = tid;
  asm volatile("" : "+v"(tid_e));  // addresses derived here, after the loop, not carried through it
  const int lane_e = tid_e & 63;
  const int c_e = lane_e & 31, g_e = lane_e >> 5;
  const int row = wave_row0 + c_e;
  if (row < Lq) {
    if (p.out_f32) {
      float *op32 = static_cast<float *>(p.out) + (int64_t)(q_begin + row) * p.o_row + (int64_t)h * p.o_head;
#pragma unroll
      for (int dt = 0; dt < NDT; dt++)
#pragma unroll
        for (int a = 0; a < 4; a++) {
          const int dcol = dt * 32 + a * 8 + g_e * 4;
          if (dcol < p.d) {
            f32x4_t r;
#pragma unroll
            for (int i = 0; i < 4; i++) r[i] = acc[dt][a * 4 + i] * inv;
            *reinterpret_cast<f32x4_t *>(op32 + dcol) = r;
          }
        }
    } else {
      T *op = static_cast<T *>(p.out) + (int64_t)(q_begin + row) * p.o_row + (int64_t)h * p.o_head;
#pragma unroll
      for (int dt = 0; dt < NDT; dt++)
#pragma unroll
        for (int a = 0; a < 4; a++) {
          const int dcol = dt * 32 + a * 8 + g_e * 4;
          if (dcol < p.d) {
            T r[4];
#pragma unroll
            for (int i = 0; i < 4; i++) r[i] = from_float<T>(acc[dt][a * 4 + i] * inv);
            *reinterpret_cast<u32x2_t *>(op + dcol) = *reinterpret_cast<u32x2_t *>(r);
          }
        }
    }
    if (p.lse != nullptr && g_e == 0 && row < p.lse_pitch) {
      // Natural-log sum-exp of the scaled scores; +inf for a row without keys (flash_fwd_kernel.h:629-668).
      const float lse = l_tot > 0.f ? (m_run + __builtin_amdgcn_logf(l_tot)) * kLn2 : INFINITY;
      p.lse[((int64_t)b * p.Hq + h) * p.lse_pitch + row] = lse;
    }
  }
}

template <typename T, int HDP>
void launch_r3(PrefillParams p, hipStream_t stream) {
  static bool attr_set = false;  // benign race: setting twice is harmless
  auto kernel = prefill_varlen_r3_kernel<T, HDP>;
  constexpr size_t lds_bytes = (size_t)10 * XBN * HDP * sizeof(T);
  if (!attr_set) {
    HA_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)lds_bytes));
    attr_set = true;
  }
  // Four heads of a kv group per workgroup where the GQA ratio allows (all wavefronts of a group then sit at
  // the same rows and reach the diagonal together), else one head; the tuning switch prefill_wg_heads = 1
  // forces one head.
  const int hl = (p.G % 4 == 0 && tuning().prefill_wg_heads != 1) ? 2 : 0;
  p.wg_heads_log2 = hl;
  const int bm = (32 * NW) >> hl;
  p.n_qblocks = (p.max_q + bm - 1) / bm;
  const int64_t n_wg = (int64_t)p.n_qblocks * p.batch * (p.Hq >> hl);
  HA_CHECK(n_wg <= 0x7fffffff, "mha_varlen_fwd: too many workgroups");
  kernel<<<dim3((unsigned)n_wg), 64 * NW, lds_bytes, stream>>>(p);
  check_launch("mha_varlen_fwd");
}

template <typename T>
bool dispatch_r3(const PrefillParams &p, hipStream_t stream) {
  const int hdp = ((p.d + 31) / 32) * 32;
  switch (hdp) {
    case 32: launch_r3<T, 32>(p, stream); return true;
    case 64: launch_r3<T, 64>(p, stream); return true;
    case 96: launch_r3<T, 96>(p, stream); return true;
    case 128: launch_r3<T, 128>(p, stream); return true;
    default: return false;
  }
}

}  // namespace

// Never the library's own choice: measured on MI355X with the two kernels taking turns on a warm device (causal,
// 32 q / 8 kv heads, head size 128) the eight-wavefront kernel is ahead by 2 to 8 % from 64 x 512 to 8 x 3072 tokens
// and by 1 % at 8 x 4096; at head size 64 this one is ahead by 0 to 2 %.  (Timed one after the other, whichever
// kernel runs second looks 3 to 6 % better: the part raises its clock under matrix load for tens of milliseconds.)
// The kernel stays selectable (prefill_kernel = 4) and tested.
bool prefer_prefill_r3(const PrefillParams &) { return false; }

bool launch_prefill_r3(const PrefillParams &p, int dtype, hipStream_t stream) {
  // causal or unmasked only; a tile's 32 rows are addressed with unsigned 32-bit byte offsets
  const bool plain = p.win_left < 0 && p.win_right <= 0;
  const bool fits = p.k_row >= 0 && p.k_row < (1 << 23) && p.v_row >= 0 && p.v_row < (1 << 23);
  if (!plain || !fits || p.d > 128 || p.block_tables != nullptr) return false;
  return dtype == HIPATTN_F16 ? dispatch_r3<half_t>(p, stream) : dispatch_r3<bf16_t>(p, stream);
}

}  // namespace hipattn


