// Paged decode attention for gfx950: one query token per sequence attends to
// its whole context through the block table.  Replaces the reference's
// paged_attention_v1 / v2 (rllm/tch-cuda/kernels/vllm/attention/
// attention_kernels.cu:79-546) with a bandwidth-first design:
//
//  * two launch strategies over the same per-block-pair code: long steps are
//    one list of block pairs cut into equal contiguous ranges, one per
//    wavefront of a launch sized to the chip (paged_decode_flat_kernel); short
//    ones hand (sequence, kv head, context partition) items to workgroups whose
//    4 wavefronts take the partition's block pairs round-robin and merge once
//    through LDS (paged_decode_kernel);
//  * all query heads of a GQA group ride along as MFMA columns, so every K/V
//    byte is fetched once per kv head (the reference re-reads it per q head);
//  * the vLLM cache layout is consumed as it lies in memory: a K block
//    [d/8][16 tokens][8] read as 64 lanes x 16 B is exactly the A operand of
//    v_mfma_f32_16x16x32 (row = token, k = 8 head elements), and a V block
//    [d][16 tokens] read as 64 lanes x 8 B is the A operand of the P.V
//    product (row = head element, k = 4 tokens) -- every load instruction
//    covers one contiguous 1 KiB / 512 B run, nothing is shuffled or staged;
//  * split-K: ranges / partitions that do not cover a whole context write
//    (max, sum, unnormalised fp32 accumulator) and a small second kernel
//    merges them.
//
// Numerics: q.k products and all accumulation in fp32; probabilities are
// exp2((s - max) * log2e-folded scale), rounded to the cache dtype only as the
// MFMA operand of P.V; the normaliser is the fp32 sum of the unrounded
// probabilities.
#include <algorithm>
#include <atomic>

#include "paged_decode.h"
#include "paged_decode_generic.h"
#include "paged_decode_parts.h"
#include "workspace.h"

namespace hipattn {

namespace {

template <typename T, bool V2FMT, int BS>
void dispatch_head(const DecodeParams &p, int head_size, int64_t S, hipStream_t stream) {
  switch (head_size) {
    case 64: launch_decode<T, 64, V2FMT, BS>(p, S, stream); break;
    case 80: launch_decode<T, 80, V2FMT, BS>(p, S, stream); break;
    case 96: launch_decode<T, 96, V2FMT, BS>(p, S, stream); break;
    case 112: launch_decode<T, 112, V2FMT, BS>(p, S, stream); break;
    case 128: launch_decode<T, 128, V2FMT, BS>(p, S, stream); break;
    case 256: launch_decode<T, 256, V2FMT, BS>(p, S, stream); break;
    default: fail("paged_attention: unsupported head size %d (supported: 64, 80, 96, 112, 128, 256)", head_size);
  }
}

template <typename T, bool V2FMT>
void dispatch_block_size(const DecodeParams &p, int head_size, int block_size, int64_t S, hipStream_t stream) {
  switch (block_size) {
    case 8: dispatch_head<T, V2FMT, 8>(p, head_size, S, stream); break;
    case 16: dispatch_head<T, V2FMT, 16>(p, head_size, S, stream); break;
    case 32: dispatch_head<T, V2FMT, 32>(p, head_size, S, stream); break;
    default: fail("paged_attention: unsupported block size %d (supported: 8, 16, 32)", block_size);
  }
}

// The head sizes the MFMA kernels are built for (the reference's list, attention_kernels.cu:663-699).
bool mfma_head_size(int d) { return d == 64 || d == 80 || d == 96 || d == 112 || d == 128 || d == 256; }

// Which calls the plain fp32 kernel takes: fp32 caches, and 8- / 32-token blocks at head sizes outside
// that list (which it serves for any multiple of x up to 256, the MFMA kernels do not).
bool takes_generic_kernel(int dtype, int block_size, int head_size) {
  return dtype == HIPATTN_F32 || (block_size != kBlockSize && !mfma_head_size(head_size));
}

// Workgroups of the flat kernel that the device holds at once, per device (asked of the runtime once).
template <typename T, int HD>
int flat_resident_workgroups() {
  constexpr int kDevices = 64;
  static std::atomic<int> resident[kDevices];
  int dev = 0;
  HA_HIP(hipGetDevice(&dev));
  HA_CHECK(dev >= 0 && dev < kDevices, "device index %d out of range", dev);
  int r = resident[dev].load(std::memory_order_relaxed);
  if (r == 0) {
    int per_cu = 0;
    HA_HIP(hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, paged_decode_flat_kernel<T, HD, kBlockSize>, 256, 0));
    r = (per_cu > 0 ? per_cu : 1) * compute_units();
    resident[dev].store(r, std::memory_order_relaxed);
  }
  return r;
}

int flat_resident_workgroups(int dtype, int head_size) {
#define HA_RES(H) \
  case H: return dtype == HIPATTN_F16 ? flat_resident_workgroups<half_t, H>() : flat_resident_workgroups<bf16_t, H>()
  switch (head_size) {
    HA_RES(64);
    HA_RES(80);
    HA_RES(96);
    HA_RES(112);
    HA_RES(128);
    HA_RES(256);
    default: fail("paged_attention: unsupported head size %d (supported: 64, 80, 96, 112, 128, 256)", head_size);
  }
#undef HA_RES
}

// Partition length used by v1, in KV blocks: a multiple of 8 (one block pair per wavefront and round).  Long steps have some 2048
// workgroups: fewer fp32 partial results and start-ups per byte, and contexts of different lengths still even out.  With up to 128 (sequence,
// kv head) pairs partitions are longer: a workgroup's start-up and its partial result cost about what one more round does, so as long as
// leaves some 320 workgroups, one and a bit per compute unit, up to 32 blocks, and 64 where there are that many several times over (but 8
// where those are at most one to a compute unit, of 17 to 1023 blocks: heads of 256, us, 8 / 16 blocks, 8 / 2: 24 x 500 12.2 / 14.8, 8 x 1300 11.7 /
// 14.1, 12 x 1600 19.5 / 15.4; 8 / 1: 128 x 256 14.7 / 12.4, 2 x 16384 19.1 / 18.1).  A
// whole context of up to 64 blocks where that leaves as many: nothing to merge then (but where a few of them would be left for a
// last round, 17 x 630 at 32 kv heads 33.0 / 34.7).  Work is counted in blocks of 128 head elements.
// us, 2048 workgroups wanted / this rule, contexts of that length (uniform from a tenth of it), 32 / 8 heads of 128: 4 x 4096 19.0 / 16.4
// (18.9 / 14.9), 8 x 2048 18.5 / 16.4 (16.7 / 14.1), 8 x 4096 29.7 / 26.0 (25.9 / 22.0), 16 x 1600 25.0 / 22.7 (19.7 / 19.2), 16 x
// 2048 29.0 / 25.9 (23.5 / 20.3), 96 x 700 51.7 / 44.2 (36.7 / 31.5); 32 / 32 of 80: 2 x 4096 19.7 / 18.1 (18.7 / 16.5), 16 x 700 23.7 /
// 20.6 (19.1 / 16.3).  With more pairs: 24 x 1600 31.0 / 31.8 (22.9 / 24.5), 48 x 2048 from 204 on 45.0 / 47.8, 53 x 385..1541 42.6 / 44.6.
// 4528 calls (eight kinds of heads, 1 to 508 sequences of up to 256..131072 tokens): 0.966 of the time of the 2048; 2.5 % of them are more than
// 5 % slower, most of them 64 to 120 pairs of 500 to 1100 tokens that differ in length (12 x 70..700 12.6 / 11.6, 11 x 102..1024 13.7 / 12.3) -- what
// gains there (partitions rounded down) loses as much where lengths are alike.
// The tuning switch decode_part_blocks overrides the choice.
int choose_part_blocks(int64_t S, int Hkv, int col_groups, int head_size, int max_ctx) {
  const int forced = tuning().decode_part_blocks;
  if (forced >= 2 && forced <= 64) return forced + (forced & 1);
  const int64_t max_blocks = (max_ctx + kBlockSize - 1) / kBlockSize;
  const int64_t items = S * Hkv * col_groups;  // workgroups per partition index
  const int64_t work = items * max_blocks * (head_size < 64 ? 64 : head_size) / 128;
  const int64_t want_wgs = 2048;
  int64_t parts = (want_wgs + items - 1) / (items > 0 ? items : 1);
  if (parts < 1) parts = 1;
  int64_t pb = (max_blocks + parts - 1) / parts;
  if (max_blocks <= 64 && work > 32 * 320 && (items <= 512 || items % 512 == 0 || items % 512 >= 256))
    pb = 64;
  else if (items <= 128 && (items * ((max_blocks + 7) / 8) > 256 || max_blocks <= 16 || max_blocks >= 1024))
    pb = std::max(pb, work >= 65536 ? (int64_t)64 : std::min<int64_t>(32, (work + 319) / 320));
  pb = ((pb + 7) / 8) * 8;
  if (pb < 8) pb = 8;
  if (pb > 64) pb = 64;
  return (int)pb;
}

constexpr size_t kStaticScratchBytes = (size_t)16 << 20;  // of hipattn_paged_attention_v1_static

}  // namespace

DecodePlan plan_decode(int64_t S, int Hq, int Hkv, int head_size, int block_size, int dtype, int max_context_len) {
  DecodePlan pl;
  pl.generic = takes_generic_kernel(dtype, block_size, head_size);
  if (S <= 0 || Hq <= 0) return pl;
  if (pl.generic) {
    int64_t P = ((int64_t)max_context_len + kGenericPartTokens - 1) / kGenericPartTokens;
    if (P < 1) P = 1;
    HA_CHECK(P <= 65535, "paged_attention: max_context_len %d is too long", max_context_len);
    pl.num_parts = (int)P;
    if (P > 1) pl.slots = (size_t)S * Hq * P;
  } else {
    const int G = Hq / Hkv, col_groups = (G + 15) / 16;
    pl.flat = use_flat_split(S, Hkv * col_groups, max_context_len);
    if (pl.flat) {
      // What the device holds at once, but no more than gives every wavefront two units of the largest
      // possible step.
      int64_t wgs = tuning().decode_flat_wgs > 0 ? tuning().decode_flat_wgs : flat_resident_workgroups(dtype, head_size);
      const int64_t cap = (flat_units(S, Hkv * col_groups, max_context_len) + 7) / 8;
      if (wgs > cap) wgs = cap;
      pl.flat_wgs = (int)(wgs < 1 ? 1 : wgs);
      pl.flat_scratch = flat_scratch(S, G, head_size, pl.flat_wgs);
      pl.bytes = pl.flat_scratch.bytes;
      return pl;
    } else {
      pl.part_blocks = choose_part_blocks(S, Hkv, col_groups, head_size, max_context_len);
      const int64_t max_blocks = ((int64_t)max_context_len + kBlockSize - 1) / kBlockSize;
      // A whole context per workgroup of eight wavefronts instead of partitions and their merge.  The merge costs about 3 us;
      // each block pair a wavefront takes after its first costs 2.4 us where only a few compute units run (head size 128; 1.5
      // at 64), and nothing where the launch is bound by memory.  So: contexts of one pair per wavefront, two pairs of small
      // heads, and whatever fits one lane-held slice of the table once the workgroups share the memory (128 of them; 192 for
      // the longest contexts of larger heads, which otherwise end last and alone).  Beyond two such workgroups per compute unit
      // they gain nothing, and their last round loses, but at small heads, which keep winning up to 1024, and but where the partitions'
      // results would not fit the built-in array (sixteen query heads per kv head, a thousand contexts), so that the entry point
      // that uses it can serve them.  us, partitions / one workgroup, all contexts of that length (lengths uniform up to it):
      //   32 q / 8 kv x 128: 1 x 256 8.5 / 6.8, 1 x 512 8.3 / 9.7, 1 x 700 9.2 / 11.7, 16 x 512 13.6 / 12.5 (11.6 / 10.9), 16 x 1024 20.3 /
      //   20.1 (15.1 / 17.1), 24 x 1024 26.2 / 22.5 (20.2 / 18.5), 40 x 512 23.0 / 24.7 (18.4 / 15.8), 40 x 1024 36.7 / 40.9 (26.2 / 23.6),
      //   64 x 512 30.2 / 27.6, 72 x 512 35.6 / 38.6 (25.8 / 24.7), 104 x 512 47.4 / 51.5 (32.6 / 34.3); 32 / 32 x 80: 1 x 512 8.1 / 7.7,
      //   4 x 512 9.9 / 8.4, 1 x 1023 8.7 / 11.2, 26 x 200 19.2 / 21.1 (15.0 / 16.9); 16 / 2 x 64: 1 x 512 7.2 / 6.4, 16 x 1023 8.5 / 9.6,
      //   64 x 1024 14.0 / 12.0 (12.8 / 10.7), 508 x 512 33.6 / 31.2 (24.5 / 22.1).
      const int64_t wgs = S * Hkv * col_groups;
      const bool small = head_size <= 64;
      const bool one_wg = max_blocks <= 16 || (max_blocks <= 32 && small) || (max_blocks <= 64 && wgs >= (small || max_blocks <= 48 ? 128 : 192));
      const size_t partials = (size_t)S * Hq * ((max_blocks + pl.part_blocks - 1) / pl.part_blocks) * (head_size + 2) * sizeof(float);
      const int64_t most_wgs = small || partials > kStaticScratchBytes ? 1023 : 512;
      if (tuning().decode_part_blocks <= 0 && head_size <= 128 && max_blocks > pl.part_blocks && wgs <= most_wgs && one_wg) {
        pl.part_blocks = 64;
        // (beyond one such workgroup per compute unit the usual four wavefronts do: 64 x 700 34.5 / 31.9, 96 x 700 51.7 / 44.2)
        if (small || wgs <= 256) pl.waves = 8;
      } else if (tuning().decode_part_blocks <= 0 && head_size > 64 && head_size < 128 && max_blocks > 32 && max_blocks <= pl.part_blocks &&
                 wgs <= 256 && one_wg) {
        // Contexts that are whole already.  With heads of 128 four wavefronts do there too (32 x 1024 24.9 / 24.1), with smaller ones they lose
        // where lengths differ: us, eight / four, 12 / 4 x 112, 48 x 102..1024 16.3 / 18.1 (all 1024: 19.0 / 19.8), 32 / 4 x 96, 64 x 102..1024
        // 15.4 / 16.8 (20.4 / 19.9).
        pl.waves = 8;
      }
      int64_t P = (max_blocks + pl.part_blocks - 1) / pl.part_blocks;
      if (P < 1) P = 1;
      pl.num_parts = (int)P;
      if (P > 1) pl.slots = (size_t)S * Hq * P;
    }
  }
  pl.bytes = pl.slots * (size_t)(head_size + 2) * sizeof(float);
  return pl;
}

namespace {

// Where a call's scratch memory comes from.
struct Scratch {
  enum Kind { LIBRARY, CALLER, STATIC } kind = LIBRARY;
  void *ptr = nullptr;  // CALLER
  int64_t bytes = 0;    // CALLER
};

// The scratch array of hipattn_paged_attention_v1_static, the entry point that allocates nothing: device
// memory that exists from the moment the code object is loaded, one copy per device.  In host code the
// array's name is only a handle for hipGetSymbolAddress; kernels get the address that call returns.
static __device__ __align__(256) unsigned char scratch[kStaticScratchBytes];

// The address of `scratch` on the current device, asked of the runtime once per device.
char *static_scratch() {
  constexpr int kDevices = 64;
  static std::atomic<char *> address[kDevices];
  int dev = 0;
  HA_HIP(hipGetDevice(&dev));
  HA_CHECK(dev >= 0 && dev < kDevices, "device index %d out of range", dev);
  char *ptr = address[dev].load(std::memory_order_acquire);
  if (ptr == nullptr) {
    HA_HIP(hipGetSymbolAddress(reinterpret_cast<void **>(&ptr), HIP_SYMBOL(scratch)));
    HA_CHECK(ptr != nullptr, "hipGetSymbolAddress returned no address for the scratch array");
    address[dev].store(ptr, std::memory_order_release);
  }
  return ptr;
}

// The scratch memory of one call (pl.bytes of it; nothing in it outlives the call), the library's held for it.
HeldWorkspace scratch_memory(const Scratch &from, const DecodePlan &pl, hipStream_t stream, const char *op) {
  HeldWorkspace ws;
  if (pl.bytes == 0) return ws;
  switch (from.kind) {
    case Scratch::CALLER:
      HA_CHECK(from.ptr != nullptr, "%s: workspace is NULL but %zu bytes are needed", op, pl.bytes);
      HA_CHECK((reinterpret_cast<uintptr_t>(from.ptr) & 255) == 0, "%s: workspace must be 256-byte aligned", op);
      HA_CHECK(from.bytes >= 0 && (size_t)from.bytes >= pl.bytes,
               "%s: workspace of %lld bytes is too small, %zu are needed (hipattn_paged_attention_workspace_size)", op,
               (long long)from.bytes, pl.bytes);
      ws.ptr = from.ptr;
      return ws;
    case Scratch::STATIC:
      HA_CHECK(pl.bytes <= kStaticScratchBytes,
               "%s: this call needs %zu bytes of scratch memory, more than the %zu bytes of the built-in array; use "
               "hipattn_paged_attention_v1 or hipattn_paged_attention_v1_ws for it",
               op, pl.bytes, kStaticScratchBytes);
      ws.ptr = static_scratch();
      return ws;
    default:
      return library_workspace(WS_PAGED_ATTENTION, pl.bytes, stream);
  }
}

template <typename T>
void dispatch_head_flat(const DecodeParams &p, int head_size, int block_size, const DecodePlan &pl, char *ws,
                        hipStream_t stream) {
  switch (head_size) {
    case 64: launch_decode_flat<T, 64>(p, pl, block_size, ws, stream); break;
    case 80: launch_decode_flat<T, 80>(p, pl, block_size, ws, stream); break;
    case 96: launch_decode_flat<T, 96>(p, pl, block_size, ws, stream); break;
    case 112: launch_decode_flat<T, 112>(p, pl, block_size, ws, stream); break;
    case 128: launch_decode_flat<T, 128>(p, pl, block_size, ws, stream); break;
    case 256: launch_decode_flat<T, 256>(p, pl, block_size, ws, stream); break;
    default: fail("paged_attention: unsupported head size %d (supported: 64, 80, 96, 112, 128, 256)", head_size);
  }
}

GenericDecodeParams generic_params(const DecodeParams &p, int head_size, int block_size, float scale) {
  GenericDecodeParams g;
  memset(&g, 0, sizeof g);
  g.q = p.q;
  g.q_stride = p.q_stride;
  g.kc = p.kc;
  g.vc = p.vc;
  g.k_block_stride = p.k_block_stride;
  g.k_head_stride = p.k_head_stride;
  g.v_block_stride = p.v_block_stride;
  g.v_head_stride = p.v_head_stride;
  g.num_blocks = p.num_blocks;
  g.block_tables = p.block_tables;
  g.table_stride = p.max_blocks;
  g.table_cols = p.table_cols;
  g.context_lens = p.context_lens;
  g.alibi = p.alibi;
  g.scale = scale;
  g.Hq = p.Hq;
  g.G = p.G;
  g.head_size = head_size;
  g.block_size = block_size;
  g.num_seqs = p.num_seqs;
  g.max_ctx = p.max_ctx;
  g.out = p.out;
  g.out_stride = p.out_stride;
  return g;
}

}  // namespace

// (the names of the arguments in its messages are those of hipattn_paged_attention_v1)
bool decode_params(const DecodeCall &c, hipattn_tensor *out, DecodeParams &p) {
  const hipattn_tensor *query = c.query, *key_cache = c.key_cache, *value_cache = c.value_cache, *block_tables = c.block_tables,
                       *context_lens = c.context_lens, *alibi = c.alibi;
  const int num_kv_heads = c.num_kv_heads, block_size = c.block_size, max_context_len = c.max_context_len;
  const float scale = c.scale;
  const char *op = c.op;
  check_tensor(out, "out", 3);
  check_tensor(query, "query", 3);
  check_tensor(key_cache, "key_cache", 5);
  check_tensor(value_cache, "value_cache", 4);
  check_tensor(block_tables, "block_tables", 2);
  check_tensor(context_lens, "context_lens", 1);
  HA_CHECK(is_float_dtype(query->dtype), "%s: unsupported data type %s (supported: f16, bf16, f32)", op,
           dtype_name(query->dtype));
  HA_CHECK(out->dtype == query->dtype && key_cache->dtype == query->dtype && value_cache->dtype == query->dtype,
           "%s: out, query and caches must share a dtype", op);
  HA_CHECK(block_tables->dtype == HIPATTN_I32 && context_lens->dtype == HIPATTN_I32,
           "%s: block_tables and context_lens must be int32", op);
  HA_CHECK(block_size == 8 || block_size == 16 || block_size == 32,
           "%s: unsupported block size %d (supported: 8, 16, 32)", op, block_size);
  // The MFMA kernels take the 2-byte types at the reference's head sizes; fp32 caches go to the fp32-FMA kernel.
  const bool generic = takes_generic_kernel(query->dtype, block_size, (int)query->sizes[2]);
  const int x = 16 / dtype_size(query->dtype);
  const int64_t S = query->sizes[0];
  const int Hq = (int)query->sizes[1];
  const int hd = (int)query->sizes[2];
  HA_CHECK(out->sizes[0] == S && out->sizes[1] == Hq && out->sizes[2] == hd, "%s: out and query shapes differ", op);
  HA_CHECK(num_kv_heads > 0 && Hq % num_kv_heads == 0, "%s: %d query heads not divisible by %d kv heads", op, Hq,
           num_kv_heads);
  HA_CHECK(key_cache->sizes[1] == num_kv_heads && key_cache->sizes[2] * key_cache->sizes[4] == hd &&
               key_cache->sizes[3] == block_size && key_cache->sizes[4] == x,
           "%s: key_cache shape does not match [nb, %d, %d/%d, %d, %d]", op, num_kv_heads, hd, x, block_size, x);
  HA_CHECK(value_cache->sizes[0] == key_cache->sizes[0] && value_cache->sizes[1] == num_kv_heads &&
               value_cache->sizes[2] == hd && value_cache->sizes[3] == block_size,
           "%s: value_cache shape does not match [nb, %d, %d, %d]", op, num_kv_heads, hd, block_size);
  HA_CHECK(key_cache->strides[4] == 1 && key_cache->strides[3] == x && key_cache->strides[2] == x * block_size &&
               value_cache->strides[3] == 1 && value_cache->strides[2] == block_size,
           "%s: cache inner dims must be contiguous", op);
  HA_CHECK(key_cache->strides[0] % x == 0 && key_cache->strides[1] % x == 0 &&
               (reinterpret_cast<uintptr_t>(key_cache->data) & 15) == 0,
           "%s: key_cache blocks and heads must keep 16-byte alignment", op);
  HA_CHECK((hd <= 1 || (query->strides[2] == 1 && out->strides[2] == 1)) && query->strides[1] == hd &&
               out->strides[1] == hd,
           "%s: query/out heads must be contiguous", op);
  if (!generic) {
    HA_CHECK(value_cache->strides[0] % 4 == 0 && value_cache->strides[1] % 4 == 0,
             "%s: cache block/head strides must keep 16-byte alignment", op);
    HA_CHECK((reinterpret_cast<uintptr_t>(value_cache->data) & 15) == 0 &&
                 (reinterpret_cast<uintptr_t>(query->data) & 15) == 0 && (reinterpret_cast<uintptr_t>(out->data) & 7) == 0,
             "%s: tensors must be 16-byte aligned", op);
    HA_CHECK(query->strides[0] % 8 == 0 && out->strides[0] % 4 == 0,
             "%s: query/out need an aligned row stride", op);
  }
  HA_CHECK(block_tables->sizes[0] == S && context_lens->sizes[0] == S, "%s: block_tables/context_lens need %lld rows", op,
           (long long)S);
  check_contiguous(context_lens, "context_lens");
  HA_CHECK(block_tables->sizes[1] <= 1 || block_tables->strides[1] == 1, "%s: block_tables rows must be contiguous", op);
  HA_CHECK(max_context_len >= 0, "%s: negative max_context_len", op);
  HA_CHECK(((int64_t)max_context_len + block_size - 1) / block_size <= block_tables->sizes[1],
           "%s: max_context_len %d needs more than the %lld block-table columns", op, max_context_len,
           (long long)block_tables->sizes[1]);
  if (alibi) {
    check_tensor(alibi, "alibi_slopes", 1);
    HA_CHECK(alibi->dtype == HIPATTN_F32 && alibi->sizes[0] == Hq, "%s: alibi_slopes must be f32 [%d]", op, Hq);
    check_contiguous(alibi, "alibi_slopes");
    check_data(alibi, "alibi_slopes");
  }
  if (S == 0 || Hq == 0) return false;
  HA_CHECK(S <= 65535, "%s: at most 65535 sequences per call", op);
  HA_CHECK(key_cache->sizes[0] > 0, "%s: the cache has no blocks", op);
  check_data(out, "out");
  check_data(query, "query");
  check_data(key_cache, "key_cache");
  check_data(value_cache, "value_cache");
  check_data(block_tables, "block_tables");
  check_data(context_lens, "context_lens");
  memset(&p, 0, sizeof p);
  p.q = query->data;
  p.q_stride = query->strides[0];
  p.kc = key_cache->data;
  p.vc = value_cache->data;
  p.k_block_stride = key_cache->strides[0];
  p.k_head_stride = key_cache->strides[1];
  p.v_block_stride = value_cache->strides[0];
  p.v_head_stride = value_cache->strides[1];
  p.num_blocks = key_cache->sizes[0];
  p.block_tables = static_cast<const int32_t *>(block_tables->data);
  p.max_blocks = block_tables->strides[0];
  p.table_cols = (int)block_tables->sizes[1];
  p.context_lens = static_cast<const int32_t *>(context_lens->data);
  p.alibi = alibi ? static_cast<const float *>(alibi->data) : nullptr;
  p.scale_log2 = scale * kLog2e;
  p.Hq = Hq;
  p.Hkv = num_kv_heads;
  p.G = Hq / num_kv_heads;
  p.col_groups = (p.G + 15) / 16;
  p.num_seqs = (int)S;
  p.out = out->data;
  p.out_stride = out->strides[0];
  // A context length beyond max_context_len (which sized the launch and the scratch memory) or beyond
  // what a table row describes is cut there, in every kernel alike.
  p.max_ctx = (int)std::min<int64_t>(max_context_len, block_tables->sizes[1] * block_size);
  return true;
}

size_t decode_scratch_bytes(const DecodeCall &c) {
  return plan_decode(c.query->sizes[0], (int)c.query->sizes[1], c.num_kv_heads, (int)c.query->sizes[2], c.block_size, c.query->dtype,
                     c.max_context_len)
      .bytes;
}

FlatScratch flat_scratch(int64_t S, int G, int head_size, int workgroups) {
  FlatScratch f;
  f.cols = G < 16 ? G : 16;
  f.prefix_bytes = (((size_t)S + 1) * sizeof(int) + 255) & ~(size_t)255;
  f.slots = (size_t)2 * workgroups * 4 * f.cols;
  f.bytes = f.prefix_bytes + f.slots * (size_t)(head_size + 2) * sizeof(float);
  return f;
}

void flat_scratch_set(DecodeParams &p, const FlatScratch &f, int workgroups, int head_size, char *ws) {
  p.flat_waves = workgroups * 4;
  p.flat_cols = f.cols;
  p.flat_prefix = reinterpret_cast<int *>(ws);
  p.ws_acc = reinterpret_cast<float *>(ws + f.prefix_bytes);
  p.ws_m = p.ws_acc + f.slots * head_size;
  p.ws_l = p.ws_m + f.slots;
}

int64_t flat_units(int64_t S, int heads, int max_context_len) {
  return S * heads * (((int64_t)max_context_len + 2 * kBlockSize - 1) / (2 * kBlockSize));
}

bool flat_split_counts(int64_t S, int heads, int max_context_len) {
  return S <= kFlatMaxSeqs && max_context_len > 0 && flat_units(S, heads, max_context_len) < (int64_t)1 << 30;
}

// v1 takes the flat split for long steps: measured on MI355X it wins a few
// percent once every wavefront of the launch has tens of block pairs to
// stream, and loses to the partitioned launch (whose many short workgroups
// hide the per-segment load chains behind each other) on short contexts or
// small batches.  Its bookkeeping also needs the sequence table to fit in LDS
// and unit indices in 32 bits.  The tuning switch decode_flat forces the choice.
bool use_flat_split(int64_t S, int hk, int max_context_len) {
  if (!flat_split_counts(S, hk, max_context_len)) return false;
  if (tuning().decode_flat >= 0) return tuning().decode_flat != 0;
  return max_context_len >= 1024 && flat_units(S, hk, max_context_len) >= 32 * 2048;
}

int compute_units() {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices];
  int dev = 0;
  HA_HIP(hipGetDevice(&dev));
  HA_CHECK(dev >= 0 && dev < kDevices, "device index %d out of range", dev);
  int cus = known[dev].load(std::memory_order_relaxed);
  if (cus == 0) {
    HA_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    if (cus < 1) cus = 1;
    known[dev].store(cus, std::memory_order_relaxed);
  }
  return cus;
}

namespace {

void paged_attention_impl(hipattn_tensor *out, hipattn_tensor *exp_sums, hipattn_tensor *max_logits,
                          hipattn_tensor *tmp_out, const hipattn_tensor *query, const hipattn_tensor *key_cache,
                          const hipattn_tensor *value_cache, int num_kv_heads, float scale,
                          const hipattn_tensor *block_tables, const hipattn_tensor *context_lens, int block_size,
                          int max_context_len, const hipattn_tensor *alibi, bool v2, const Scratch &scratch_from,
                          const char *op, void *stream_arg) {
  DecodeParams p;
  const DecodeCall call{query, key_cache, value_cache, num_kv_heads, scale, block_tables, context_lens, block_size, max_context_len, alibi, op};
  if (!decode_params(call, out, p)) return;
  const int64_t S = query->sizes[0];
  const int Hq = (int)query->sizes[1], hd = (int)query->sizes[2];
  // The MFMA kernels take the 2-byte types at the reference's head sizes; fp32 caches go to the fp32-FMA kernel.
  const bool generic = takes_generic_kernel(query->dtype, block_size, hd);
  hipStream_t stream = resolve_stream(stream_arg);
  HeldWorkspace held;  // over all launches
  if (v2) {
    check_tensor(exp_sums, "exp_sums", 3);
    check_tensor(max_logits, "max_logits", 3);
    check_tensor(tmp_out, "tmp_out", 4);
    const int64_t P = exp_sums->sizes[2];
    HA_CHECK(P >= 1, "%s: exp_sums has no partitions", op);
    HA_CHECK(exp_sums->dtype == HIPATTN_F32 && max_logits->dtype == HIPATTN_F32 && tmp_out->dtype == query->dtype,
             "%s: exp_sums/max_logits must be f32 and tmp_out the cache dtype", op);
    HA_CHECK(exp_sums->sizes[0] == S && exp_sums->sizes[1] == Hq && max_logits->sizes[0] == S &&
                 max_logits->sizes[1] == Hq && max_logits->sizes[2] == P && tmp_out->sizes[0] == S &&
                 tmp_out->sizes[1] == Hq && tmp_out->sizes[2] == P && tmp_out->sizes[3] == hd,
             "%s: workspace shapes must be [S,Hq,P], [S,Hq,P], [S,Hq,P,d]", op);
    check_contiguous(exp_sums, "exp_sums");
    check_contiguous(max_logits, "max_logits");
    check_contiguous(tmp_out, "tmp_out");
    check_data(exp_sums, "exp_sums");
    check_data(max_logits, "max_logits");
    check_data(tmp_out, "tmp_out");
    HA_CHECK((reinterpret_cast<uintptr_t>(tmp_out->data) & 7) == 0, "%s: tmp_out must be 8-byte aligned", op);
    if (generic) {
      GenericDecodeParams g = generic_params(p, hd, block_size, scale);
      g.num_parts = (int)P;
      g.ws_l = static_cast<float *>(exp_sums->data);
      g.ws_m = static_cast<float *>(max_logits->data);
      g.tmp_out = tmp_out->data;
      paged_decode_generic(g, query->dtype, true, max_context_len, (int)P, nullptr, stream);
      return;
    }
    // partition length in runs of 16 tokens, whatever the cache's block size
    const int64_t max_runs = ((int64_t)max_context_len + kBlockSize - 1) / kBlockSize;
    int64_t pb = (max_runs + P - 1) / P;
    if (pb < 2) pb = 2;
    pb += pb & 1;
    HA_CHECK(pb <= 64, "%s: %lld partitions are too few for max_context_len %d (at most 1024 tokens each)", op,
             (long long)P, max_context_len);
    p.part_blocks = (int)pb;
    p.num_parts = (int)P;
    p.ws_l = static_cast<float *>(exp_sums->data);
    p.ws_m = static_cast<float *>(max_logits->data);
    p.tmp_out = tmp_out->data;
  } else {
    const DecodePlan pl = plan_decode(S, Hq, num_kv_heads, hd, block_size, query->dtype, max_context_len);
    held = scratch_memory(scratch_from, pl, stream, op);
    char *ws = static_cast<char *>(held.ptr);
    if (pl.generic) {
      paged_decode_generic(generic_params(p, hd, block_size, scale), query->dtype, false, max_context_len, pl.num_parts,
                           reinterpret_cast<float *>(ws), stream);
      return;
    }
    if (pl.flat) {
      if (query->dtype == HIPATTN_F16)
        dispatch_head_flat<half_t>(p, hd, block_size, pl, ws, stream);
      else
        dispatch_head_flat<bf16_t>(p, hd, block_size, pl, ws, stream);
      return;
    }
    p.part_blocks = pl.part_blocks;
    p.num_parts = pl.num_parts;
    p.waves = pl.waves;
    if (pl.num_parts > 1) {
      p.ws_acc = reinterpret_cast<float *>(ws);
      p.ws_m = p.ws_acc + pl.slots * hd;
      p.ws_l = p.ws_m + pl.slots;
    }
  }
#define HA_PA(TT)                                                          \
  if (v2) dispatch_block_size<TT, true>(p, hd, block_size, S, stream);     \
  else dispatch_block_size<TT, false>(p, hd, block_size, S, stream)
  if (query->dtype == HIPATTN_F16) {
    HA_PA(half_t);
  } else {
    HA_PA(bf16_t);
  }
#undef HA_PA
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" char *hipattn_paged_attention_v1(hipattn_tensor *out, const hipattn_tensor *query,
                                            const hipattn_tensor *key_cache, const hipattn_tensor *value_cache,
                                            int num_kv_heads, float scale, const hipattn_tensor *block_tables,
                                            const hipattn_tensor *context_lens, int block_size, int max_context_len,
                                            const hipattn_tensor *alibi_slopes, void *stream) {
  HA_PROTECT(paged_attention_impl(out, nullptr, nullptr, nullptr, query, key_cache, value_cache, num_kv_heads, scale,
                                  block_tables, context_lens, block_size, max_context_len, alibi_slopes, false, Scratch(),
                                  "paged_attention_v1", stream));
}

extern "C" char *hipattn_paged_attention_v1_ws(hipattn_tensor *out, const hipattn_tensor *query,
                                               const hipattn_tensor *key_cache, const hipattn_tensor *value_cache,
                                               int num_kv_heads, float scale, const hipattn_tensor *block_tables,
                                               const hipattn_tensor *context_lens, int block_size, int max_context_len,
                                               const hipattn_tensor *alibi_slopes, void *workspace,
                                               int64_t workspace_bytes, void *stream) {
  HA_PROTECT({
    Scratch from;
    from.kind = Scratch::CALLER;
    from.ptr = workspace;
    from.bytes = workspace_bytes;
    paged_attention_impl(out, nullptr, nullptr, nullptr, query, key_cache, value_cache, num_kv_heads, scale, block_tables,
                         context_lens, block_size, max_context_len, alibi_slopes, false, from, "paged_attention_v1_ws",
                         stream);
  });
}

extern "C" char *hipattn_paged_attention_v1_static(hipattn_tensor *out, const hipattn_tensor *query,
                                                   const hipattn_tensor *key_cache, const hipattn_tensor *value_cache,
                                                   int num_kv_heads, float scale, const hipattn_tensor *block_tables,
                                                   const hipattn_tensor *context_lens, int block_size,
                                                   int max_context_len, const hipattn_tensor *alibi_slopes, void *stream) {
  HA_PROTECT({
    Scratch from;
    from.kind = Scratch::STATIC;
    paged_attention_impl(out, nullptr, nullptr, nullptr, query, key_cache, value_cache, num_kv_heads, scale, block_tables,
                         context_lens, block_size, max_context_len, alibi_slopes, false, from, "paged_attention_v1_static",
                         stream);
  });
}

extern "C" char *hipattn_init(void) {
  HA_PROTECT({
    (void)static_scratch();
    for (int dtype : {HIPATTN_F16, HIPATTN_BF16})
      for (int hd : {64, 80, 96, 112, 128, 256}) (void)flat_resident_workgroups(dtype, hd);
  });
}

extern "C" char *hipattn_paged_attention_workspace_size(int64_t num_seqs, int num_heads, int num_kv_heads, int head_size,
                                                        int block_size, int max_context_len, int32_t dtype,
                                                        int64_t *bytes) {
  HA_PROTECT({
    HA_CHECK(bytes != nullptr, "paged_attention_workspace_size: bytes is NULL");
    HA_CHECK(num_seqs >= 0 && num_heads >= 0 && max_context_len >= 0, "paged_attention_workspace_size: negative size");
    HA_CHECK(is_float_dtype(dtype), "paged_attention_workspace_size: unsupported data type %s", dtype_name(dtype));
    HA_CHECK(block_size == 8 || block_size == 16 || block_size == 32,
             "paged_attention_workspace_size: unsupported block size %d (supported: 8, 16, 32)", block_size);
    HA_CHECK(num_kv_heads > 0 && num_heads % num_kv_heads == 0,
             "paged_attention_workspace_size: %d query heads not divisible by %d kv heads", num_heads, num_kv_heads);
    *bytes = (int64_t)plan_decode(num_seqs, num_heads, num_kv_heads, head_size, block_size, dtype, max_context_len).bytes;
  });
}

extern "C" char *hipattn_paged_attention_v2(hipattn_tensor *out, hipattn_tensor *exp_sums, hipattn_tensor *max_logits,
                                            hipattn_tensor *tmp_out, const hipattn_tensor *query,
                                            const hipattn_tensor *key_cache, const hipattn_tensor *value_cache,
                                            int num_kv_heads, float scale, const hipattn_tensor *block_tables,
                                            const hipattn_tensor *context_lens, int block_size, int max_context_len,
                                            const hipattn_tensor *alibi_slopes, void *stream) {
  HA_PROTECT(paged_attention_impl(out, exp_sums, max_logits, tmp_out, query, key_cache, value_cache, num_kv_heads, scale,
                                  block_tables, context_lens, block_size, max_context_len, alibi_slopes, true, Scratch(),
                                  "paged_attention_v2", stream));
}
