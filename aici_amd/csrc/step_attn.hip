// The attention of an engine step that holds both kinds of rows -- chunks of prompts over what is cached already, and sequences that decode
// a token each -- as one launch and the merge behind it, instead of a prefill launch, a decode launch and its merge one after the
// other (rllm/rllm-cuda/src/llm/mod.rs:318-354 calls them in turn).
//
// What bounds the two apart: prefill the vector unit and, with few workgroups, the longest row block (some 1.2 us per tile of 64 keys, one
// after the other: 3 new tokens over 3000 cached ones take as long as 128 of them); decode the memory.  Here a workgroup of decode rows
// (the flat split: equal shares, whatever the contexts) sits on every compute unit beside one of prefill, in four wavefronts each,
// and a row block's keys go to several workgroups where the launch has places for them (plan_step).  Both bodies are those of
// the launches by themselves; registers and LDS are the larger of the two, which leaves two workgroups to a compute unit.
//
// us without the cache write, by the gathered copy / from the cache in separate launches / here (query, kv heads x head size):
//   120 decode rows of 1k..8k tokens + 4 x 512 new tokens over 0..3072, 32 / 32 x 80    1012 / 983 / 920 (the decode rows alone: 897)
//   24 of 128..4096 + 4 x 17..512 over 0..1024, 32 / 8 x 128                              83 / 71 / 51
//   118 of 78..312 + 4 x 2..8 over 0..3000, 32 / 8 x 128                                 102 / 89 / 33
//   18 of 489..1957 + 6 x 36 over 0..3000, 32 / 8 x 128                                  110 / 94 / 44
//   15 of 253 + 4 x 65..263 over 0..3000, 32 / 32 x 80                                   103 / 79 / 39
//   20 of 100..2000 + 3 x 50..300 over 0..2000, 16 / 2 x 64                               49 / 46 / 31
// Geometric mean over 3825 batches (nine kinds of heads; 0..120 rows of up to 3000 tokens beside 17 sets of 1..8 chunks of 3..4096 over
// up to 12000): 1.37 times the separate launches' speed; 2.5 % of them more than 3 % slower than those, at most 14 %.
#include <algorithm>

#include "paged_decode.h"
#include "prefill_parts.h"
#include "prefill_w8.h"
#include "step_attn.h"

namespace hipattn {

namespace {

template <typename T, int HD>
struct StepDecode {
  struct Params : PrefillParams {
    DecodeParams decode;
    int decode_at, decode_wgs;  // which workgroups of the launch
    int n_parts, part_tiles;   // pieces of a row block's keys at most, and 64-key tiles in each
    float *part_acc, *part_ml;  // of piece i of row r and head h, at (i * total_q + r) * Hq + h: d sums; maximum and sum
  };
  static constexpr bool value = true, parts = true, window = false;
  static constexpr int block = kBlockSize;
  static __device__ __forceinline__ void decode(const Params &p, int wg, unsigned char *lds) {
    decode_flat<T, HD, kBlockSize>(p.decode, wg, *reinterpret_cast<FlatLds<HD> *>(lds));
  }
};

// The merge: a workgroup per (decode row, query head), and per (prefill row, kMergeHeads heads) where row blocks were cut.
template <typename T, int HD>
__global__ __launch_bounds__(128) void step_merge_kernel(typename StepDecode<T, HD>::Params p) {
  const int decode_merges = p.decode.Hq * p.decode.num_seqs;
  int id = blockIdx.x;
  if (id < decode_merges) {
    decode_flat_merge<T, HD>(p.decode, id % p.decode.Hq, id / p.decode.Hq);
    return;
  }
  id -= decode_merges;
  const int groups = (p.Hq + kMergeHeads - 1) / kMergeHeads;
  const int r = id / groups, h0 = id % groups * kMergeHeads;
  const int b = sequence_of_row(p.cu_q, p.batch, r);
  if (b < 0) return;
  const int q_begin = p.cu_q[b], Lq = p.cu_q[b + 1] - q_begin, Lk = p.context_lens[b], BM = 128 >> p.wg_heads_log2;
  const int last_row = min((r - q_begin) / BM * BM + BM, Lq) - 1;  // of the row's block
  const int tiles = (max(p.causal ? min(Lk, last_row + Lk - Lq + 1) : Lk, 0) + BN - 1) / BN;
  if (tiles <= p.part_tiles) return;  // whole, and written
  const int parts = min((tiles + p.part_tiles - 1) / p.part_tiles, p.n_parts);
  merge_parts<T, HD>(p, r, h0, parts);
}

// A stream's buffer, allocated once (buffers that grow with the batch are all kept): the flat split's partial results, 17 MB at most, and
// the pieces of row blocks.
constexpr size_t kStepScratchBytes = (size_t)64 << 20;

struct StepPlan {
  int decode_wgs, n_parts, part_tiles, heads_log2;
  bool decode_last;
  FlatScratch flat;
  size_t flat_bytes, part_rows;
};

// False where the launches by themselves are the better choice.
bool plan_step(const PrefillParams &pp, const DecodeParams &dp, int hd, StepPlan &pl) {
  const int heads = dp.Hkv * dp.col_groups, cus = compute_units();
  const bool decode = dp.num_seqs > 0;
  if (decode && !flat_split_counts(dp.num_seqs, heads, dp.max_ctx)) return false;
  pl = StepPlan{};
  const int64_t units = decode ? flat_units(dp.num_seqs, heads, dp.max_ctx) : 0;  // block pairs: 32 tokens of a kv head
  if (decode) {
    // Fewer workgroups than compute units where a wavefront would get fewer than two block pairs, of long contexts fewer than eight:
    // every piece of a context has to be merged (4 kv heads x 112, one context of 7484 tokens in pieces of eight pairs 24 us, two of up to
    // 7609 in pieces of two 30, either in partitions 17).
    const int least = std::min(std::max(dp.max_ctx / 256, 2), 8);
    const int64_t wgs = std::min<int64_t>(cus, (units + 4 * least - 1) / (4 * least));
    pl.decode_wgs = (int)((wgs + 7) & ~(int64_t)7);  // (a multiple of the XCDs: prefill workgroups keep theirs)
    pl.flat = flat_scratch(dp.num_seqs, dp.G, hd, pl.decode_wgs);
    pl.flat_bytes = (pl.flat.bytes + 255) & ~(size_t)255;
    if (pl.flat_bytes > kStepScratchBytes) return false;
  }
  pl.heads_log2 = prefill_heads_log2(pp, 2);
  const int tiles = std::max((pp.max_k + BN - 1) / BN, 1), bm = 128 >> pl.heads_log2;
  const int64_t wgs = (pp.total_q / bm + (pp.batch + 1) / 2) * (pp.Hq >> pl.heads_log2);  // of prefill with whole row blocks, about
  // Pieces: as many as make the longest row block's tiles, or the decode rows behind which they pass, cheaper by more than writing and
  // merging the pieces costs, all in us.  A tile: measured beside decode rows and without.  A piece: 8 bytes per element there and back, of
  // which about 60 % of the rows have one, and twice that with what a workgroup's start costs.  The merge's launch is there for the
  // decode rows anyway; without them it costs 7.  Pieces of fewer than three tiles are all set-up.  Two workgroups of a compute unit have a tile
  // in little less than twice the time of one, so pieces pay while there are compute units without work, up to seven workgroups on four
  // of them, and two where the rows alone (padding aside) leave some idle and the chain is long.  us, apart / whole / 2 / 3 / 4 / 6 pieces: 1 x 300
  // over 6000, 32 / 8 x 128 (80 workgroups) 110 / 97 / 65 / 52 / 48 / 55; 1 x 1000 over 1000 (256) 46 / 45 / 52 / 54 / 54 / 54, over 6000
  // 136 / 128 / 112 / 126 / 125 / 126; 8 x 500 over 1000, 12 / 4 x 112 (420) 49 / 44 / 68 / 64 / 64 / 64; 8 x 50 over 3000, 40 / 8 x 112 (280,
  // 125 of them rows) 91 / 91 / 65 / 64 / 58 / 62.  Three also where long chains are some more workgroups than there are places, so that a last round
  // would run nearly alone (16 / 2 x 64, 8 x 600 over 12000, 616 of 512: 304 / 272 / 293 / 256).
  const double per_tile = hd > 96 ? (decode ? 1.6 : 1.2) : (decode ? 1.2 : 0.9);
  const double per_part = (double)pp.total_q * pp.Hq * (hd + 2) * 2e-6;
  const double decode_us = units * hd * 128 * 1e-7;  // contexts of 0.65 of the longest at 6.5 TB/s
  const size_t part_bytes = (size_t)pp.total_q * pp.Hq * (hd + 2) * sizeof(float);
  int most = (int)std::min<int64_t>(std::max<int64_t>(7 * (int64_t)cus / 4 / std::max<int64_t>(wgs, 1), 1), kMostParts);
  if (most == 1 && pp.total_q * pp.Hq / 128 <= cus && tiles >= 30) most = 2;
  if (most == 1 && tiles >= 128 && wgs > 2 * cus && 2 * wgs < 5 * (int64_t)cus) most = 3;
  double best = 0;
  int parts = 1;
  for (int n = 1; n <= most; n++) {
    if (n > 1 && (n * 3 > tiles || pl.flat_bytes + n * part_bytes > kStepScratchBytes)) break;
    const double t = std::max(per_tile * ((tiles + n - 1) / n), decode_us) + (n > 1 ? (decode ? 2 : 7) + n * per_part : 0);
    if (n == 1 || t < best) {
      best = t;
      parts = n;
    }
  }
  if (parts == 1 && !decode) return false;
  // A round of workgroups over the launch's places, tiles as if every row block saw half of the longest context, takes 2.8 us a tile.
  const double prefill_us = std::max(per_tile * ((tiles + parts - 1) / parts), 2.8 * 0.5 * tiles * wgs / (2.0 * cus));
  if (parts == 1) {
    // Apart where what passes behind the decode rows is not worth what the flat split costs them, if they would not take it alone (70 rows of
    // 77..778 tokens, 32 heads x 80, beside 3 x 2..14: 59 us apart, 66 here), or where the chunks by themselves run in a form that is faster by
    // more than the decode rows are worth: narrow heads with a third workgroup on a compute unit or eight alternating wavefronts
    // (16 / 2 x 64, 8 x 512 over 1000: beside 30 rows of up to 2048 tokens 42 / 45, 60 of up to 4096 53 / 53; 2 x 1500 over 500 47 / 51 and 59 /
    // 50; with fewer workgroups, or some more and contexts of 12000, 304 / 272), heads of 128 with eight wavefronts once there are several
    // workgroups per compute unit (32 / 8 x 128, one row beside 1 x 4096 over 4096: 373 / 405; 64 / 8 x 128, 8 rows beside 4 x 1024 over 4000
    // 436 / 458; 120 rows of up to 3000 beside 8 x 600 over 12000: 768 / 697).
    if (!use_flat_split(dp.num_seqs, heads, dp.max_ctx) && prefill_us < 0.3 * decode_us) return false;
    const bool many = 2 * wgs >= 7 * (int64_t)cus;
    if (hd <= 96 && 2 * wgs >= 3 * (int64_t)cus && (many || tiles <= 128) && decode_us < 0.3 * prefill_us) return false;
    if (hd > 112 && many && decode_us < 0.25 * prefill_us) return false;
  }
  // The decode rows behind the chunks where they pass in the shadow of the last of them, else in front, where the chunks pass in theirs
  // (32 / 8 x 128, 8 x 512 over 1000, front / behind: 30 rows of up to 2048 tokens 92 / 85, 60 of up to 4096 139 / 169).
  pl.decode_last = decode_us < 0.6 * prefill_us;
  pl.part_tiles = (tiles + parts - 1) / parts;
  pl.n_parts = (tiles + pl.part_tiles - 1) / pl.part_tiles;
  pl.part_rows = pl.n_parts > 1 ? (size_t)pl.n_parts * pp.total_q * pp.Hq : 0;
  return true;
}

template <typename T, int HD>
void launch_step(const PrefillParams &pp, const DecodeParams &dp, const StepPlan &pl, char *ws, hipStream_t stream) {
  constexpr int HDP = (HD + 31) / 32 * 32, MODE = HD == HDP ? W8_PAGED_DMA : W8_PAGED_DMA_PART;
  typedef StepDecode<T, HD> Step;
  constexpr size_t tiles_bytes = (size_t)w8_stages(HDP, 4) * 2 * BN * HDP * 2;
  constexpr size_t lds_bytes = tiles_bytes > sizeof(FlatLds<HD>) ? tiles_bytes : sizeof(FlatLds<HD>);
  static bool attr_set = false;  // benign race: setting twice is harmless
  auto kernel = prefill_varlen_w8_kernel<T, HDP, MODE, Step, 4>;
  if (!attr_set) {
    HA_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_bytes));
    attr_set = true;
  }
  typename Step::Params p;
  static_cast<PrefillParams &>(p) = pp;
  p.decode = dp;
  if (pl.decode_wgs > 0) flat_scratch_set(p.decode, pl.flat, pl.decode_wgs, HD, ws);
  p.n_parts = pl.n_parts;
  p.part_tiles = pl.part_tiles;
  p.part_acc = reinterpret_cast<float *>(ws + pl.flat_bytes);
  p.part_ml = p.part_acc + pl.part_rows * HD;
  p.wg_heads_log2 = pl.heads_log2;
  const int bm = 128 >> pl.heads_log2;
  p.n_qblocks = (p.max_q + bm - 1) / bm;
  const int64_t n_wg = pl.decode_wgs + (int64_t)p.n_qblocks * p.batch * (p.Hq >> pl.heads_log2) * pl.n_parts;
  HA_CHECK(n_wg <= 0x7fffffff, "varlen_attn: too many workgroups");
  p.decode_wgs = pl.decode_wgs;
  p.decode_at = pl.decode_last ? (int)n_wg - pl.decode_wgs : 0;
  kernel<<<dim3((unsigned)n_wg), 256, lds_bytes, stream>>>(p);
  check_launch("varlen_attn (prefill and decode rows)");
  const int64_t merges = (int64_t)dp.Hq * dp.num_seqs + (pl.n_parts > 1 ? p.total_q * ((p.Hq + kMergeHeads - 1) / kMergeHeads) : 0);
  HA_CHECK(merges <= 0x7fffffff, "varlen_attn: too many rows");
  step_merge_kernel<T, HD><<<dim3((unsigned)merges), 128, 0, stream>>>(p);
  check_launch("varlen_attn (merge)");
}

template <typename T>
bool dispatch_step(const PrefillParams &pp, const DecodeParams &dp, const StepPlan &pl, int hd, char *ws, hipStream_t stream) {
  switch (hd) {
    case 64: launch_step<T, 64>(pp, dp, pl, ws, stream); return true;
    case 80: launch_step<T, 80>(pp, dp, pl, ws, stream); return true;
    case 96: launch_step<T, 96>(pp, dp, pl, ws, stream); return true;
    case 112: launch_step<T, 112>(pp, dp, pl, ws, stream); return true;
    case 128: launch_step<T, 128>(pp, dp, pl, ws, stream); return true;
    default: return false;
  }
}

}  // namespace

bool step_attention(const PagedPrefillCall &chunks, hipattn_tensor *chunks_out, const DecodeCall *rows, hipattn_tensor *rows_out, void *stream_arg) {
  const int hd = (int)chunks.q->sizes[2], dtype = chunks.q->dtype, tiles = (chunks.max_k + BN - 1) / BN;
  if (hd != 64 && hd != 80 && hd != 96 && hd != 112 && hd != 128) return false;
  // Up to three tiles of keys the launches by themselves are as fast, and with few decode rows of long contexts faster (5 x 2337 tokens,
  // 4 kv heads x 112, beside 5 x 20: 17.5 / 20.8 us); chunks alone have to be long to be worth a merge.
  if (rows == nullptr ? tiles < 12 : tiles <= 3 && !use_flat_split(rows->query->sizes[0], rows->num_kv_heads, rows->max_context_len)) return false;
  const Tuning &tn = tuning();  // switches that ask for a kernel of one of the two
  if (tn.prefill_kernel != 0 || tn.decode_flat >= 0 || tn.decode_flat_wgs > 0 || tn.decode_part_blocks > 0) return false;
  PrefillParams pp;
  DecodeParams dp;
  memset(&dp, 0, sizeof dp);
  if (!paged_prefill_params(chunks, chunks_out, nullptr, pp) || !paged_prefill_copies_images(pp) || pp.out_f32) return false;
  if (rows != nullptr && (rows->block_size != kBlockSize || !decode_params(*rows, rows_out, dp))) return false;
  StepPlan pl;
  if (!plan_step(pp, dp, hd, pl)) return false;
  // Under capture, without memory, and on hipStreamPerThread (one handle for a stream of each thread's own): the launches by themselves.
  // The two launches here stay next to one another where several threads use one stream.
  hipStream_t stream = resolve_stream(stream_arg);
  if (stream == hipStreamPerThread) return false;
  // A capture of this step will run them, and cannot allocate the decode rows' scratch memory: this call is the one made ahead of it.
  if (rows != nullptr) reserve_library_workspace(WS_PAGED_ATTENTION, decode_scratch_bytes(*rows), stream);
  const HeldWorkspace ws = try_library_workspace(WS_STEP_ATTENTION, kStepScratchBytes, stream);
  if (ws.ptr == nullptr) return false;
  return dtype == HIPATTN_BF16 ? dispatch_step<bf16_t>(pp, dp, pl, hd, static_cast<char *>(ws.ptr), stream)
                               : dispatch_step<half_t>(pp, dp, pl, hd, static_cast<char *>(ws.ptr), stream);
}

}  // namespace hipattn
