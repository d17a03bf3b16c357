// Varlen prefill over the paged cache with a sliding window and sinks: new tokens of a sequence, causal, each against the window_left
// tokens before it, itself and the sequence's first sink_tokens ones.  The reference has windows without sinks and over rows of k / v alone
// (rllm/tch-cuda/kernels/flash_attn/flash_api.cpp:113-120, softmax.h:142-179); rLLM passes none.
//
//   row r of the sequence, at position r + Lk - Lq, sees key j iff j <= r + Lk - Lq and (j >= r + Lk - Lq - window_left or j < sinks).
//
// The kernels are those of hipattn_mha_varlen_fwd_paged -- block images of the cache copied into LDS, two wavefronts of a SIMD that alternate
// between the matrix pipe and the vector ALU, or workgroups of four wavefronts several to a compute unit -- over the 64-key tiles that hold a
// key some row of the workgroup sees (prefill_w8.h, STEP::window).  What bounds them is the matrix pipe and the vector unit on
// (window + rows of a block) keys a row, and with few workgroups the chain of a row block's tiles.  Measured: 2 x 4096 new tokens, 32 / 8 x 128 bf16,
// a window of 4096 535 us, 0.96 PFLOP/s of what is seen (causal prefill of 8 x 4096 without a window 1.0 to 1.1); 8 chunks of
// 65 to 1001 tokens, 16 / 2 x 64 fp16, a window of 1001 40 to 50 us by the order of the chunks, 0.31 to 0.39 PFLOP/s: the softmax of narrow heads, and
// 552 workgroups, two or three to a compute unit (8 x 512 tokens, 512 workgroups, 39).  Head sizes above 128 and those below 64 but 32 take tiles
// staged through registers (prefill_varlen.hip), a row block's keys by one workgroup: 8 / 2 x 256, 1 x 2000 behind 4096 279 us, 0.24 PFLOP/s.
// Probabilities are rounded to the cache's type as operands of the second product, as in all attention here; scores, sums and pieces are fp32.
#include <algorithm>

#include "paged_decode.h"
#include "prefill_parts.h"
#include "prefill_window_params.h"
#include "window_rows.h"

namespace hipattn {

namespace {

constexpr int kTileKeys = 64;

// Tiles of the longest chain: what a row block of `rows` rows sees at most.
int64_t most_tiles(const PrefillParams &p, int rows) {
  auto tiles = [](int64_t keys) { return (keys + kTileKeys - 1) / kTileKeys; };
  return std::min<int64_t>(tiles(p.max_k), tiles(p.sinks) + tiles((int64_t)p.win_left + rows) + 1);
}

// Workgroups of eight wavefronts instead of four: what their alternation between the pipes gains a tile is lost again where a block of twice as many
// rows is filled less, or where one of them ends before the others and leaves its compute unit idle.  So only where they fill the compute units
// once and nearly all, with chains alike and long: chunks of like lengths, all of whose rows see a whole window.  us, eight / four: 1 x 2000 new tokens
// behind 4096 (256 workgroups, 224 to 256 take the same) with a window of 4096, 32 / 8 x 128 149 / 155, 32 / 8 x 112 147 / 156, 32 / 32 x 80 127 / 147;
// 1 x 4000, 16 / 2 x 96 128 / 138; behind nothing 64 / 57, 64 / 59, 59 / 60, 111 / 105, as the first rows have few keys.  264 workgroups, 24 / 8 x 96 218 / 146.
// Heads of 128, two to ten rounds of workgroups, 96 shapes: four are 2.7 % faster on average and 14 % at most, eight 2.9 % at most.  16 / 2 x 64, 2 x
// 4096 225 / 216.
bool eight_wavefronts_pay(const PrefillParams &p) {
  const int hl = prefill_heads_log2(p, 3), rows = 256 >> hl;
  const int64_t wgs = (int64_t)p.batch * ((p.max_q + rows - 1) / rows) * (p.Hq >> hl), tiles = most_tiles(p, rows);
  const bool alike = p.total_q * 10 >= (int64_t)p.batch * p.max_q * 9 && p.max_k - p.max_q >= p.win_left;
  return alike && wgs <= compute_units() && wgs * 8 > compute_units() * 7 && p.d > 64 && tiles >= 32;
}

// Pieces that a row block's keys are dealt out in (workgroups of four wavefronts).  A workgroup's chain of tiles is bound by its own
// instructions, some 2 us a tile with a wavefront per SIMD (five tiles in LDS instead of two change nothing), so where compute units are idle
// more of them take a part each.  All in us, and fitted: what does not grow with the tiles; a tile, which takes longer from two workgroups per
// compute unit on, as two or three of them fill each other's gaps; the merge, and what writing and reading the pieces costs.  In 400 measured shapes
// (1 x 5 new tokens to 2 x 4096, alike and 63 x 20 beside one of 4096, windows of 100 to 4096, four kinds of heads) the choice among these and the
// kernel of decode rows is 1.8 % off the best on average and 20 % at most; whole blocks alone are 39 %.  In 90 whose sequences have contexts of very
// different lengths 3.2 %, at most 2.2 times: the host knows the longest context alone.  us, whole / best: 32 / 8 x 128, 1 x 5 over 4096 keys 99 / 16
// (rows), 1 x 300 106 / 48 (6 pieces), 4 x 64 over 2000 61 / 29 (4); 32 / 32 x 80, 12 of 1 to 64 over 2000 83 / 65 (2); 16 / 2 x 64, 100 x 4 over
// 2000 66 / 39 (rows).
// At most `most`; us: about what the launch takes then.
int choose_parts(const PrefillParams &p, int most, double &us) {
  const int hl = prefill_heads_log2(p, 2), rows = 128 >> hl;
  const int64_t tiles = most_tiles(p, rows);
  const double wgs = ((double)(p.total_q / rows) + 0.7 * (p.batch + 1)) * (p.Hq >> hl);
  const double fixed = p.d > 96 ? 8 : (p.d > 64 ? 16 : 9), tile = p.d > 64 ? 2.1 : 1.7;
  const double share = (p.d > 96 ? 0.62 : (p.d > 64 ? 0.45 : 0.5)) / compute_units();
  const double piece = (double)p.total_q * p.Hq * (p.d + 2) * 2e-6;
  int parts = 1;
  us = 0;
  for (int n : {1, 2, 3, 4, 6, 10, 16}) {
    const int64_t part_tiles = (tiles + n - 1) / n;
    if (n > 1 && (n > most || n > tiles || (tiles + part_tiles - 1) / part_tiles != n)) continue;
    const double t = fixed + (double)part_tiles * tile * std::max(1.0, share * wgs * n) + (n > 1 ? 5.0 + n * piece : 0.0);
    if (n == 1 || t < (parts == 1 ? 0.87 : 1.0) * us) {
      us = t;
      parts = n;
    }
  }
  return parts;
}

// What the staged form takes: workgroups of 128 rows of one head, about 3.5 us a tile of a head size of 256 (us, 8 / 2 x 256: 1 x 8 over 1024 69, 1 x
// 300 over 4096 268, 4 x 64 over 2048 156).
double staged_us(const PrefillParams &p) {
  const int64_t wgs = std::max<int64_t>(p.total_q / 128 + (p.batch + 1) / 2, 1) * p.Hq;
  return 10 + (double)most_tiles(p, 128) * 3.5 * std::max(p.d, 128) / 256 * std::max(1.0, 0.6 * (double)wgs / compute_units());
}

// A stream's buffer, allocated once; and what a call may need of it or of a caller's.
constexpr size_t kWindowScratchBytes = (size_t)64 << 20;
size_t piece_bytes(int64_t total_q, int heads, int d) { return (size_t)total_q * heads * (d + 2) * sizeof(float); }
size_t scratch_bytes(int64_t total_q, int heads, int d) {
  return kMostParts * std::min(piece_bytes(total_q, heads, d), kWindowScratchBytes / kMostParts);
}
// Pieces that it holds, at most.
int held_parts(int64_t total_q, int heads, int d) {
  return (int)std::max<size_t>(std::min<size_t>(kWindowScratchBytes / piece_bytes(total_q, heads, d), kMostParts), 1);
}

void mha_varlen_fwd_paged_window_impl(const hipattn_tensor *q, const hipattn_tensor *key_cache, const hipattn_tensor *value_cache,
                                      const hipattn_tensor *block_tables, const hipattn_tensor *cu_q, const hipattn_tensor *context_lens,
                                      int max_q, int max_k, float scale, int window_left, int sinks, hipattn_tensor *out,
                                      hipattn_tensor *lse, const hipattn_tensor *workspace, void *stream_arg) {
  const char *op = "mha_varlen_fwd_paged_window";
  HA_CHECK(window_left >= 0, "%s: window_size_left must not be negative here, got %d", op, window_left);
  HA_CHECK(sinks >= 0, "%s: sink_tokens must not be negative, got %d", op, sinks);
  if (workspace) {
    check_tensor(workspace, "workspace", 1);
    HA_CHECK(workspace->dtype == HIPATTN_U8, "%s: workspace must be u8", op);
    check_contiguous(workspace, "workspace");
  }
  WindowParams p;
  if (!paged_prefill_params(PagedPrefillCall{q, key_cache, value_cache, block_tables, cu_q, context_lens, max_q, max_k, scale, true, op}, out,
                            lse, p))
    return;
  HA_CHECK(p.table_cols > 0, "%s: block_tables has no columns", op);  // (a context says on the device whether there is one to be read)
  p.max_q = (int)std::min<int64_t>(p.max_q, p.total_q);  // (no sequence has more; what is rounded up to row blocks stays within 32 bits)
  // (no context is longer than its table: what lies beyond that sees everything, and row + Lk - Lq - window_left stays within 32 bits)
  const int64_t longest = (int64_t)p.table_cols << p.block_log2;
  p.win_left = (int)std::min<int64_t>(window_left, std::min<int64_t>(longest, 1 << 30));
  p.sinks = (int)std::min<int64_t>(sinks, std::min<int64_t>(longest, 1 << 30));
  p.win_right = 0;
  p.causal = 1;
  p.n_parts = 1;
  p.part_tiles = 1 << 24;
  p.part_acc = p.part_ml = nullptr;
  const int force = tuning().prefill_kernel;
  const bool lse_or_f32 = lse != nullptr || p.out_f32;  // (neither the merges nor the kernel of decode rows have them)
  const bool merged_head = p.d == 64 || p.d == 80 || p.d == 96 || p.d == 112 || p.d == 128;  // (there is a merge for it; 256: decode rows alone)
  const int possible = lse_or_f32 || force != 0 || !(merged_head || p.d == 256) ? 1 : held_parts(p.total_q, p.Hq, p.d);
  char *given = nullptr;
  if (workspace && possible > 1) {  // (else there is nothing to put there)
    const size_t need = possible * piece_bytes(p.total_q, p.Hq, p.d);
    HA_CHECK(workspace->data != nullptr && (reinterpret_cast<uintptr_t>(workspace->data) & 255) == 0,
             "%s: workspace must be 256-byte aligned", op);
    HA_CHECK((size_t)workspace->sizes[0] >= need,
             "%s: workspace of %lld bytes is too small, %zu are needed (hipattn_mha_varlen_fwd_paged_window_workspace_size)", op,
             (long long)workspace->sizes[0], need);
    given = static_cast<char *>(workspace->data);
  }
  hipStream_t stream = resolve_stream(stream_arg);
  // Block images go into LDS as they are where they fill most of their place there; else tiles are staged through registers.
  const bool images = p.vc_block % 8 == 0 && p.vc_head % 8 == 0 && tuning().paged_prefill_dma != 0 && p.d <= 128 && (p.d >= 64 || p.d == 32);
  const int pieces = images && merged_head ? tuning().window_parts : 0;
  const bool eight = images && (force == 1 || (force == 0 && pieces == 0 && eight_wavefronts_pay(p)));
  // What pieces need lies in the caller's workspace or a buffer of the stream's, of one size, so that either gives the same bits; without it -- in a
  // capture, for shapes beyond it, on hipStreamPerThread, one handle for a stream of each thread's own -- nothing is cut that has to be merged.
  HeldWorkspace ws;
  void *scratch = given;
  int most = (stream == hipStreamPerThread && !given) || eight ? 1 : possible;
  for (;;) {
    int parts = 1;
    double us = images ? 0 : staged_us(p);
    if (pieces > 0) parts = std::min(pieces, most);
    else if (images && !eight) parts = choose_parts(p, merged_head ? most : 1, us);
    RowsPlan rows;
    const bool as_rows = force == 0 && pieces == 0 && !eight && !lse_or_f32 && plan_window_rows(p, most, rows) && rows.us < us;
    if (as_rows) parts = rows.num_parts;
    if (parts > 1 && !given) {
      ws = try_library_workspace(WS_WINDOW_CHUNKS, kWindowScratchBytes, stream);
      scratch = ws.ptr;
      if (scratch == nullptr) {
        most = 1;
        continue;
      }
    }
    if (as_rows) {
      launch_window_rows(p, rows, q->dtype, scratch, stream);
      return;
    }
    if (parts > 1) {
      const int64_t tiles = most_tiles(p, 128 >> prefill_heads_log2(p, 2));
      p.part_tiles = (int)((tiles + parts - 1) / parts);
      p.n_parts = (int)((tiles + p.part_tiles - 1) / p.part_tiles);
      p.part_acc = static_cast<float *>(scratch);
      p.part_ml = p.part_acc + (size_t)p.n_parts * p.total_q * p.Hq * p.d;
    }
    break;
  }
  if (!images) {
    launch_staged_window(p, q->dtype, stream);
    return;
  }
  const int waves = eight ? 8 : 4;
  switch (p.block_log2) {
    case 3: launch_window_images_8(p, waves, q->dtype, stream); break;
    case 5: launch_window_images_32(p, waves, q->dtype, stream); break;
    default: launch_window_images_16(p, waves, q->dtype, stream); break;
  }
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" char *hipattn_mha_varlen_fwd_paged_window(const hipattn_tensor *q, const hipattn_tensor *key_cache,
                                                     const hipattn_tensor *value_cache, const hipattn_tensor *block_tables,
                                                     const hipattn_tensor *cu_seqlens_q, const hipattn_tensor *context_lens,
                                                     int max_seqlen_q, int max_seqlen_k, float softmax_scale, int window_size_left,
                                                     int sink_tokens, hipattn_tensor *out, hipattn_tensor *softmax_lse,
                                                     const hipattn_tensor *workspace, void *stream) {
  HA_PROTECT(mha_varlen_fwd_paged_window_impl(q, key_cache, value_cache, block_tables, cu_seqlens_q, context_lens, max_seqlen_q,
                                              max_seqlen_k, softmax_scale, window_size_left, sink_tokens, out, softmax_lse, workspace,
                                              stream));
}

extern "C" char *hipattn_mha_varlen_fwd_paged_window_workspace_size(int64_t total_q, int num_heads, int head_size, int64_t *bytes) {
  HA_PROTECT({
    const char *op = "mha_varlen_fwd_paged_window_workspace_size";
    HA_CHECK(bytes != nullptr, "%s: bytes is NULL", op);
    HA_CHECK(total_q >= 0 && total_q <= 0x7fffffff && num_heads >= 0 && num_heads <= 1 << 20, "%s: a size is negative or too large", op);
    HA_CHECK(head_size >= 0 && head_size <= 256, "%s: head size %d not supported (at most 256)", op, head_size);
    *bytes = (int64_t)scratch_bytes(total_q, num_heads, head_size);
  });
}
