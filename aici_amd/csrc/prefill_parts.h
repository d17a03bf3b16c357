// Row blocks whose keys several workgroups of prefill_varlen_w8_kernel share (STEP::parts): the merge of what they leave, for a step's
// attention (step_attn.hip) and that of windows (prefill_window.hip); the search for a row's sequence is also that of trees (tree_attn.hip).  Device code.
#pragma once

#include "prefill_common.h"

namespace hipattn {

namespace {

constexpr int kMostParts = 16;
constexpr int kMergeHeads = 8;  // query heads of a row per workgroup of the merge

// The sequence that holds row r of all sequences' rows, -1: none; by a whole wavefront.
__device__ __forceinline__ int sequence_of_row(const int32_t *cu_q, int batch, int r) {
  const int lane = threadIdx.x & 63;
  if (r < cu_q[0]) return -1;
  for (int s0 = 0; s0 < batch; s0 += 64) {
    const unsigned long long past = __ballot(s0 + lane < batch && cu_q[min(s0 + lane, batch - 1) + 1] > r);
    if (past != 0) return s0 + __builtin_ctzll(past);
  }
  return -1;
}

// Adds up the `parts` pieces of row r (of all sequences) for the kMergeHeads heads from h0 on, a workgroup of 128 threads.
template <typename T, int HD, typename P>
__device__ __forceinline__ void merge_parts(const P &p, const int r, const int h0, const int parts) {
  constexpr int QUADS = HD / 4;
  for (int i = threadIdx.x; i < kMergeHeads * QUADS; i += 128) {
    const int h = h0 + i / QUADS, e = i % QUADS * 4;
    if (h >= p.Hq) break;
    float m[kMostParts], l[kMostParts];
    f32x4_t a[kMostParts];
#pragma unroll
    for (int k = 0; k < kMostParts; k++) {
      m[k] = -INFINITY;
      l[k] = 0.f;
      a[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (k < parts) {
        const int64_t at = ((int64_t)k * p.total_q + r) * p.Hq + h;
        const float2 ml = *reinterpret_cast<const float2 *>(p.part_ml + 2 * at);
        m[k] = ml.x;
        l[k] = ml.y;
        a[k] = *reinterpret_cast<const f32x4_t *>(p.part_acc + at * HD + e);
      }
    }
    float most = m[0];
#pragma unroll
    for (int k = 1; k < kMostParts; k++) most = fmaxf(most, m[k]);
    const float base = most == -INFINITY ? 0.f : most;
    float sum = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kMostParts; k++) {
      const float w = fast_exp2(m[k] - base);
      sum += w * l[k];
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] += w * a[k][j];
    }
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;
    T out[4];
#pragma unroll
    for (int j = 0; j < 4; j++) out[j] = from_float<T>(o[j] * inv);
    *reinterpret_cast<u32x2_t *>(static_cast<T *>(p.out) + (int64_t)r * p.o_row + (int64_t)h * p.o_head + e) = *reinterpret_cast<u32x2_t *>(out);
  }
}

}  // namespace
}  // namespace hipattn
