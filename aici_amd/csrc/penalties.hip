// Penalties for tokens that a sequence has said already, the controller's bias and its allow-mask, on the logits of a batch: what goes in
// front of hipattn_bias_argmax / hipattn_bias_sample (rllm/rllm-cuda/src/llm/tmodel.rs:277-283 applies the bias alone).
//
//   x = l; said: x = x > 0 ? x / repetition : x * repetition; x -= frequency * count + presence * (count > 0); x += bias; barred: x = -inf
//
// with `said` over all of a sequence's tokens and `count` over those behind its prompt.  Computed in fp32, rounded once to the type of the
// output.
//
// What it cannot do without is the logits in and out, the bias and the bits: it is bound by memory.  A workgroup owns a tile of a row's
// vocabulary: it asks for its logits, counts the sequence's tokens that fall into the tile in LDS -- whole numbers, so that the order of the
// additions does not matter -- while they are on their way, and then goes over them.  A sequence's tokens are read once per tile, from L2: the
// tiles of a row lie on one XCD.
#include "common.h"
#include "device_types.h"

namespace hipattn {

namespace {

constexpr unsigned kSaid = 0x80000000u;  // in a token's word: said at all; the rest counts what lies behind the prompt

struct PenaltyParams {
  const void *logits;
  void *out;
  int64_t logit_stride, out_stride;
  int vocab, tiles, num_seqs;
  const int32_t *history;
  int64_t n_history;
  const void *offsets;  // [S + 1] int64 or int32
  bool offsets64;
  const int32_t *prompt;  // [S] or null
  const float *repetition, *frequency, *presence;  // [S] or null
  const float *bias;  // [rows, >= vocab] or null
  int64_t bias_stride, bias_rows;
  const uint8_t *mask;
  int64_t mask_stride, mask_bytes, mask_rows;
  const int32_t *rows;  // [S] or null
};

// A barrier for what is handed over in LDS alone: __syncthreads() would wait for the tile's loads too.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Threads, and runs of 8 tokens for each.  us, 512 x 2 / 1024 x 2 / 1024 x 1 / 256 x 4 / 256 x 2 / 512 x 4: 64 x 128256 bf16 under a mask, 0.5k..4k
// tokens said 11.5 / 11.3 / 13.4 / 13.7 / 12.6 / 13.2; 256 x 128256 to fp32 with a bias, up to 16k said 73 (4.6 TB/s) / 71 / 73 / 80 / 81 / 79; 1 x
// 50003 fp16, launch and latency alone, 5.6 / 5.4 / 5.5 / 6.2 / 5.3 / 6.3; seven others, 5 to 40 us, 512 x 2 the fastest on average.
constexpr int kThreads = 512, kRuns = 2;
constexpr int kTile = 8 * kRuns * kThreads;

template <typename T, typename O, bool BIAS, bool MASK>
__global__ __launch_bounds__(kThreads) void penalties_kernel(PenaltyParams p) {
  constexpr int WORDS = 8 * (int)sizeof(T) / 16;  // 16-byte loads per run
  __shared__ __attribute__((aligned(16))) unsigned s_count[kTile];
  const int tid = threadIdx.x;
  // Workgroup -> (row, tile): consecutive ids go to the 8 XCDs in turn, so eight rows at a time, a row's tiles 8 ids apart.
  const int seq = (int)(blockIdx.x / (8u * p.tiles)) * 8 + (int)(blockIdx.x & 7u);
  const int tile = (int)(blockIdx.x >> 3) % p.tiles;
  if (seq >= p.num_seqs) return;
  int64_t begin = p.offsets64 ? static_cast<const int64_t *>(p.offsets)[seq] : static_cast<const int32_t *>(p.offsets)[seq];
  int64_t end = p.offsets64 ? static_cast<const int64_t *>(p.offsets)[seq + 1] : static_cast<const int32_t *>(p.offsets)[seq + 1];
  begin = min(max(begin, (int64_t)0), p.n_history);  // (offsets that are none read wrong tokens, never outside)
  const int said = (int)(min(max(end, begin), p.n_history) - begin);
  const int32_t *history = p.history + begin;
  const int behind = p.prompt ? p.prompt[seq] : 0;
  // The history in fours between its 16-byte boundaries, the first of them asked for ahead of everything else; the ends one by one.
  const int up = min((int)(4 - ((reinterpret_cast<uintptr_t>(history) >> 2) & 3)) & 3, said);
  const int quads = (said - up) >> 2, last = up + 4 * quads;
  const int4 *quad = reinterpret_cast<const int4 *>(history + up);
  constexpr int AHEAD = 2;
  int4 ahead[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; k++) {
    ahead[k] = make_int4(-1, -1, -1, -1);
    if (tid + k * kThreads < quads) ahead[k] = quad[tid + k * kThreads];
  }
  int end_token = -1, end_at = 0;
  if (tid < up) {
    end_at = tid;
    end_token = history[end_at];
  } else if (tid >= 64 && tid - 64 < said - last) {
    end_at = last + tid - 64;
    end_token = history[end_at];
  }
  const T *lg = static_cast<const T *>(p.logits) + seq * p.logit_stride;
  O *out = static_cast<O *>(p.out) + seq * p.out_stride;
  // Runs lie on 16-byte boundaries of the logits' memory: run c holds tokens [8 c - lead, 8 c - lead + 8) of the row.
  const int lead = (int)((reinterpret_cast<uintptr_t>(lg) & 15) / sizeof(T));
  const int v0 = tile * kTile - lead;  // the tile's first token
  auto whole = [&](int v) { return v >= 0 && v + 8 <= p.vocab; };
  const int64_t row = p.rows ? (int64_t)p.rows[seq] : seq;  // (a bad row index reads a wrong row, never outside)
  const float *bias = BIAS ? p.bias + min(max(row, (int64_t)0), p.bias_rows - 1) * p.bias_stride : nullptr;
  const uint8_t *mask = MASK ? p.mask + min(max(row, (int64_t)0), p.mask_rows - 1) * p.mask_stride : nullptr;
  const bool bias_aligned = ((reinterpret_cast<uintptr_t>(bias) - (uintptr_t)lead * sizeof(float)) & 15) == 0;
  auto bits_at = [&](int byte) -> unsigned { return byte < p.mask_bytes ? mask[byte] : 0u; };
  // Everything the tile needs is asked for in front of the count (64 x 128256 as above: 20 us with one token per thread and load, 13.9 with
  // runs of 8, 11.5 with the history's first loads and these ahead of it, 9 without history and mask; a plain copy 5.8).
  uint4 raw[kRuns][WORDS], raw_bias[BIAS ? kRuns : 1][2];
  unsigned bits[MASK ? kRuns : 1];
#pragma unroll
  for (int k = 0; k < kRuns; k++) {
    const int v = v0 + 8 * (tid + k * kThreads);
#pragma unroll
    for (int w = 0; w < WORDS; w++)
      if (whole(v)) raw[k][w] = load16_once(reinterpret_cast<const char *>(lg + v) + 16 * w);
    if (BIAS && bias_aligned && whole(v)) {
      raw_bias[k][0] = load16_once(bias + v);
      raw_bias[k][1] = load16_once(bias + v + 4);
    }
    if (MASK && whole(v)) bits[k] = (v & 7) == 0 ? bits_at(v >> 3) : (bits_at(v >> 3) | bits_at((v >> 3) + 1) << 8) >> (v & 7);
  }
#pragma unroll
  for (int i = 0; i < kTile / 4; i += kThreads) reinterpret_cast<uint4 *>(s_count)[i + tid] = make_uint4(0, 0, 0, 0);
  const float repetition = p.repetition ? p.repetition[seq] : 1.f, frequency = p.frequency ? p.frequency[seq] : 0.f,
              presence = p.presence ? p.presence[seq] : 0.f;
  lds_barrier();
  auto count = [&](int token, int i) {
    const unsigned t = (unsigned)(token - v0);
    if (t < (unsigned)kTile && (unsigned)token < (unsigned)p.vocab) {
      if (i >= behind) atomicAdd(&s_count[t], 1u);
      else atomicOr(&s_count[t], kSaid);
    }
  };
  auto count4 = [&](int4 q, int i) {
    count(q.x, i);
    count(q.y, i + 1);
    count(q.z, i + 2);
    count(q.w, i + 3);
  };
  count(end_token, end_at);
#pragma unroll
  for (int k = 0; k < AHEAD; k++) count4(ahead[k], up + 4 * (tid + k * kThreads));
  for (int i = tid + AHEAD * kThreads; i < quads; i += 4 * kThreads) {
    int4 q[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      q[k] = make_int4(-1, -1, -1, -1);
      if (i + k * kThreads < quads) q[k] = quad[i + k * kThreads];
    }
#pragma unroll
    for (int k = 0; k < 4; k++) count4(q[k], up + 4 * (i + k * kThreads));
  }
  lds_barrier();
  auto penalized = [&](float x, unsigned c) -> float {
    if (c != 0) {
      x = x > 0.f ? x / repetition : x * repetition;
      const unsigned times = c & ~kSaid;
      if (times != 0) x -= frequency * (float)times + presence;
    }
    return x;
  };
  const bool out_aligned = ((reinterpret_cast<uintptr_t>(out) - (uintptr_t)lead * sizeof(O)) & 15) == 0;
#pragma unroll
  for (int k = 0; k < kRuns; k++) {
    const int at = 8 * (tid + k * kThreads), v = v0 + at;
    if (whole(v)) {
      unsigned c[8];
      *reinterpret_cast<uint4 *>(c) = *reinterpret_cast<const uint4 *>(s_count + at);
      *reinterpret_cast<uint4 *>(c + 4) = *reinterpret_cast<const uint4 *>(s_count + at + 4);
      float x[8];
      T t[8];
      __builtin_memcpy(t, raw[k], sizeof t);
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = to_float(t[j]);
      if ((c[0] | c[1] | c[2] | c[3] | c[4] | c[5] | c[6] | c[7]) != 0) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = penalized(x[j], c[j]);
      }
      if constexpr (BIAS) {
        float b[8];
        if (bias_aligned) {
          __builtin_memcpy(b, raw_bias[k], sizeof b);
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) b[j] = bias[v + j];
        }
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] += b[j];
      }
      if constexpr (MASK) {
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (!((bits[k] >> j) & 1)) x[j] = -INFINITY;
      }
      O o[8];
#pragma unroll
      for (int j = 0; j < 8; j++) o[j] = from_float<O>(x[j]);
      if (out_aligned) {
        uint4 words[8 * sizeof(O) / 16];
        __builtin_memcpy(words, o, sizeof o);
#pragma unroll
        for (int w = 0; w < (int)(8 * sizeof(O) / 16); w++) *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(out + v) + 16 * w) = words[w];
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) out[v + j] = o[j];
      }
    } else if (v + 8 > 0 && v < p.vocab) {  // the row's ends
      for (int j = max(-v, 0); j < 8 && v + j < p.vocab; j++) {
        float x = penalized(to_float(lg[v + j]), s_count[at + j]);
        if (BIAS) x += bias[v + j];
        if (MASK && !((bits_at((v + j) >> 3) >> ((v + j) & 7)) & 1)) x = -INFINITY;
        out[v + j] = from_float<O>(x);
      }
    }
  }
}

void check_floats(const hipattn_tensor *t, const char *name, int64_t S) {
  if (t == nullptr) return;
  check_tensor(t, name, 1);
  HA_CHECK(t->dtype == HIPATTN_F32 && t->sizes[0] == S, "penalize_logits: %s must be f32 [%lld]", name, (long long)S);
  check_contiguous(t, name);
  check_data(t, name);
}

void penalize_logits_impl(hipattn_tensor *out, const hipattn_tensor *logits, const hipattn_tensor *history, const hipattn_tensor *offsets,
                          const hipattn_tensor *prompt_lens, const hipattn_tensor *repetition, const hipattn_tensor *frequency,
                          const hipattn_tensor *presence, const hipattn_tensor *bias, const hipattn_tensor *mask,
                          const hipattn_tensor *rows, void *stream_arg) {
  check_tensor(logits, "logits", 2);
  check_tensor(out, "out", 2);
  const int64_t S = logits->sizes[0], V = logits->sizes[1];
  HA_CHECK(is_float_dtype(logits->dtype), "penalize_logits: logits must be f32/f16/bf16");
  HA_CHECK(out->dtype == logits->dtype || out->dtype == HIPATTN_F32, "penalize_logits: out must have the type of logits or be f32");
  HA_CHECK(out->sizes[0] == S && out->sizes[1] == V, "penalize_logits: out and logits shapes differ");
  HA_CHECK(V <= 0x3ffffff0, "penalize_logits: vocabulary too large");
  HA_CHECK(V <= 1 || (logits->strides[1] == 1 && out->strides[1] == 1), "penalize_logits: rows must be contiguous");
  HA_CHECK(S <= 1 || out->strides[0] >= V, "penalize_logits: rows of out must not overlap");
  check_tensor(history, "history", 1);
  HA_CHECK(history->dtype == HIPATTN_I32, "penalize_logits: history must be int32, got %s", dtype_name(history->dtype));
  check_contiguous(history, "history");
  HA_CHECK(history->sizes[0] <= 0x3ffffff0, "penalize_logits: history too long");
  check_data(history, "history");
  check_index_tensor(offsets, "history_offsets", 1);
  HA_CHECK(offsets->sizes[0] == S + 1, "penalize_logits: history_offsets must hold %lld entries", (long long)S + 1);
  if (prompt_lens) {
    check_tensor(prompt_lens, "prompt_lens", 1);
    HA_CHECK(prompt_lens->dtype == HIPATTN_I32 && prompt_lens->sizes[0] == S, "penalize_logits: prompt_lens must be int32 [%lld]",
             (long long)S);
    check_contiguous(prompt_lens, "prompt_lens");
    check_data(prompt_lens, "prompt_lens");
  }
  check_floats(repetition, "repetition", S);
  check_floats(frequency, "frequency", S);
  check_floats(presence, "presence", S);
  if (bias) {
    check_tensor(bias, "bias", 2);
    HA_CHECK(bias->dtype == HIPATTN_F32, "penalize_logits: bias must be f32");
    HA_CHECK(bias->sizes[1] >= V, "penalize_logits: bias rows have %lld entries, vocabulary is %lld", (long long)bias->sizes[1], (long long)V);
    HA_CHECK(bias->sizes[1] <= 1 || bias->strides[1] == 1, "penalize_logits: bias rows must be contiguous");
    check_data(bias, "bias");
  }
  if (mask) {
    check_tensor(mask, "mask", 2);
    HA_CHECK(mask->dtype == HIPATTN_U8, "penalize_logits: mask must be u8");
    HA_CHECK(mask->sizes[1] <= 1 || mask->strides[1] == 1, "penalize_logits: mask rows must be contiguous");
    check_data(mask, "mask");
  }
  if (rows) {
    check_tensor(rows, "bias_rows", 1);
    HA_CHECK(rows->dtype == HIPATTN_I32 && rows->sizes[0] == S, "penalize_logits: bias_rows must be int32 [%lld]", (long long)S);
    check_contiguous(rows, "bias_rows");
    check_data(rows, "bias_rows");
  }
  for (const hipattn_tensor *t : {bias, mask})
    HA_CHECK(t == nullptr || S == 0 || t->sizes[0] >= (rows ? 1 : S), "penalize_logits: %lld bias or mask rows for %lld sequences",
             (long long)t->sizes[0], (long long)S);
  if (S == 0 || V == 0) return;
  HA_CHECK(S <= 0x7ffffff0, "penalize_logits: too many sequences");
  check_data(logits, "logits");
  check_data(out, "out");
  HA_CHECK(apart(out, logits) || (out->data == logits->data && out->dtype == logits->dtype && (S == 1 || out->strides[0] == logits->strides[0])),
           "penalize_logits: out must be logits or lie apart from them");
  for (const hipattn_tensor *in : {history, offsets, prompt_lens, repetition, frequency, presence, bias, mask, rows})
    HA_CHECK(in == nullptr || apart(out, in), "penalize_logits: out lies over an input other than logits");
  PenaltyParams p;
  memset(&p, 0, sizeof p);
  p.logits = logits->data;
  p.out = out->data;
  p.logit_stride = logits->strides[0];
  p.out_stride = out->strides[0];
  p.vocab = (int)V;
  p.history = static_cast<const int32_t *>(history->data);
  p.n_history = history->sizes[0];
  p.offsets = offsets->data;
  p.offsets64 = offsets->dtype == HIPATTN_I64;
  p.prompt = prompt_lens ? static_cast<const int32_t *>(prompt_lens->data) : nullptr;
  p.repetition = repetition ? static_cast<const float *>(repetition->data) : nullptr;
  p.frequency = frequency ? static_cast<const float *>(frequency->data) : nullptr;
  p.presence = presence ? static_cast<const float *>(presence->data) : nullptr;
  if (bias) {
    p.bias = static_cast<const float *>(bias->data);
    p.bias_stride = bias->strides[0];
    p.bias_rows = bias->sizes[0];
  }
  if (mask) {
    p.mask = static_cast<const uint8_t *>(mask->data);
    p.mask_stride = mask->strides[0];
    p.mask_bytes = mask->sizes[1];
    p.mask_rows = mask->sizes[0];
  }
  p.rows = rows ? static_cast<const int32_t *>(rows->data) : nullptr;
  hipStream_t stream = resolve_stream(stream_arg);
  p.num_seqs = (int)S;
  p.tiles = (int)((V + 7 + kTile - 1) / kTile);  // (a row may begin up to 7 tokens behind a boundary)
  const int64_t n_wg = (S + 7) / 8 * 8 * p.tiles;
  HA_CHECK(n_wg <= 0x7fffffff, "penalize_logits: too many workgroups");
  const dim3 grid((unsigned)n_wg);
#define HA_PEN(TT, OO)                                                                        \
  if (bias && mask) penalties_kernel<TT, OO, true, true><<<grid, kThreads, 0, stream>>>(p);   \
  else if (bias) penalties_kernel<TT, OO, true, false><<<grid, kThreads, 0, stream>>>(p);     \
  else if (mask) penalties_kernel<TT, OO, false, true><<<grid, kThreads, 0, stream>>>(p);     \
  else penalties_kernel<TT, OO, false, false><<<grid, kThreads, 0, stream>>>(p)
  const bool wide = out->dtype == HIPATTN_F32;
  switch (logits->dtype) {
    case HIPATTN_F32: HA_PEN(float, float); break;
    case HIPATTN_F16:
      if (wide) { HA_PEN(half_t, float); } else { HA_PEN(half_t, half_t); }
      break;
    default:
      if (wide) { HA_PEN(bf16_t, float); } else { HA_PEN(bf16_t, bf16_t); }
      break;
  }
#undef HA_PEN
  check_launch("penalize_logits");
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" char *hipattn_penalize_logits(hipattn_tensor *out, const hipattn_tensor *logits, const hipattn_tensor *history,
                                         const hipattn_tensor *history_offsets, const hipattn_tensor *prompt_lens,
                                         const hipattn_tensor *repetition, const hipattn_tensor *frequency, const hipattn_tensor *presence,
                                         const hipattn_tensor *bias, const hipattn_tensor *mask, const hipattn_tensor *bias_rows,
                                         void *stream) {
  HA_PROTECT(penalize_logits_impl(out, logits, history, history_offsets, prompt_lens, repetition, frequency, presence, bias, mask, bias_rows,
                                  stream));
}
