// Penalties for tokens that a sequence has said already, the controller's bias and its allow-mask, on the logits of a batch: what goes in
// front of hipattn_bias_argmax / hipattn_bias_sample (rllm/rllm-cuda/src/llm/tmodel.rs:277-283 applies the bias alone).
//
//   x = l; said: x = x > 0 ? x / repetition : x * repetition; x -= frequency * count + presence * (count > 0); x += bias; barred: x = -inf
//
// with `said` over all of a sequence's tokens and `count` over those behind its prompt.  Computed in fp32, rounded once to the type of the
// output.  A workgroup owns a tile of a row's vocabulary: it counts the sequence's tokens that fall into it in LDS -- whole numbers, so that
// the order of the additions does not matter -- and then streams the logits through.
#include "common.h"
#include "device_types.h"

namespace hipattn {

namespace {

constexpr unsigned kSaid = 0x80000000u;  // in a token's word: said at all; the rest counts what lies behind the prompt

struct PenaltyParams {
  const void *logits;
  void *out;
  int64_t logit_stride, out_stride;
  int vocab, tile;
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

template <typename T, typename O>
__global__ __launch_bounds__(512) void penalties_kernel(PenaltyParams p) {
  extern __shared__ unsigned s_count[];
  const int64_t seq = blockIdx.y;
  const int v0 = blockIdx.x * p.tile, n = min(p.tile, p.vocab - v0);
  const int tid = threadIdx.x;
  for (int i = tid; i < n; i += 512) s_count[i] = 0;
  __syncthreads();
  int64_t begin = p.offsets64 ? static_cast<const int64_t *>(p.offsets)[seq] : static_cast<const int32_t *>(p.offsets)[seq];
  int64_t end = p.offsets64 ? static_cast<const int64_t *>(p.offsets)[seq + 1] : static_cast<const int32_t *>(p.offsets)[seq + 1];
  begin = min(max(begin, (int64_t)0), p.n_history);  // (offsets that are none read wrong tokens, never outside)
  end = min(max(end, begin), p.n_history);
  const int64_t behind = begin + (p.prompt ? p.prompt[seq] : 0);
  for (int64_t i = begin + tid; i < end; i += 512) {
    const int t = p.history[i] - v0;
    if (t >= 0 && t < n) {
      if (i >= behind) atomicAdd(&s_count[t], 1u);
      else atomicOr(&s_count[t], kSaid);
    }
  }
  __syncthreads();
  const float repetition = p.repetition ? p.repetition[seq] : 1.f, frequency = p.frequency ? p.frequency[seq] : 0.f,
              presence = p.presence ? p.presence[seq] : 0.f;
  const int64_t row = p.rows ? (int64_t)p.rows[seq] : seq;
  const T *lg = static_cast<const T *>(p.logits) + seq * p.logit_stride + v0;
  O *out = static_cast<O *>(p.out) + seq * p.out_stride + v0;
  const float *bias = p.bias ? p.bias + min(max(row, (int64_t)0), p.bias_rows - 1) * p.bias_stride + v0 : nullptr;
  const uint8_t *mask = p.mask ? p.mask + min(max(row, (int64_t)0), p.mask_rows - 1) * p.mask_stride : nullptr;
  for (int i = tid; i < n; i += 512) {
    float x = to_float(lg[i]);
    const unsigned c = s_count[i];
    if (c != 0) {
      x = x > 0.f ? x / repetition : x * repetition;
      const unsigned times = c & ~kSaid;
      if (times != 0) x -= frequency * (float)times + presence;
    }
    if (bias) x += bias[i];
    if (mask) {
      const int64_t byte = (v0 + i) >> 3;
      if (byte >= p.mask_bytes || !((mask[byte] >> ((v0 + i) & 7)) & 1)) x = -INFINITY;
    }
    out[i] = from_float<O>(x);
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
  HA_CHECK(S <= 65535, "penalize_logits: at most 65535 sequences per call");
  check_data(logits, "logits");
  check_data(out, "out");
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
  p.tile = 8192;
  const dim3 grid((unsigned)((V + p.tile - 1) / p.tile), (unsigned)S);
  const size_t lds = (size_t)p.tile * sizeof(unsigned);
#define HA_PEN(TT)                                                                                \
  if (out->dtype == logits->dtype) penalties_kernel<TT, TT><<<grid, 512, lds, stream>>>(p);       \
  else penalties_kernel<TT, float><<<grid, 512, lds, stream>>>(p)
  switch (logits->dtype) {
    case HIPATTN_F32: HA_PEN(float); break;
    case HIPATTN_F16: HA_PEN(half_t); break;
    default: HA_PEN(bf16_t); break;
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
