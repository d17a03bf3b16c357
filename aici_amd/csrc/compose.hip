// One layer's attention as rLLM composes it from the kernels
// (rllm/rllm-cuda/src/llm/mod.rs:132-354 `save_attn`, `compute_varlen_attn`,
// `compute_paged_attn`, `varlen_attn`).
#include "common.h"
#include "step_attn.h"

namespace hipattn {
namespace {

// Rows [begin, end) of a tensor whose first dimension is tokens.
hipattn_tensor rows(const hipattn_tensor *t, int64_t begin, int64_t end) {
  hipattn_tensor r = *t;
  r.sizes[0] = end - begin;
  r.data = static_cast<char *>(t->data) + begin * t->strides[0] * dtype_size(t->dtype);
  return r;
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" char *hipattn_varlen_attn(const hipattn_tensor *q, const hipattn_tensor *k, const hipattn_tensor *v,
                                     hipattn_tensor *key_cache, hipattn_tensor *value_cache,
                                     const hipattn_tensor *slot_mapping, const hipattn_tensor *gather_mapping,
                                     const hipattn_tensor *seqlens_q, const hipattn_tensor *seqlens_k, int64_t q_multi,
                                     int max_seqlen_q, int max_seqlen_k, const hipattn_tensor *paged_block_tables,
                                     const hipattn_tensor *paged_context_lens, int paged_block_size,
                                     int paged_max_context_len, float softmax_scale, hipattn_tensor *gather_k,
                                     hipattn_tensor *gather_v, hipattn_tensor *y, void *stream) {
  HA_PROTECT({
    check_tensor(q, "q", 3);
    check_tensor(k, "k", 3);
    check_tensor(v, "v", 3);
    check_tensor(y, "y", 3);
    const int64_t T = q->sizes[0];
    HA_CHECK(k->sizes[0] == T && v->sizes[0] == T && y->sizes[0] == T, "varlen_attn: q, k, v, y disagree on the token count");
    HA_CHECK(q_multi >= 0 && q_multi <= T, "varlen_attn: q_multi %lld outside [0, %lld]", (long long)q_multi, (long long)T);
    const int num_kv_heads = (int)k->sizes[1];

    // save_attn: every new token's K/V goes into the paged cache first (mod.rs:132-166) -- unless the
    // caller has put it there already (hipattn_rotary_embedding_and_cache) and passes no slots.
    if (slot_mapping) raise(hipattn_reshape_and_cache(k, v, key_cache, value_cache, slot_mapping, stream));

    // compute_varlen_attn (mod.rs:168-278): gather the whole context of the
    // multi-token sequences, then varlen causal attention.  The reference
    // repeats K/V for GQA (mod.rs:214-215); the kernel maps heads instead.
    if (q_multi > 0) {
      HA_CHECK(gather_mapping && gather_k && gather_v && seqlens_q && seqlens_k,
               "varlen_attn: multi-token rows need gather_mapping, gather scratch and seqlens");
      raise(hipattn_gather_cached_kv(gather_k, gather_v, key_cache, value_cache, gather_mapping, stream));
      hipattn_tensor qm = rows(q, 0, q_multi);
      hipattn_tensor ym = rows(y, 0, q_multi);
      raise(hipattn_mha_varlen_fwd(&qm, gather_k, gather_v, seqlens_q, seqlens_k, nullptr, max_seqlen_q, max_seqlen_k, 0.f,
                                   softmax_scale, false, true, -1, -1, &ym, nullptr, stream));
    }
    // compute_paged_attn (mod.rs:280-316): single-token rows.
    if (q_multi < T) {
      HA_CHECK(paged_block_tables && paged_context_lens, "varlen_attn: single-token rows need block tables and context lens");
      hipattn_tensor qs = rows(q, q_multi, T);
      hipattn_tensor ys = rows(y, q_multi, T);
      raise(hipattn_paged_attention_v1(&ys, &qs, key_cache, value_cache, num_kv_heads, softmax_scale, paged_block_tables,
                                       paged_context_lens, paged_block_size, paged_max_context_len, nullptr, stream));
    }
  });
}

extern "C" char *hipattn_varlen_attn_paged(const hipattn_tensor *q, const hipattn_tensor *k, const hipattn_tensor *v,
                                           hipattn_tensor *key_cache, hipattn_tensor *value_cache,
                                           const hipattn_tensor *slot_mapping, const hipattn_tensor *multi_block_tables,
                                           const hipattn_tensor *seqlens_q, const hipattn_tensor *multi_context_lens,
                                           int64_t q_multi, int max_seqlen_q, int max_seqlen_k,
                                           const hipattn_tensor *paged_block_tables,
                                           const hipattn_tensor *paged_context_lens, int paged_block_size,
                                           int paged_max_context_len, float softmax_scale, hipattn_tensor *y,
                                           void *stream) {
  HA_PROTECT({
    check_tensor(q, "q", 3);
    check_tensor(k, "k", 3);
    check_tensor(v, "v", 3);
    check_tensor(y, "y", 3);
    const int64_t T = q->sizes[0];
    HA_CHECK(k->sizes[0] == T && v->sizes[0] == T && y->sizes[0] == T, "varlen_attn: q, k, v, y disagree on the token count");
    HA_CHECK(q_multi >= 0 && q_multi <= T, "varlen_attn: q_multi %lld outside [0, %lld]", (long long)q_multi, (long long)T);
    const int num_kv_heads = (int)k->sizes[1];
    if (slot_mapping) raise(hipattn_reshape_and_cache(k, v, key_cache, value_cache, slot_mapping, stream));
    HA_CHECK(q_multi == 0 || (multi_block_tables && multi_context_lens && seqlens_q),
             "varlen_attn: multi-token rows need their block tables, context lens and seqlens_q");
    hipattn_tensor qm = rows(q, 0, q_multi);
    hipattn_tensor ym = rows(y, 0, q_multi);
    hipattn_tensor qs = rows(q, q_multi, T);
    hipattn_tensor ys = rows(y, q_multi, T);
    if (q_multi > 0 && (q_multi == T || (paged_block_tables && paged_context_lens))) {
      const DecodeCall singles{&qs, key_cache, value_cache, num_kv_heads, softmax_scale, paged_block_tables, paged_context_lens,
                               paged_block_size, paged_max_context_len, nullptr, "paged_attention_v1"};
      if (step_attention(PagedPrefillCall{&qm, key_cache, value_cache, multi_block_tables, seqlens_q, multi_context_lens, max_seqlen_q,
                                          max_seqlen_k, softmax_scale, true},
                         &ym, q_multi < T ? &singles : nullptr, &ys, stream))
        return nullptr;
    }
    if (q_multi > 0)
      raise(hipattn_mha_varlen_fwd_paged(&qm, key_cache, value_cache, multi_block_tables, seqlens_q, multi_context_lens,
                                         max_seqlen_q, max_seqlen_k, softmax_scale, true, &ym, nullptr, stream));
    if (q_multi < T) {
      HA_CHECK(paged_block_tables && paged_context_lens, "varlen_attn: single-token rows need block tables and context lens");
      raise(hipattn_paged_attention_v1(&ys, &qs, key_cache, value_cache, num_kv_heads, softmax_scale, paged_block_tables,
                                       paged_context_lens, paged_block_size, paged_max_context_len, nullptr, stream));
    }
  });
}

extern "C" char *hipattn_varlen_attn_paged_window_ws(const hipattn_tensor *q, const hipattn_tensor *k, const hipattn_tensor *v,
                                                     hipattn_tensor *key_cache, hipattn_tensor *value_cache,
                                                     const hipattn_tensor *slot_mapping, const hipattn_tensor *multi_block_tables,
                                                     const hipattn_tensor *seqlens_q, const hipattn_tensor *multi_context_lens,
                                                     int64_t q_multi, int max_seqlen_q, int max_seqlen_k,
                                                     const hipattn_tensor *paged_block_tables, const hipattn_tensor *paged_context_lens,
                                                     int paged_block_size, int paged_max_context_len, float softmax_scale,
                                                     int window_size_left, int sink_tokens, hipattn_tensor *y,
                                                     const hipattn_tensor *workspace, void *stream) {
  HA_PROTECT({
    check_tensor(q, "q", 3);
    check_tensor(k, "k", 3);
    check_tensor(v, "v", 3);
    check_tensor(y, "y", 3);
    const int64_t T = q->sizes[0];
    HA_CHECK(k->sizes[0] == T && v->sizes[0] == T && y->sizes[0] == T, "varlen_attn: q, k, v, y disagree on the token count");
    HA_CHECK(q_multi >= 0 && q_multi <= T, "varlen_attn: q_multi %lld outside [0, %lld]", (long long)q_multi, (long long)T);
    HA_CHECK(window_size_left >= 0 && sink_tokens >= 0, "varlen_attn: window_size_left and sink_tokens must not be negative here");
    HA_CHECK(q_multi == 0 || (multi_block_tables && multi_context_lens && seqlens_q),
             "varlen_attn: multi-token rows need their block tables, context lens and seqlens_q");
    HA_CHECK(q_multi == T || (paged_block_tables && paged_context_lens), "varlen_attn: single-token rows need block tables and context lens");
    if (slot_mapping) raise(hipattn_reshape_and_cache(k, v, key_cache, value_cache, slot_mapping, stream));
    if (q_multi > 0) {
      hipattn_tensor qm = rows(q, 0, q_multi);
      hipattn_tensor ym = rows(y, 0, q_multi);
      raise(hipattn_mha_varlen_fwd_paged_window(&qm, key_cache, value_cache, multi_block_tables, seqlens_q, multi_context_lens, max_seqlen_q,
                                                max_seqlen_k, softmax_scale, window_size_left, sink_tokens, &ym, nullptr, workspace, stream));
    }
    if (q_multi < T) {
      hipattn_tensor qs = rows(q, q_multi, T);
      hipattn_tensor ys = rows(y, q_multi, T);
      raise(hipattn_paged_attention_window(&ys, &qs, key_cache, value_cache, (int)k->sizes[1], softmax_scale, paged_block_tables,
                                           paged_context_lens, paged_block_size, paged_max_context_len, window_size_left, sink_tokens,
                                           nullptr, workspace, stream));
    }
  });
}

extern "C" char *hipattn_varlen_attn_paged_window(const hipattn_tensor *q, const hipattn_tensor *k, const hipattn_tensor *v,
                                                  hipattn_tensor *key_cache, hipattn_tensor *value_cache,
                                                  const hipattn_tensor *slot_mapping, const hipattn_tensor *multi_block_tables,
                                                  const hipattn_tensor *seqlens_q, const hipattn_tensor *multi_context_lens,
                                                  int64_t q_multi, int max_seqlen_q, int max_seqlen_k,
                                                  const hipattn_tensor *paged_block_tables, const hipattn_tensor *paged_context_lens,
                                                  int paged_block_size, int paged_max_context_len, float softmax_scale,
                                                  int window_size_left, int sink_tokens, hipattn_tensor *y, void *stream) {
  return hipattn_varlen_attn_paged_window_ws(q, k, v, key_cache, value_cache, slot_mapping, multi_block_tables, seqlens_q, multi_context_lens,
                                             q_multi, max_seqlen_q, max_seqlen_k, paged_block_tables, paged_context_lens, paged_block_size,
                                             paged_max_context_len, softmax_scale, window_size_left, sink_tokens, y, nullptr, stream);
}
