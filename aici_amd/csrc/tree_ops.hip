// Trees of drafted tokens: the positions and masks of their rows, and what of them the model confirms.
//
// A drafter proposes several continuations of a sequence at once, a tree whose root is the sequence's newest token; the model then takes all
// rows of the tree in one step (tree_attn.hip), and the continuation that its own choices follow is kept.  No counterpart in the reference,
// which generates a token at a time.
//
//   tree_rows: a row sees itself and its ancestors, and lies as many tokens behind the context as it has ancestors.  With up(i) the parent:
//     mask(i) |= mask(up(i)), up(i) = up(up(i)) until every up has passed a root: ceil(log2(depth)) rounds in LDS instead of a walk per row
//     (each step of a walk is a load that depends on the last one); the number of ancestors is that of the mask's bits.
//   tree_accept: from row 0, which is no draft, on to the lowest row whose parent is the row in hand and whose token the model has chosen there.
//     The keys and values of the rows on that way then move to the slots right behind the context, in every layer, where the next step looks
//     for them.  A way only goes up in rows and row k of it comes from row k or later: a thread that takes the rows of the way one after the
//     other never overwrites what it still has to read.
#include "cache_geom.h"
#include "common.h"
#include "device_types.h"

namespace hipattn {

namespace {

constexpr int kMostRows = 1024;  // of a tree

struct TreeRowsParams {
  const int32_t *parents, *cu, *context_lens;
  int64_t *positions, *mask;
  int R, T, words;
};

__global__ __launch_bounds__(256) void tree_rows_kernel(TreeRowsParams p) {
  extern __shared__ unsigned long long masks[];  // [rows][words], and the rows' `up` behind them
  const int r = blockIdx.x, tid = threadIdx.x, W = p.words;
  const int begin = p.cu[r], rows = p.cu[r + 1] - begin, first = max(begin, 0), last = min(begin + max(rows, 0), p.T);
  const int n = begin < 0 ? 0 : min(last - first, 64 * W);  // rows that the mask has bits for
  int *up = reinterpret_cast<int *>(masks + (int64_t)64 * W * W);
  for (int i = tid; i < n; i += 256) {
    const int parent = p.parents[begin + i];
    up[i] = parent < i ? parent : -1;  // (a parent comes first)
  }
  for (int i = tid; i < n * W; i += 256) {
    const int row = i / W, w = i - row * W;
    masks[i] = row >> 6 == w ? 1ull << (row & 63) : 0ull;
  }
  __syncthreads();
  for (;;) {
    // Bits are only ever added, those of rows further up: a mask that is read while another thread adds to it holds what it held, or more.
    bool more = false;
    for (int i = tid; i < n * W; i += 256) {
      const int row = i / W, w = i - row * W, a = up[row];
      if (a >= 0) {
        masks[i] |= masks[a * W + w];
        more = true;
      }
    }
    if (!__syncthreads_or(more)) break;
    int next[kMostRows / 256];
#pragma unroll
    for (int k = 0; k < kMostRows / 256; k++) {
      const int i = tid + 256 * k, a = i < n ? up[i] : -1;
      next[k] = a >= 0 ? up[a] : -1;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kMostRows / 256; k++)
      if (tid + 256 * k < n) up[tid + 256 * k] = next[k];
    __syncthreads();
  }
  const int64_t front = (int64_t)p.context_lens[r] - rows;
  for (int i = tid; i < n; i += 256) {
    int depth = -1;
    for (int w = 0; w < W; w++) depth += __popcll(masks[i * W + w]);
    p.positions[begin + i] = front + depth;
  }
  for (int i = tid; i < n * W; i += 256) p.mask[(int64_t)begin * W + i] = (int64_t)masks[i];
  // Rows of no tree, and those beyond max_seqlen_q: nothing is seen.
  auto clear = [&](int from, int to) {
    for (int i = from + tid; i < to; i += 256) {
      p.positions[i] = 0;
      for (int w = 0; w < W; w++) p.mask[(int64_t)i * W + w] = 0;
    }
  };
  clear(first + n, last);
  if (r == 0) clear(0, min(max(p.cu[0], 0), p.T));
  if (r == p.R - 1) clear(min(max(p.cu[p.R], 0), p.T), p.T);
}

struct TreeAcceptParams {
  const int32_t *tokens, *parents, *chosen, *cu;
  const void *slots;
  bool slot64;
  const int64_t *key_ptrs, *value_ptrs;  // [layers]
  CacheGeom g;
  int layers, T, most;  // most: columns of path
  int32_t *lens, *path, *next;
};

// One workgroup per (sequence, layer): each finds the way for itself, the first of a sequence's says it.  A token's values lie in a cache line of
// their own with those of its neighbours for every element of d, and its keys 256 bytes apart, so that what is touched of a few tokens is every line of V in
// their blocks and half of K's: 64 trees of 16 to 61 rows, 8 heads of 128, 32 layers move 33 MB and touch 271 to 279 (lines of 128 bytes, counted from
// their slots; 211 to 219 in sectors of 32), 57 to 59 us at a large copy's rate.  The kernel takes 106 to 114 by itself, the call 144 to 157 among other work (one
// token after the other, not eight at a time, 175): it is not the lines but the waits.  The caches' addresses come out of memory, so loads and stores
// are flat ones, each load stands behind a condition, and compiled each is waited for by itself; K's eight go by way of scratch memory.
constexpr int kBatch = 8;
template <typename E>
__global__ __launch_bounds__(256) void tree_accept_kernel(TreeAcceptParams p) {
  constexpr int X = 16 / sizeof(E);
  __shared__ int s_parent[kMostRows], s_token[kMostRows], s_chosen[kMostRows], s_path[kMostRows], s_len;
  const int r = blockIdx.x, tid = threadIdx.x;
  const int begin = max(p.cu[r], 0), n = min(min(p.cu[r + 1], p.T) - begin, p.most);
  for (int i = tid; i < n; i += 256) {
    s_parent[i] = p.parents[begin + i];
    s_token[i] = p.tokens[begin + i];
    s_chosen[i] = p.chosen[begin + i];
  }
  __syncthreads();
  if (tid < 64) {
    int len = 0, at = n > 0 ? 0 : -1;
    while (at >= 0) {
      if (tid == 0) s_path[len] = at;
      len++;
      const int want = s_chosen[at], from = at;
      at = -1;
      for (int c0 = from + 1; c0 < n && at < 0; c0 += 64) {
        const int c = c0 + tid;
        const unsigned long long hit = __ballot(c < n && s_parent[c] == from && s_token[c] == want);
        if (hit != 0) at = c0 + __builtin_ctzll(hit);
      }
    }
    if (tid == 0) s_len = len;
  }
  __syncthreads();
  const int len = s_len;
  if (blockIdx.y == 0) {
    for (int k = tid; k < p.most; k += 256) p.path[(int64_t)r * p.most + k] = k < len ? s_path[k] : -1;
    if (tid == 0) {
      p.lens[r] = len;
      p.next[r] = len > 0 ? s_chosen[s_path[len - 1]] : -1;
    }
  }
  if (p.slots == nullptr) return;
  // The rows that move, as the elements of the first head's cache where a row of K begins and where the first of V's lies.
  __shared__ int s_moves;
  __shared__ int64_t s_key[2][kBatch], s_value[2][kBatch];
  const int layer = blockIdx.y;
  E *kc = reinterpret_cast<E *>(p.key_ptrs[layer]), *vc = reinterpret_cast<E *>(p.value_ptrs[layer]);
  const int runs = p.g.head_size / X, key_items = p.g.num_heads * runs, items = key_items + p.g.num_heads * p.g.head_size;
  for (int k0 = 1; k0 < len; k0 += kBatch) {
    __syncthreads();
    if (tid < 64) {
      bool moves = false;
      int64_t from = -1, to = -1;
      int from_off = 0, to_off = 0;
      if (tid < kBatch && k0 + tid < len && s_path[k0 + tid] != k0 + tid) {
        const int rows[2] = {s_path[k0 + tid], k0 + tid};
        int64_t slot[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
          slot[i] = p.slot64 ? static_cast<const int64_t *>(p.slots)[begin + rows[i]] : (int64_t)static_cast<const int32_t *>(p.slots)[begin + rows[i]];
        from = slot_block(slot[0], p.g, from_off);
        to = slot_block(slot[1], p.g, to_off);
        moves = from >= 0 && to >= 0;
      }
      const unsigned long long all = __ballot(moves);
      const int at = __popcll(all & ((1ull << tid) - 1));
      if (moves) {
        s_key[0][at] = from * p.g.k_block_stride + from_off * X;
        s_key[1][at] = to * p.g.k_block_stride + to_off * X;
        s_value[0][at] = from * p.g.v_block_stride + from_off;
        s_value[1][at] = to * p.g.v_block_stride + to_off;
      }
      if (tid == 0) s_moves = __popcll(all);
    }
    __syncthreads();
    const int moves = s_moves;
    // All that a batch reads is read before anything is written: a row of the way comes from one that no earlier row of it goes to.
    for (int i = tid; i < items; i += 256) {
      if (i < key_items) {
        const int head = i / runs;
        E *base = kc + head * p.g.k_head_stride + (int64_t)(i - head * runs) * p.g.block_size * X;
        uint4 v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; k++)
          if (k < moves) v[k] = *reinterpret_cast<const uint4 *>(base + s_key[0][k]);
#pragma unroll
        for (int k = 0; k < kBatch; k++)
          if (k < moves) *reinterpret_cast<uint4 *>(base + s_key[1][k]) = v[k];
      } else {
        const int e = i - key_items, head = e / p.g.head_size;
        E *base = vc + head * p.g.v_head_stride + (int64_t)(e - head * p.g.head_size) * p.g.block_size;
        E v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; k++)
          if (k < moves) v[k] = base[s_value[0][k]];
#pragma unroll
        for (int k = 0; k < kBatch; k++)
          if (k < moves) base[s_value[1][k]] = v[k];
      }
    }
  }
}

const int32_t *i32_vector(const hipattn_tensor *t, const char *name, int64_t n, const char *op) {
  check_tensor(t, name, 1);
  HA_CHECK(t->dtype == HIPATTN_I32, "%s: %s must be int32, got %s", op, name, dtype_name(t->dtype));
  HA_CHECK(t->sizes[0] == n, "%s: %s has %lld elements, expected %lld", op, name, (long long)t->sizes[0], (long long)n);
  check_contiguous(t, name);
  check_data(t, name);
  return static_cast<const int32_t *>(t->data);
}

// The sequences' first rows; how many sequences.
int sequences(const hipattn_tensor *cu, const char *op) {
  check_tensor(cu, "seqlens_q", 1);
  HA_CHECK(cu->sizes[0] >= 1 && cu->sizes[0] <= 65536, "%s: seqlens_q must hold the number of sequences (at most 65535) + 1 entries, got %lld", op,
           (long long)cu->sizes[0]);
  return (int)cu->sizes[0] - 1;
}

int tree_rows_of(const hipattn_tensor *parents, const char *op) {
  check_tensor(parents, "parents", 1);
  HA_CHECK(parents->sizes[0] < (int64_t)1 << 30, "%s: %lld rows, below 2^30 are supported", op, (long long)parents->sizes[0]);
  return (int)parents->sizes[0];
}

void tree_rows_impl(const hipattn_tensor *parents, const hipattn_tensor *cu, const hipattn_tensor *context_lens, int max_q,
                    hipattn_tensor *positions, hipattn_tensor *mask, void *stream_arg) {
  const char *op = "tree_rows";
  TreeRowsParams p{};
  p.T = tree_rows_of(parents, op);
  p.R = sequences(cu, op);
  HA_CHECK(max_q >= 0 && max_q <= kMostRows, "%s: trees of at most %d rows, got max_seqlen_q %d", op, kMostRows, max_q);
  p.words = (max_q + 63) / 64;
  p.parents = i32_vector(parents, "parents", p.T, op);
  p.cu = i32_vector(cu, "seqlens_q", p.R + 1, op);
  p.context_lens = i32_vector(context_lens, "context_lens", p.R, op);
  check_tensor(positions, "positions", 1);
  check_tensor(mask, "mask", 2);
  HA_CHECK(positions->dtype == HIPATTN_I64 && mask->dtype == HIPATTN_I64, "%s: positions and mask must be int64", op);
  HA_CHECK(positions->sizes[0] == p.T && mask->sizes[0] == p.T && mask->sizes[1] == p.words,
           "%s: positions must be [%d] and mask [%d, %d]", op, p.T, p.T, p.words);
  check_contiguous(positions, "positions");
  check_contiguous(mask, "mask");
  check_data(positions, "positions");
  check_data(mask, "mask");
  for (const hipattn_tensor *in : {parents, cu, context_lens})
    HA_CHECK(apart(in, positions) && apart(in, mask), "%s: an output lies over an input", op);
  HA_CHECK(p.R > 0 || p.T == 0, "%s: %d rows of no sequence", op, p.T);
  if (p.T == 0 || p.R == 0) return;
  p.positions = static_cast<int64_t *>(positions->data);
  p.mask = static_cast<int64_t *>(mask->data);
  const size_t lds = (size_t)64 * p.words * (p.words * 8 + 4);
  static bool attr_set = false;  // benign race: setting twice is harmless
  if (!attr_set) {
    HA_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(tree_rows_kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                               kMostRows * (kMostRows / 8 + 4)));
    attr_set = true;
  }
  tree_rows_kernel<<<dim3((unsigned)p.R), 256, lds, resolve_stream(stream_arg)>>>(p);
  check_launch(op);
}

void tree_accept_impl(const hipattn_tensor *tokens, const hipattn_tensor *parents, const hipattn_tensor *chosen, const hipattn_tensor *cu, int max_q,
                      const hipattn_tensor *slots, const hipattn_tensor *key_ptrs, const hipattn_tensor *value_ptrs, hipattn_tensor *key0,
                      hipattn_tensor *value0, hipattn_tensor *lens, hipattn_tensor *path, hipattn_tensor *next, void *stream_arg) {
  const char *op = "tree_accept";
  TreeAcceptParams p{};
  p.T = tree_rows_of(parents, op);
  const int R = sequences(cu, op);
  HA_CHECK(max_q >= 0 && max_q <= kMostRows, "%s: trees of at most %d rows, got max_seqlen_q %d", op, kMostRows, max_q);
  p.most = max_q;
  p.tokens = i32_vector(tokens, "tokens", p.T, op);
  p.parents = i32_vector(parents, "parents", p.T, op);
  p.chosen = i32_vector(chosen, "chosen", p.T, op);
  p.cu = i32_vector(cu, "seqlens_q", R + 1, op);
  p.lens = const_cast<int32_t *>(i32_vector(lens, "lens", R, op));
  p.next = const_cast<int32_t *>(i32_vector(next, "next", R, op));
  check_tensor(path, "path", 2);
  HA_CHECK(path->dtype == HIPATTN_I32 && path->sizes[0] == R && path->sizes[1] == max_q, "%s: path must be int32 [%d, %d]", op, R, max_q);
  check_contiguous(path, "path");
  check_data(path, "path");
  p.path = static_cast<int32_t *>(path->data);
  for (const hipattn_tensor *in : {tokens, parents, chosen, cu})
    HA_CHECK(apart(in, lens) && apart(in, path) && apart(in, next), "%s: an output lies over an input", op);
  p.layers = 1;
  int elt = 2;
  if (key_ptrs != nullptr || value_ptrs != nullptr || slots != nullptr) {
    HA_CHECK(key_ptrs != nullptr && value_ptrs != nullptr && slots != nullptr && key0 != nullptr && value0 != nullptr,
             "%s: keys and values are moved with slot_mapping and the caches, or not at all", op);
    check_tensor(key_ptrs, "key_cache_ptrs", 1);
    check_tensor(value_ptrs, "value_cache_ptrs", 1);
    HA_CHECK(key_ptrs->dtype == HIPATTN_I64 && value_ptrs->dtype == HIPATTN_I64 && key_ptrs->sizes[0] == value_ptrs->sizes[0],
             "%s: key_cache_ptrs and value_cache_ptrs must be int64, one for each layer", op);
    check_contiguous(key_ptrs, "key_cache_ptrs");
    check_contiguous(value_ptrs, "value_cache_ptrs");
    check_data(key_ptrs, "key_cache_ptrs");
    check_data(value_ptrs, "value_cache_ptrs");
    HA_CHECK(key_ptrs->sizes[0] <= 65535, "%s: at most 65535 layers, got %lld", op, (long long)key_ptrs->sizes[0]);
    check_index_tensor(slots, "slot_mapping", 1);
    HA_CHECK(slots->sizes[0] == p.T, "%s: %lld slots for %d rows", op, (long long)slots->sizes[0], p.T);
    for (const hipattn_tensor *in : {slots, key_ptrs, value_ptrs})
      HA_CHECK(apart(in, lens) && apart(in, path) && apart(in, next), "%s: an output lies over an input", op);
    p.g = cache_geometry(key0, value0, op);
    elt = dtype_size(key0->dtype);
    HA_CHECK((reinterpret_cast<uintptr_t>(key0->data) & 15) == 0 && p.g.k_block_stride % p.g.x == 0 && p.g.k_head_stride % p.g.x == 0,
             "%s: rows of the key caches' heads must start on 16-byte boundaries", op);
    if (key_ptrs->sizes[0] > 0) {
      p.layers = (int)key_ptrs->sizes[0];
      p.slots = slots->data;
      p.slot64 = slots->dtype == HIPATTN_I64;
      p.key_ptrs = static_cast<const int64_t *>(key_ptrs->data);
      p.value_ptrs = static_cast<const int64_t *>(value_ptrs->data);
    }
  }
  if (R == 0) return;
  hipStream_t stream = resolve_stream(stream_arg);
  const dim3 grid((unsigned)R, (unsigned)p.layers);
  if (elt == 4) tree_accept_kernel<uint32_t><<<grid, 256, 0, stream>>>(p);
  else tree_accept_kernel<uint16_t><<<grid, 256, 0, stream>>>(p);
  check_launch(op);
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" char *hipattn_tree_rows(const hipattn_tensor *parents, const hipattn_tensor *seqlens_q, const hipattn_tensor *context_lens,
                                   int max_seqlen_q, hipattn_tensor *positions, hipattn_tensor *mask, void *stream) {
  HA_PROTECT(tree_rows_impl(parents, seqlens_q, context_lens, max_seqlen_q, positions, mask, stream));
}

extern "C" char *hipattn_tree_accept(const hipattn_tensor *tokens, const hipattn_tensor *parents, const hipattn_tensor *chosen,
                                     const hipattn_tensor *seqlens_q, int max_seqlen_q, const hipattn_tensor *slot_mapping,
                                     const hipattn_tensor *key_cache_ptrs, const hipattn_tensor *value_cache_ptrs, hipattn_tensor *key0,
                                     hipattn_tensor *value0, hipattn_tensor *lens, hipattn_tensor *path, hipattn_tensor *next,
                                     void *stream) {
  HA_PROTECT(tree_accept_impl(tokens, parents, chosen, seqlens_q, max_seqlen_q, slot_mapping, key_cache_ptrs, value_cache_ptrs, key0, value0,
                              lens, path, next, stream));
}
