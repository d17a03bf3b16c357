// A step's block bookkeeping on the device: from how many tokens every request brings, the blocks of the paged cache that go back to the
// pool and those that are taken, the block tables, and every row's position and slot.  What BlockAllocator and BatchInfoBuilder do on the
// host (rllm/rllm-cuda/src/llm/paged/blocks.rs:157-243, batch_info.rs:196-315) for sequences that share no blocks, so that a step needs
// nothing from the host but its launches.
//
//   held = ceil(kv / BS); back = the columns [ceil(sinks / BS), floor((kv - window_left) / BS)) that are not gone yet, or all of a request
//   that has ended; need = ceil((kv + new) / BS) - held.  Blocks leave the ring of free blocks at its head and come back at its tail, in
//   the order of requests and columns; a request is served as long as the sums of `need` and of `new` up to it stay within what is free
//   and within the rows.
//
// It is bound by latency: three running sums over the requests, and a few words per request, row and block.  step_requests_kernel, one
// workgroup, does the sums and what is said of each request; step_rows, spread over the launch's threads, moves the blocks and fills the
// rows, each finding its request by a search in the sums.  Small steps have both in the one workgroup.
#include "common.h"
#include "device_types.h"

namespace hipattn {

namespace {

struct StepParams {
  const int32_t *new_lens;  // [R]
  const int2 *state;        // [R]: tokens in the cache, columns gone
  int32_t *tables;          // [R, cols]
  int64_t table_stride;
  int32_t *ring;  // [nb]
  const int64_t *ends;  // head, tail
  int R, cols, nb, log2_bs, T, per_request, window_left, sinks;
  int2 *state_out;
  int64_t *ends_out;
  int32_t *served, *context_lens, *cu, *logit_idxs;
  int64_t *positions;
  int32_t *slots, *totals;
  int4 *moves;  // [R + 1]: blocks given back and taken by the requests in front, columns [0, z) and from w on that are given back
};

// Sums in front of each thread's value, over the workgroup's wavefronts; `total` is all of them.  Order and result do not depend on anything
// but the values.
template <typename V>
__device__ __forceinline__ V sums_before(V v, V *s_wave, V &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  V inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V t = __shfl_up(inc, o, 64);
    if (lane >= o) inc += t;
  }
  __syncthreads();  // s_wave may still be read from the sums before
  if (lane == 63) s_wave[wave] = inc;
  __syncthreads();
  V before = inc - v;
  total = 0;
  for (int w = 0; w < waves; w++) {
    const V x = s_wave[w];
    before += w < wave ? x : 0;
    total += x;
  }
  return before;
}

// The last request whose sum is at most i; sums[0] = 0 and i < sums[n].
__device__ __forceinline__ int owner_of(const int *sums, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Blocks back to the ring, blocks out of it into the tables, and the rows.  back, taken, cu: [R + 1] sums.  Nothing that is read here is
// written here: what is given back lies in columns that are held, what is taken goes to columns behind them, and what is read of the
// ring are the blocks that were free -- where a step needs more, it finds those that come back in the table they come from.
__device__ __forceinline__ void step_rows(const StepParams &p, const int *back, const int *taken, const int *cu, int first, int stride) {
  const int n_back = back[p.R], n_taken = taken[p.R], bs = 1 << p.log2_bs;
  const int64_t head = p.ends_out[0] - n_taken, tail = p.ends_out[1] - n_back;
  const int64_t free_before = tail - head;
  const unsigned nb = (unsigned)p.nb, head_at = (unsigned)((head % p.nb + p.nb) % p.nb), tail_at = (unsigned)((tail % p.nb + p.nb) % p.nb);
  auto given_back = [&](int i) -> int32_t {
    const int r = owner_of(back, p.R, i);
    const int j = i - back[r];
    const int4 m = p.moves[r];
    return p.tables[r * p.table_stride + (j < m.z ? j : m.w + (j - m.z))];
  };
  auto taken_block = [&](int i) -> int32_t {
    return i < free_before ? p.ring[(head_at + (unsigned)i) % nb] : given_back((int)(i - free_before));
  };
  for (int i = first; i < n_back; i += stride) p.ring[(tail_at + (unsigned)i) % nb] = given_back(i);
  auto held_before = [&](int r) -> int {  // tokens that were in the cache
    return p.state_out[r].x - (cu[r + 1] - cu[r]);
  };
  for (int i = first; i < n_taken; i += stride) {
    const int r = owner_of(taken, p.R, i);
    const int held = (held_before(r) + bs - 1) >> p.log2_bs;
    p.tables[r * p.table_stride + held + (i - taken[r])] = taken_block(i);
  }
  const int rows = p.per_request > 0 ? p.R * p.per_request : cu[p.R];
  for (int t = first; t < p.T; t += stride) {
    int64_t pos = 0;
    int slot = -1;
    if (t < rows) {
      const int r = p.per_request > 0 ? t / p.per_request : owner_of(cu, p.R, t);
      const int at = t - (p.per_request > 0 ? r * p.per_request : cu[r]);
      if (at < cu[r + 1] - cu[r]) {
        const int kv = held_before(r), held = (kv + bs - 1) >> p.log2_bs;
        pos = kv + at;
        const int col = (kv + at) >> p.log2_bs;
        const int block = col < held ? p.tables[r * p.table_stride + col] : taken_block(taken[r] + col - held);
        slot = block * bs + ((kv + at) & (bs - 1));
      }
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
}

constexpr int kFusedRequests = 1024;  // what the one workgroup keeps the sums of in LDS

// FUSED: at most kFusedRequests requests, and the blocks and rows as well.
template <bool FUSED>
__global__ __launch_bounds__(1024) void step_requests_kernel(StepParams p) {
  __shared__ int64_t s_wide[16];
  __shared__ int s_wave[16];
  __shared__ int s_back[FUSED ? kFusedRequests + 1 : 1], s_taken[FUSED ? kFusedRequests + 1 : 1], s_cu[FUSED ? kFusedRequests + 1 : 1];
  __shared__ int s_refused;
  const int tid = threadIdx.x, N = blockDim.x, bs = 1 << p.log2_bs;
  const int64_t head = p.ends[0], tail = p.ends[1];
  const int sunk = p.window_left >= 0 ? (p.sinks + bs - 1) >> p.log2_bs : 0;
  if (tid == 0) s_refused = 0;

  struct Request {
    int kv, gone, added, held, dead;
  };
  auto request = [&](int r) -> Request {
    Request q = {0, 0, 0, 0, 0};
    if (r < p.R) {
      const int2 s = p.state[r];
      q.added = p.new_lens[r];
      q.kv = min(max(s.x, 0), p.cols << p.log2_bs);  // (a state that is none reads a wrong column, never outside)
      q.held = (q.kv + bs - 1) >> p.log2_bs;
      q.gone = min(max(s.y, 0), q.held);
      q.dead = p.window_left >= 0 ? max(q.gone, max(q.kv - p.window_left, 0) >> p.log2_bs) : q.gone;
    }
    return q;
  };

  // What goes back.
  int n_back = 0;
  for (int r0 = 0; r0 < p.R; r0 += N) {
    const int r = r0 + tid;
    const Request q = request(r);
    const bool ended = q.added < 0;
    // columns [0, in_sinks) and [behind, end)
    const int in_sinks = ended ? min(sunk, q.held) : 0, behind = max(q.gone, sunk), end = ended ? q.held : q.dead;
    int total;
    const int before = n_back + sums_before(in_sinks + max(end - behind, 0), s_wave, total);
    if (r < p.R) {
      p.moves[r] = make_int4(before, 0, in_sinks, behind);
      if (FUSED) s_back[r] = before;
    }
    n_back += total;
  }
  const int64_t free_blocks = tail - head + n_back;

  // Who is served.  The sums run over everyone who could be, so that nobody overtakes a request that has to wait.
  int64_t want_before = 0, need_before = 0;
  int n_rows = 0, n_taken = 0;
  for (int r0 = 0; r0 < p.R; r0 += N) {
    const int r = r0 + tid;
    const Request q = request(r);
    const bool fits = (int64_t)q.kv + q.added <= ((int64_t)p.cols << p.log2_bs) && q.added <= (p.per_request > 0 ? p.per_request : p.T);
    const int want = q.added > 0 && fits ? q.added : 0;
    const int need = want > 0 ? ((q.kv + want + bs - 1) >> p.log2_bs) - q.held : 0;
    int64_t want_total, need_total;
    const int64_t want_to = want_before + sums_before<int64_t>(want, s_wide, want_total) + want;
    const int64_t need_to = need_before + sums_before<int64_t>(need, s_wide, need_total) + need;
    want_before += want_total;
    need_before += need_total;
    const bool lasts = need_to <= free_blocks && (p.per_request > 0 || want_to <= p.T);
    const int given = lasts ? want : 0, taken = lasts ? need : 0;
    int rows_total, taken_total;
    const int row = n_rows + sums_before(given, s_wave, rows_total);
    const int block = n_taken + sums_before(taken, s_wave, taken_total);
    n_rows += rows_total;
    n_taken += taken_total;
    if (r < p.R) {
      const bool ended = q.added < 0;
      const int served = q.added > 0 && !fits ? -2 : (want > 0 && !lasts ? -1 : given);
      if (served < 0) atomicAdd(&s_refused, 1);
      p.state_out[r] = ended ? make_int2(0, 0) : make_int2(q.kv + given, q.dead);
      p.served[r] = served;
      p.context_lens[r] = given > 0 ? q.kv + given : 0;
      p.cu[r] = row;
      p.logit_idxs[r] = given > 0 ? (p.per_request > 0 ? r * p.per_request : row) + given - 1 : 0;
      p.moves[r].y = block;
      if (FUSED) {
        s_cu[r] = row;
        s_taken[r] = block;
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    p.cu[p.R] = n_rows;
    p.moves[p.R] = make_int4(n_back, n_taken, 0, 0);
    p.ends_out[0] = head + n_taken;
    p.ends_out[1] = tail + n_back;
    p.totals[0] = n_rows;
    p.totals[1] = s_refused;
    p.totals[2] = (int)(tail + n_back - head - n_taken);
    p.totals[3] = n_taken;
    if (FUSED) {
      s_cu[p.R] = n_rows;
      s_back[p.R] = n_back;
      s_taken[p.R] = n_taken;
    }
  }
  if constexpr (FUSED) {
    __syncthreads();
    step_rows(p, s_back, s_taken, s_cu, tid, N);
  }
}

constexpr int kSearchRequests = 4096;  // more are searched in memory

__global__ __launch_bounds__(256) void step_rows_kernel(StepParams p) {
  __shared__ int s_back[kSearchRequests + 1], s_taken[kSearchRequests + 1], s_cu[kSearchRequests + 1];
  // (the sums of back and taken lie four words apart in `moves`)
  for (int r = threadIdx.x; r <= p.R; r += 256) {
    const int4 m = p.moves[r];
    s_back[r] = m.x;
    s_taken[r] = m.y;
    s_cu[r] = p.cu[r];
  }
  __syncthreads();
  step_rows(p, s_back, s_taken, s_cu, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

void check_i32(const hipattn_tensor *t, const char *name, int ndim, int64_t a, int64_t b = 0) {
  check_tensor(t, name, ndim);
  HA_CHECK(t->dtype == HIPATTN_I32, "step_blocks: %s must be int32, got %s", name, dtype_name(t->dtype));
  HA_CHECK(t->sizes[0] == a && (ndim < 2 || t->sizes[1] == b), "step_blocks: %s has the wrong shape", name);
  check_contiguous(t, name);
  check_data(t, name);
}

void check_i64(const hipattn_tensor *t, const char *name, int64_t a) {
  check_tensor(t, name, 1);
  HA_CHECK(t->dtype == HIPATTN_I64, "step_blocks: %s must be int64, got %s", name, dtype_name(t->dtype));
  HA_CHECK(t->sizes[0] == a, "step_blocks: %s has the wrong shape", name);
  check_contiguous(t, name);
  check_data(t, name);
}

void step_blocks_impl(const hipattn_tensor *new_lens, const hipattn_tensor *state, hipattn_tensor *tables, hipattn_tensor *ring,
                      const hipattn_tensor *ends, int block_size, int per_request, int window_left, int sinks, hipattn_tensor *state_out,
                      hipattn_tensor *ends_out, hipattn_tensor *served, hipattn_tensor *context_lens, hipattn_tensor *cu,
                      hipattn_tensor *logit_idxs, hipattn_tensor *positions, hipattn_tensor *slots, hipattn_tensor *totals,
                      hipattn_tensor *moves, void *stream_arg) {
  check_tensor(new_lens, "new_lens", 1);
  const int64_t R = new_lens->sizes[0];
  HA_CHECK(R >= 1, "step_blocks: no requests");
  HA_CHECK(R <= kSearchRequests, "step_blocks: %lld requests, at most %d", (long long)R, kSearchRequests);
  HA_CHECK(block_size == 8 || block_size == 16 || block_size == 32, "step_blocks: unsupported block size %d (supported: 8, 16, 32)",
           block_size);
  HA_CHECK(sinks >= 0, "step_blocks: sink_tokens must not be negative, got %d", sinks);
  HA_CHECK(per_request >= 0, "step_blocks: rows_per_request must not be negative, got %d", per_request);
  check_i32(new_lens, "new_lens", 1, R);
  check_i32(state, "state", 2, R, 2);
  check_i32(state_out, "state_out", 2, R, 2);
  HA_CHECK(((reinterpret_cast<uintptr_t>(state->data) | reinterpret_cast<uintptr_t>(state_out->data)) & 7) == 0,
           "step_blocks: state must be 8-byte aligned");
  check_tensor(tables, "block_tables", 2);
  HA_CHECK(tables->dtype == HIPATTN_I32, "step_blocks: block_tables must be int32, got %s", dtype_name(tables->dtype));
  const int64_t cols = tables->sizes[1];
  HA_CHECK(tables->sizes[0] == R && cols >= 1, "step_blocks: block_tables needs %lld rows and a column", (long long)R);
  HA_CHECK(cols == 1 || tables->strides[1] == 1, "step_blocks: block_tables rows must be contiguous");
  HA_CHECK(R == 1 || tables->strides[0] >= cols, "step_blocks: block_tables rows must not overlap");
  HA_CHECK(cols * block_size < (int64_t)1 << 30 && R * cols < (int64_t)1 << 31, "step_blocks: block_tables is too large");
  check_data(tables, "block_tables");
  check_tensor(ring, "free_ring", 1);
  const int64_t nb = ring->sizes[0];
  check_i32(ring, "free_ring", 1, nb);
  HA_CHECK(nb >= 1 && nb * block_size < (int64_t)1 << 31, "step_blocks: the slots of %lld blocks do not fit 32 bits, or there are none",
           (long long)nb);
  check_i64(ends, "ring_ends", 2);
  check_i64(ends_out, "ring_ends_out", 2);
  check_i32(served, "served", 1, R);
  check_i32(context_lens, "context_lens", 1, R);
  check_i32(cu, "seqlens_q", 1, R + 1);
  check_i32(logit_idxs, "logit_idxs", 1, R);
  check_tensor(positions, "positions", 1);
  const int64_t T = positions->sizes[0];
  HA_CHECK(T >= 1 && T < (int64_t)1 << 30, "step_blocks: %lld rows, at least 1 and below 2^30", (long long)T);
  HA_CHECK(R * per_request <= T, "step_blocks: %lld requests of %d rows each do not fit %lld rows", (long long)R, per_request, (long long)T);
  check_i64(positions, "positions", T);
  check_i32(slots, "slot_mapping", 1, T);
  check_i32(totals, "totals", 1, 4);
  check_i32(moves, "workspace", 2, R + 1, 4);
  HA_CHECK((reinterpret_cast<uintptr_t>(moves->data) & 15) == 0, "step_blocks: workspace must be 16-byte aligned");
  StepParams p;
  p.new_lens = static_cast<const int32_t *>(new_lens->data);
  p.state = static_cast<const int2 *>(state->data);
  p.tables = static_cast<int32_t *>(tables->data);
  p.table_stride = tables->strides[0];
  p.ring = static_cast<int32_t *>(ring->data);
  p.ends = static_cast<const int64_t *>(ends->data);
  p.R = (int)R;
  p.cols = (int)cols;
  p.nb = (int)nb;
  p.log2_bs = block_size == 8 ? 3 : (block_size == 16 ? 4 : 5);
  p.T = (int)T;
  p.per_request = per_request;
  p.window_left = window_left < 0 ? -1 : window_left;
  p.sinks = sinks < 1 << 30 ? sinks : 1 << 30;
  p.state_out = static_cast<int2 *>(state_out->data);
  p.ends_out = static_cast<int64_t *>(ends_out->data);
  p.served = static_cast<int32_t *>(served->data);
  p.context_lens = static_cast<int32_t *>(context_lens->data);
  p.cu = static_cast<int32_t *>(cu->data);
  p.logit_idxs = static_cast<int32_t *>(logit_idxs->data);
  p.positions = static_cast<int64_t *>(positions->data);
  p.slots = static_cast<int32_t *>(slots->data);
  p.totals = static_cast<int32_t *>(totals->data);
  p.moves = static_cast<int4 *>(moves->data);
  hipStream_t stream = resolve_stream(stream_arg);
  if (R <= kFusedRequests && T <= 4096) {
    step_requests_kernel<true><<<1, R <= 256 && T <= 256 ? 256 : 1024, 0, stream>>>(p);
    check_launch("step_blocks");
    return;
  }
  step_requests_kernel<false><<<1, 1024, 0, stream>>>(p);
  check_launch("step_blocks");
  const int64_t wgs = (T + 255) / 256;
  step_rows_kernel<<<dim3((unsigned)(wgs < 256 ? 256 : (wgs > 1024 ? 1024 : wgs))), 256, 0, stream>>>(p);
  check_launch("step_blocks (rows)");
}

}  // namespace
}  // namespace hipattn

using namespace hipattn;

extern "C" char *hipattn_step_blocks(const hipattn_tensor *new_lens, const hipattn_tensor *state, hipattn_tensor *block_tables,
                                     hipattn_tensor *free_ring, const hipattn_tensor *ring_ends, int block_size, int rows_per_request,
                                     int window_size_left, int sink_tokens, hipattn_tensor *state_out, hipattn_tensor *ring_ends_out,
                                     hipattn_tensor *served, hipattn_tensor *context_lens, hipattn_tensor *seqlens_q,
                                     hipattn_tensor *logit_idxs, hipattn_tensor *positions, hipattn_tensor *slot_mapping,
                                     hipattn_tensor *totals, hipattn_tensor *workspace, void *stream) {
  HA_PROTECT(step_blocks_impl(new_lens, state, block_tables, free_ring, ring_ends, block_size, rows_per_request, window_size_left,
                              sink_tokens, state_out, ring_ends_out, served, context_lens, seqlens_q, logit_idxs, positions, slot_mapping,
                              totals, workspace, stream));
}
