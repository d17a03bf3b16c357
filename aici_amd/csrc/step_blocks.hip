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
// It is bound by latency: running sums over the requests, and a few words per request, row and block.  step_requests_kernel, one workgroup,
// does the sums in one round and what is said of each request; step_work, spread over a launch's threads, moves the blocks and fills the
// rows, each item finding its request by a search in the sums.  Small steps have both in the one workgroup; larger ones a launch of workgroups
// that each do the sums for themselves, or, where the state is updated in place, two launches.
// us on the device (a call from Python 10.5, what the host takes to make its outputs): 64 requests, a row each, 5.4 (13.2 with a round of sums
// each for what comes back, is wanted, needed and given, and the three kinds of items one after the other); 301 requests, 8192 rows 6.9 in one
// launch, 4.2 + 4.4 in two; 2048 requests, 131072 rows 8.2, 6.4 + 8.1 in two.  paged.DeviceBlocks updates in place: calls of 9.2, 12.7 and 15.5 us.
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
  int4 *moves;  // [R + 1]: blocks given back and taken by the requests in front, columns [0, z) and those from w on are given back
};

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

// What goes back of a request: columns [0, in_sinks) and [behind, ..), as many as its part of the sums says.
struct Columns {
  int in_sinks, behind;
};

// Blocks back to the ring, blocks out of it into the tables, and the rows.  back, taken, cu: [R + 1] sums; kv(r), columns(r): a request's
// tokens before the step and what goes back of it.  Nothing that is read here is written here: what is given back lies in columns that
// are held, what is taken goes to columns behind them, and what is read of the ring are the blocks that were free -- where a step needs
// more, it finds those that come back in the table they come from.
template <typename KV, typename COLS>
__device__ __forceinline__ void step_work(const StepParams &p, const int *back, const int *taken, const int *cu, KV kv_of, COLS columns_of,
                                          int64_t head, int64_t tail, int first, int stride) {
  const int n_back = back[p.R], n_taken = taken[p.R], bs = 1 << p.log2_bs;
  const int64_t free_before = tail - head;
  const unsigned nb = (unsigned)p.nb, head_at = (unsigned)((head % p.nb + p.nb) % p.nb), tail_at = (unsigned)((tail % p.nb + p.nb) % p.nb);
  auto given_back = [&](int i) -> int32_t {
    const int r = owner_of(back, p.R, i);
    const int j = i - back[r];
    const Columns c = columns_of(r);
    return p.tables[r * p.table_stride + (j < c.in_sinks ? j : c.behind + (j - c.in_sinks))];
  };
  auto taken_block = [&](int i) -> int32_t {
    return i < free_before ? p.ring[(head_at + (unsigned)i) % nb] : given_back((int)(i - free_before));
  };
  const int rows = p.per_request > 0 ? p.R * p.per_request : cu[p.R];
  // One run over all items: a thread's next one does not wait for the stores of the last.
  const int64_t items = (int64_t)p.T + n_taken + n_back;
  for (int64_t item = first; item < items; item += stride) {
    if (item < p.T) {
      const int t = (int)item;
      int64_t pos = 0;
      int slot = -1;
      if (t < rows) {
        const int r = p.per_request > 0 ? t / p.per_request : owner_of(cu, p.R, t);
        const int at = t - (p.per_request > 0 ? r * p.per_request : cu[r]);
        if (at < cu[r + 1] - cu[r]) {
          const int kv = kv_of(r), held = (kv + bs - 1) >> p.log2_bs;
          pos = kv + at;
          const int col = (kv + at) >> p.log2_bs;
          const int block = col < held ? p.tables[r * p.table_stride + col] : taken_block(taken[r] + col - held);
          slot = block * bs + ((kv + at) & (bs - 1));
        }
      }
      p.positions[t] = pos;
      p.slots[t] = slot;
    } else if (item < (int64_t)p.T + n_taken) {
      const int i = (int)(item - p.T);
      const int r = owner_of(taken, p.R, i);
      const int held = (kv_of(r) + bs - 1) >> p.log2_bs;
      p.tables[r * p.table_stride + held + (i - taken[r])] = taken_block(i);
    } else {
      const int i = (int)(item - p.T - n_taken);
      p.ring[(tail_at + (unsigned)i) % nb] = given_back(i);
    }
  }
}

constexpr int kThreads = 1024;

// SUMS: one workgroup, the sums and what is said of each request, for step_work_kernel behind it.  ONE: the blocks and rows as well.  MANY: the
// same in several workgroups, each of which does the sums for itself; only the first writes what is said of the requests, which must not lie
// over what the others still read (state_out, ring_ends_out apart from state, ring_ends).
enum { STEP_SUMS, STEP_ONE, STEP_MANY };

// A thread has PER consecutive requests (PER * kThreads >= R).
template <int MODE, int PER>
__global__ __launch_bounds__(kThreads) void step_requests_kernel(StepParams p) {
  constexpr bool FUSED = MODE != STEP_SUMS;
  constexpr int WAVES = kThreads / 64, KEPT = FUSED ? PER * kThreads : 0;
  __shared__ int64_t s_want[WAVES];
  __shared__ int s_need[WAVES], s_came[WAVES];
  __shared__ int s_back[KEPT + 1], s_taken[KEPT + 1], s_cu[KEPT + 1];
  __shared__ int s_kv[PER == 1 ? KEPT + 1 : 1];  // (more of them are worked out again where they are asked for)
  __shared__ Columns s_columns[PER == 1 ? KEPT + 1 : 1];
  const bool says = MODE != STEP_MANY || blockIdx.x == 0;
  __shared__ int s_refused, s_rows, s_blocks;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bs = 1 << p.log2_bs;
  const int64_t head = p.ends[0], tail = p.ends[1];
  const int sunk = p.window_left >= 0 ? (p.sinks + bs - 1) >> p.log2_bs : 0;
  if (tid == 0) s_refused = s_rows = s_blocks = 0;

  struct Request {
    int added, kv, held, gone, dead;
    Columns columns;
  };
  auto request = [&](int r) -> Request {
    const int2 s = p.state[r];
    Request q;
    q.added = p.new_lens[r];
    q.kv = min(max(s.x, 0), p.cols << p.log2_bs);  // (a state that is none reads a wrong column, never outside)
    q.held = (q.kv + bs - 1) >> p.log2_bs;
    q.gone = min(max(s.y, 0), q.held);
    q.dead = p.window_left >= 0 ? max(q.gone, max(q.kv - p.window_left, 0) >> p.log2_bs) : q.gone;
    q.columns.in_sinks = q.added < 0 ? min(sunk, q.held) : 0;
    q.columns.behind = max(q.gone, sunk);
    return q;
  };
  Request req[PER];
  int came[PER], want[PER], need[PER];
  bool fits[PER];
  int sum_came = 0, sum_need = 0;
  int64_t sum_want = 0;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const int r = tid * PER + j;
    req[j] = Request{0, 0, 0, 0, 0, {0, 0}};
    if (r < p.R) req[j] = request(r);
    const Request &q = req[j];
    came[j] = q.columns.in_sinks + max((q.added < 0 ? q.held : q.dead) - q.columns.behind, 0);
    fits[j] = (int64_t)q.kv + q.added <= ((int64_t)p.cols << p.log2_bs) && q.added <= (p.per_request > 0 ? p.per_request : p.T);
    want[j] = q.added > 0 && fits[j] ? q.added : 0;
    need[j] = want[j] > 0 ? ((q.kv + want[j] + bs - 1) >> p.log2_bs) - q.held : 0;
    sum_came += came[j];
    sum_need += need[j];
    sum_want += want[j];
  }
  // The three sums in front of the thread's requests.
  int to_came = sum_came, to_need = sum_need;
  int64_t to_want = sum_want;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int a = __shfl_up(to_came, o, 64), b = __shfl_up(to_need, o, 64);
    const int64_t c = __shfl_up(to_want, o, 64);
    if (lane >= o) {
      to_came += a;
      to_need += b;
      to_want += c;
    }
  }
  if (lane == 63) {
    s_came[wave] = to_came;
    s_need[wave] = to_need;
    s_want[wave] = to_want;
  }
  __syncthreads();
  int back_before = to_came - sum_came, need_before = to_need - sum_need, n_back = 0, all_need = 0;
  int64_t want_before = to_want - sum_want, all_want = 0;
  const int waves = min((p.R + 64 * PER - 1) / (64 * PER), WAVES);  // (behind them nothing is wanted)
  for (int w = 0; w < waves; w++) {
    if (w == wave) {
      back_before += n_back;
      need_before += all_need;
      want_before += all_want;
    }
    n_back += s_came[w];
    all_need += s_need[w];
    all_want += s_want[w];
  }
  // Who is served: the sums run over everyone who could be, so that nobody overtakes a request that has to wait, and those served are the
  // first of them.
  const int64_t free_blocks = tail - head + n_back;
  auto lasts = [&](int64_t want_to, int need_to) { return need_to <= free_blocks && (p.per_request > 0 || want_to <= p.T); };
  int n_rows = (int)all_want, n_taken = all_need;
  if (!lasts(all_want, all_need)) {  // uniform
    int64_t to_w = want_before;
    int to_n = need_before;
    int rows = 0, blocks = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      to_w += want[j];
      to_n += need[j];
      if (lasts(to_w, to_n)) {
        rows = (int)to_w;
        blocks = to_n;
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      rows = max(rows, __shfl_xor(rows, o, 64));
      blocks = max(blocks, __shfl_xor(blocks, o, 64));
    }
    if (lane == 0) {
      atomicMax(&s_rows, rows);
      atomicMax(&s_blocks, blocks);
    }
    __syncthreads();
    n_rows = s_rows;
    n_taken = s_blocks;
  }
  int refused = 0;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const int r = tid * PER + j;
    const int row = (int)min(want_before, (int64_t)n_rows), block = min(need_before, n_taken);
    want_before += want[j];
    need_before += need[j];
    const bool given_all = want[j] > 0 && lasts(want_before, need_before);
    const int given = given_all ? want[j] : 0;
    const Request &q = req[j];
    const int served = q.added > 0 && !fits[j] ? -2 : (want[j] > 0 && !given_all ? -1 : given);
    if (r < p.R) {
      refused += served < 0;
      if (says) {
        p.state_out[r] = q.added < 0 ? make_int2(0, 0) : make_int2(q.kv + given, q.dead);
        p.served[r] = served;
        p.context_lens[r] = given > 0 ? q.kv + given : 0;
        p.cu[r] = row;
        p.logit_idxs[r] = given > 0 ? (p.per_request > 0 ? r * p.per_request : row) + given - 1 : 0;
      }
      if (FUSED) {
        s_back[r] = back_before;
        s_taken[r] = block;
        s_cu[r] = row;
        if (PER == 1) {
          s_kv[r] = q.kv;
          s_columns[r] = q.columns;
        }
      } else {
        p.moves[r] = make_int4(back_before, block, q.columns.in_sinks, q.columns.behind);
      }
    }
    back_before += came[j];
  }
  if (refused > 0) atomicAdd(&s_refused, refused);
  if (FUSED && tid == 0) {
    s_back[p.R] = n_back;
    s_taken[p.R] = n_taken;
    s_cu[p.R] = n_rows;
  }
  __syncthreads();
  if (tid == 0 && says) {
    p.cu[p.R] = n_rows;
    if (!FUSED) p.moves[p.R] = make_int4(n_back, n_taken, 0, 0);
    p.ends_out[0] = head + n_taken;
    p.ends_out[1] = tail + n_back;
    p.totals[0] = n_rows;
    p.totals[1] = s_refused;
    p.totals[2] = (int)(tail + n_back - head - n_taken);
    p.totals[3] = n_taken;
  }
  if constexpr (FUSED)
    step_work(p, s_back, s_taken, s_cu, [&](int r) { return PER == 1 ? s_kv[r] : request(r).kv; },
              [&](int r) { return PER == 1 ? s_columns[r] : request(r).columns; }, head, tail, blockIdx.x * kThreads + tid,
              gridDim.x * kThreads);
}

constexpr int kMostRequests = 4096;

__global__ __launch_bounds__(256) void step_work_kernel(StepParams p) {
  __shared__ int s_back[kMostRequests + 1], s_taken[kMostRequests + 1], s_cu[kMostRequests + 1];
  for (int r = threadIdx.x; r <= p.R; r += 256) {
    const int4 m = p.moves[r];
    s_back[r] = m.x;
    s_taken[r] = m.y;
    s_cu[r] = p.cu[r];
  }
  const int64_t head_out = p.ends_out[0], tail_out = p.ends_out[1];
  __syncthreads();
  step_work(p, s_back, s_taken, s_cu, [&](int r) { return p.state_out[r].x - (s_cu[r + 1] - s_cu[r]); },
            [&](int r) {
              const int4 m = p.moves[r];
              return Columns{m.z, m.w};
            },
            head_out - s_taken[p.R], tail_out - s_back[p.R], blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
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
  HA_CHECK(R <= kMostRequests, "step_blocks: %lld requests, at most %d", (long long)R, kMostRequests);
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
  check_i32(moves, "workspace", 1, 4 * (R + 1));
  HA_CHECK((reinterpret_cast<uintptr_t>(moves->data) & 15) == 0, "step_blocks: workspace must be 16-byte aligned");
  HA_CHECK((state->data == state_out->data || apart(state, state_out)) && (ends->data == ends_out->data || apart(ends, ends_out)),
           "step_blocks: state_out and ring_ends_out must be state and ring_ends or lie apart from them");
  for (const hipattn_tensor *in : {new_lens, state, (const hipattn_tensor *)tables, (const hipattn_tensor *)ring, ends}) {
    for (const hipattn_tensor *o : {served, context_lens, cu, logit_idxs, positions, slots, totals, moves})
      HA_CHECK(apart(in, o), "step_blocks: an output lies over an input");
    HA_CHECK((in == state || apart(in, state_out)) && (in == ends || apart(in, ends_out)),
             "step_blocks: state_out or ring_ends_out lies over another input");
  }
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
  if (R <= kThreads && T <= 4096) {
    step_requests_kernel<STEP_ONE, 1><<<1, kThreads, 0, stream>>>(p);
    check_launch("step_blocks");
    return;
  }
  if (apart(state, state_out) && apart(ends, ends_out)) {
    const int64_t wgs = (T + 511) / 512;
    const dim3 grid((unsigned)(wgs < 64 ? 64 : (wgs > 256 ? 256 : wgs)));
    if (R <= kThreads) step_requests_kernel<STEP_MANY, 1><<<grid, kThreads, 0, stream>>>(p);
    else step_requests_kernel<STEP_MANY, 4><<<grid, kThreads, 0, stream>>>(p);
    check_launch("step_blocks");
    return;
  }
  if (R <= kThreads) step_requests_kernel<STEP_SUMS, 1><<<1, kThreads, 0, stream>>>(p);
  else step_requests_kernel<STEP_SUMS, 4><<<1, kThreads, 0, stream>>>(p);
  check_launch("step_blocks");
  const int64_t wgs = (T + 255) / 256;
  step_work_kernel<<<dim3((unsigned)(wgs < 256 ? 256 : (wgs > 1024 ? 1024 : wgs))), 256, 0, stream>>>(p);
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
