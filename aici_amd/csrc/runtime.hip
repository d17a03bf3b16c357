// Device runtime plumbing of the C ABI: streams, events, memory figures,
// the calling thread's current stream and the library-owned split-K workspace.
// Counterpart of rllm/tch-cuda/kernels/cuda.cpp:32-149 without libtorch.
#include <algorithm>
#include <atomic>
#include <map>
#include <mutex>
#include <utility>
#include <vector>

#include "common.h"
#include "workspace.h"

struct hipattn_stream {
  hipStream_t raw;
  int device;
  bool owned;  // created by this library (pool stream)
  std::atomic<int> *refs;
};

struct hipattn_event {
  hipEvent_t raw;
};

namespace hipattn {

namespace {
thread_local hipStream_t tl_current_stream = nullptr;
std::mutex g_mutex;
int64_t g_peak[64];
int64_t g_lib_allocated[64], g_lib_freed[64];  // bytes of device memory this library itself has allocated / released
constexpr int kMaxDevices = 64;

// Library-owned scratch: one buffer per (op, device, stream).  `retired` holds the buffers that a
// larger one has replaced; enqueued work or a captured graph may still use them, so they live until
// hipattn_shutdown.
struct ScratchKey {
  int user, device;
  hipStream_t stream;
  uint64_t thread;  // 0 but on hipStreamPerThread, one handle for a stream of each thread's own
  bool operator<(const ScratchKey &o) const {
    if (user != o.user) return user < o.user;
    if (device != o.device) return device < o.device;
    if (stream != o.stream) return stream < o.stream;
    return thread < o.thread;
  }
};
uint64_t stream_thread(hipStream_t stream) {
  static std::atomic<uint64_t> threads{0};
  thread_local const uint64_t mine = ++threads;
  return stream == hipStreamPerThread ? mine : 0;
}
struct ScratchBuffer {
  void *ptr = nullptr;
  size_t bytes = 0;
  std::mutex holder;  // of a buffer that several launches of a call share
};
std::map<ScratchKey, ScratchBuffer> g_scratch;
std::vector<std::pair<int, void *>> g_retired;  // (device, pointer)

int env_int(const char *name, int fallback) {
  const char *e = getenv(name);
  return (e != nullptr && *e != '\0') ? atoi(e) : fallback;
}

Tuning tuning_from_env() {
  Tuning t;
  t.decode_flat = env_int("HIPATTN_DECODE_FLAT", -1);
  t.decode_flat_wgs = env_int("HIPATTN_DECODE_FLAT_WGS", 0);
  t.decode_part_blocks = env_int("HIPATTN_DECODE_PART_BLOCKS", 0);
  t.prefill_kernel = env_int("HIPATTN_PREFILL_KERNEL", 0);
  t.paged_prefill_dma = env_int("HIPATTN_PAGED_PREFILL_DMA", -1);
  t.cache_move_lds = env_int("HIPATTN_CACHE_MOVE_LDS", -1);
  t.prefill_wg_heads = env_int("HIPATTN_PREFILL_WG_HEADS", 0);
  t.prefill_rescale_log2 = env_int("HIPATTN_PREFILL_RESCALE_LOG2", 8);
  if (t.prefill_rescale_log2 < 0 || t.prefill_rescale_log2 > 16) t.prefill_rescale_log2 = 8;
  t.window_parts = env_int("HIPATTN_WINDOW_PARTS", 0);
  t.linear_tiles = env_int("HIPATTN_LINEAR_TILES", 0);
  t.linear_waves = env_int("HIPATTN_LINEAR_WAVES", 0);
  t.linear_splits = env_int("HIPATTN_LINEAR_SPLITS", 0);
  return t;
}
Tuning g_tuning = tuning_from_env();  // once, when the library is loaded

struct TuningField {
  const char *name;
  int Tuning::*field;
  int lo, hi;
};
const TuningField kTuningFields[] = {
    {"decode_flat", &Tuning::decode_flat, -1, 1},
    {"decode_flat_wgs", &Tuning::decode_flat_wgs, 0, 1 << 16},
    {"decode_part_blocks", &Tuning::decode_part_blocks, 0, 64},
    {"prefill_kernel", &Tuning::prefill_kernel, 0, 5},
    {"paged_prefill_dma", &Tuning::paged_prefill_dma, -1, 1},
    {"cache_move_lds", &Tuning::cache_move_lds, -1, 1},
    {"prefill_wg_heads", &Tuning::prefill_wg_heads, 0, 8},
    {"prefill_rescale_log2", &Tuning::prefill_rescale_log2, 0, 16},
    {"window_parts", &Tuning::window_parts, 0, 16},
    {"linear_tiles", &Tuning::linear_tiles, 0, 2},
    {"linear_waves", &Tuning::linear_waves, 0, 8},
    {"linear_splits", &Tuning::linear_splits, 0, 32},
};
}  // namespace

const Tuning &tuning() { return g_tuning; }

hipStream_t resolve_stream(void *stream) {
  if (stream != nullptr) return static_cast<hipStream_t>(stream);
  return tl_current_stream;
}

// The buffer of (user, current device, stream), at least `bytes` large; where it has to be allocated, `spare` more.  Its address as it is now
// (a larger one may replace it, which leaves this one alive), and what is to be locked while launches share it.
struct FoundScratch {
  void *ptr;
  std::mutex *holder;
};
static FoundScratch scratch_buffer(WorkspaceUser user, size_t bytes, size_t spare, hipStream_t stream) {
  int dev = 0;
  HA_HIP(hipGetDevice(&dev));
  HA_CHECK(dev >= 0 && dev < kMaxDevices, "device index %d out of range", dev);
  std::lock_guard<std::mutex> lock(g_mutex);
  ScratchBuffer &ws = g_scratch[ScratchKey{(int)user, dev, stream, stream_thread(stream)}];
  if (ws.bytes >= bytes && ws.ptr != nullptr) return FoundScratch{ws.ptr, &ws.holder};
  // Allocating is not something a capture can record, and the graph would keep the old pointer.
  hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
  const hipError_t asked = hipStreamIsCapturing(stream, &capturing);
  if (asked != hipSuccess) {
    (void)hipGetLastError();
    fail("hipStreamIsCapturing failed (%s): cannot tell whether the library's scratch buffer may grow on this stream",
         hipGetErrorString(asked));
  }
  HA_CHECK(capturing == hipStreamCaptureStatusNone,
           "the library's scratch buffer for this stream must grow to %zu bytes, which cannot happen while the stream is "
           "being captured: run the call once outside the capture first, or use the entry point that takes a workspace",
           bytes);
  const size_t want = (bytes + spare + 255) & ~(size_t)255;
  void *fresh = nullptr;
  HA_HIP(hipMalloc(&fresh, want));
  // Counters kept in the buffer start at zero.  The fill goes onto the stream that the buffer belongs to (which is
  // not being captured here), ahead of the kernels that use it.
  hipError_t e = hipMemsetAsync(fresh, 0, want, stream);
  if (e != hipSuccess) {
    (void)hipFree(fresh);
    fail("clearing a new scratch buffer failed: %s", hipGetErrorString(e));
  }
  if (ws.ptr != nullptr) g_retired.emplace_back(dev, ws.ptr);
  g_lib_allocated[dev] += (int64_t)want;
  ws.ptr = fresh;
  ws.bytes = want;
  return FoundScratch{ws.ptr, &ws.holder};
}

static HeldWorkspace hold(const FoundScratch &found) {
  HeldWorkspace ws;
  ws.ptr = found.ptr;
  if (found.holder != nullptr) ws.held = std::unique_lock<std::mutex>(*found.holder);
  return ws;
}

HeldWorkspace library_workspace(WorkspaceUser user, size_t bytes, hipStream_t stream) {
  return hold(scratch_buffer(user, bytes, bytes / 2, stream));
}

// scratch_buffer, or nulls where it throws and while the stream is being captured.
static FoundScratch try_scratch_buffer(WorkspaceUser user, size_t bytes, size_t spare, hipStream_t stream) {
  FoundScratch found = {nullptr, nullptr};
  hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &capturing) != hipSuccess) {
    (void)hipGetLastError();
    return found;
  }
  if (capturing != hipStreamCaptureStatusNone) return found;
  // A capture on some other stream forbids allocations, in every thread unless the thread says otherwise.
  hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
  if (hipThreadExchangeStreamCaptureMode(&mode) != hipSuccess) {
    (void)hipGetLastError();
    return found;
  }
  try {
    found = scratch_buffer(user, bytes, spare, stream);
  } catch (const Error &) {
    (void)hipGetLastError();
  }
  (void)hipThreadExchangeStreamCaptureMode(&mode);
  return found;
}

HeldWorkspace try_library_workspace(WorkspaceUser user, size_t bytes, hipStream_t stream) {
  return hold(try_scratch_buffer(user, bytes, 0, stream));
}

void reserve_library_workspace(WorkspaceUser user, size_t bytes, hipStream_t stream) {
  if (bytes > 0) (void)try_scratch_buffer(user, bytes, bytes / 2, stream);
}

}  // namespace hipattn

using namespace hipattn;

extern "C" void hipattn_free_error(char *msg) { free(msg); }

extern "C" const char *hipattn_version(void) { return "0.1.0"; }

extern "C" char *hipattn_shutdown(void) {
  HA_PROTECT({
    std::lock_guard<std::mutex> lock(g_mutex);
    int cur = 0;
    bool have_cur = hipGetDevice(&cur) == hipSuccess;
    std::vector<std::pair<int, void *>> all = g_retired;
    for (auto &kv : g_scratch)
      if (kv.second.ptr) all.emplace_back(kv.first.device, kv.second.ptr);
    g_retired.clear();
    g_scratch.clear();
    for (int dv = 0; dv < kMaxDevices; dv++) g_lib_freed[dv] = g_lib_allocated[dv];
    int synced = -1;
    for (auto &dp : all) {
      HA_HIP(hipSetDevice(dp.first));
      if (synced != dp.first) {
        HA_HIP(hipDeviceSynchronize());
        synced = dp.first;
      }
      HA_HIP(hipFree(dp.second));
    }
    if (have_cur) (void)hipSetDevice(cur);
  });
}

extern "C" char *hipattn_tuning_set(const char *name, int value) {
  HA_PROTECT({
    HA_CHECK(name != nullptr, "tuning_set: name is NULL");
    for (const TuningField &f : kTuningFields) {
      if (strcmp(name, f.name) == 0) {
        HA_CHECK(value >= f.lo && value <= f.hi, "tuning_set: %s takes values %d..%d, got %d", name, f.lo, f.hi, value);
        g_tuning.*(f.field) = value;
        return nullptr;
      }
    }
    fail("tuning_set: unknown switch '%s'", name);
  });
}

extern "C" char *hipattn_tuning_get(const char *name, int *value) {
  HA_PROTECT({
    HA_CHECK(name != nullptr && value != nullptr, "tuning_get: name or value is NULL");
    for (const TuningField &f : kTuningFields) {
      if (strcmp(name, f.name) == 0) {
        *value = g_tuning.*(f.field);
        return nullptr;
      }
    }
    fail("tuning_get: unknown switch '%s'", name);
  });
}

extern "C" char *hipattn_reset_peak_memory_stats(int device) {
  HA_PROTECT({
    HA_CHECK(device >= 0 && device < kMaxDevices, "device index %d out of range", device);
    std::lock_guard<std::mutex> lock(g_mutex);
    g_peak[device] = 0;
  });
}

extern "C" char *hipattn_empty_cache(void) {
  // There is no caching allocator inside this library.  The scratch buffers it owns are not released
  // here: enqueued work and captured graphs may point at them (hipattn_shutdown releases them).
  return nullptr;
}

extern "C" char *hipattn_get_stats_allocated_bytes(int device, hipattn_mem_stats *outp) {
  HA_PROTECT({
    HA_CHECK(outp != nullptr, "outp is NULL");
    HA_CHECK(device >= 0 && device < kMaxDevices, "device index %d out of range", device);
    int cur = 0;
    HA_HIP(hipGetDevice(&cur));
    if (cur != device) HA_HIP(hipSetDevice(device));
    size_t free_b = 0, total_b = 0;
    hipError_t e = hipMemGetInfo(&free_b, &total_b);
    if (cur != device) (void)hipSetDevice(cur);
    HA_HIP(e);
    std::lock_guard<std::mutex> lock(g_mutex);
    const int64_t used = (int64_t)(total_b - free_b);
    if (used > g_peak[device]) g_peak[device] = used;
    outp->current = used;
    outp->peak = g_peak[device];
    outp->allocated = g_lib_allocated[device];
    outp->freed = g_lib_freed[device];
  });
}

extern "C" char *hipattn_get_device_properties(int device, hipattn_device_props *outp) {
  HA_PROTECT({
    HA_CHECK(outp != nullptr, "outp is NULL");
    hipDeviceProp_t p;
    HA_HIP(hipGetDeviceProperties(&p, device));
    outp->major = p.major;
    outp->minor = p.minor;
    outp->multi_processor_count = p.multiProcessorCount;
    outp->max_threads_per_multi_processor = p.maxThreadsPerMultiProcessor;
    outp->total_memory = (int64_t)p.totalGlobalMem;
  });
}

// --- streams ---------------------------------------------------------------

extern "C" char *hipattn_stream_get(int typ, int device, hipattn_stream **outp) {
  HA_PROTECT({
    HA_CHECK(outp != nullptr, "outp is NULL");
    HA_CHECK(typ >= HIPATTN_STREAM_DEFAULT && typ <= HIPATTN_STREAM_LOW_PRI, "unknown stream type %d", typ);
    hipattn_stream *s = new hipattn_stream{nullptr, device, false, nullptr};
    if (typ == HIPATTN_STREAM_CURRENT) {
      s->raw = tl_current_stream;
    } else if (typ != HIPATTN_STREAM_DEFAULT) {
      // Pool streams: both kinds are created at the default priority.
      int cur = 0;
      hipError_t e = hipGetDevice(&cur);
      if (e == hipSuccess && cur != device) e = hipSetDevice(device);
      if (e == hipSuccess) e = hipStreamCreateWithFlags(&s->raw, hipStreamNonBlocking);
      if (cur != device) (void)hipSetDevice(cur);
      if (e != hipSuccess) {
        delete s;
        fail("hipStreamCreateWithFlags failed: %s", hipGetErrorString(e));
      }
      s->owned = true;
      s->refs = new std::atomic<int>(1);
    }
    *outp = s;
  });
}

extern "C" char *hipattn_stream_free(hipattn_stream *s) {
  HA_PROTECT({
    if (s == nullptr) return nullptr;
    if (s->owned && s->refs->fetch_sub(1) == 1) {
      hipError_t e = hipStreamDestroy(s->raw);
      delete s->refs;
      if (tl_current_stream == s->raw) tl_current_stream = nullptr;
      delete s;
      HA_HIP(e);
      return nullptr;
    }
    delete s;
  });
}

extern "C" char *hipattn_stream_clone(hipattn_stream *s, hipattn_stream **outp) {
  HA_PROTECT({
    HA_CHECK(s != nullptr && outp != nullptr, "stream or outp is NULL");
    if (s->owned) s->refs->fetch_add(1);
    *outp = new hipattn_stream{s->raw, s->device, s->owned, s->refs};
  });
}

extern "C" char *hipattn_stream_query(hipattn_stream *s, int *done) {
  HA_PROTECT({
    HA_CHECK(s != nullptr && done != nullptr, "stream or done is NULL");
    hipError_t e = hipStreamQuery(s->raw);
    if (e == hipSuccess) *done = 1;
    else if (e == hipErrorNotReady) *done = 0;
    else HA_HIP(e);
  });
}

extern "C" char *hipattn_stream_synchronize(hipattn_stream *s) {
  HA_PROTECT({
    HA_CHECK(s != nullptr, "stream is NULL");
    HA_HIP(hipStreamSynchronize(s->raw));
  });
}

extern "C" char *hipattn_stream_set_current(hipattn_stream *s) {
  HA_PROTECT({
    HA_CHECK(s != nullptr, "stream is NULL");
    tl_current_stream = s->raw;
  });
}

extern "C" char *hipattn_stream_device_index(hipattn_stream *s, int *id) {
  HA_PROTECT({
    HA_CHECK(s != nullptr && id != nullptr, "stream or id is NULL");
    *id = s->device;
  });
}

extern "C" char *hipattn_stream_id(hipattn_stream *s, int64_t *id) {
  HA_PROTECT({
    HA_CHECK(s != nullptr && id != nullptr, "stream or id is NULL");
    *id = (int64_t)reinterpret_cast<intptr_t>(s->raw);
  });
}

extern "C" char *hipattn_stream_raw(hipattn_stream *s, void **raw) {
  HA_PROTECT({
    HA_CHECK(s != nullptr && raw != nullptr, "stream or raw is NULL");
    *raw = static_cast<void *>(s->raw);
  });
}

// --- events ----------------------------------------------------------------

extern "C" char *hipattn_event_create(bool timing, bool blocking, hipattn_event **outp) {
  HA_PROTECT({
    HA_CHECK(outp != nullptr, "outp is NULL");
    unsigned flags = timing ? hipEventDefault : hipEventDisableTiming;
    if (blocking) flags |= hipEventBlockingSync;
    hipEvent_t ev;
    HA_HIP(hipEventCreateWithFlags(&ev, flags));
    *outp = new hipattn_event{ev};
  });
}

extern "C" char *hipattn_event_record(hipattn_event *e, hipattn_stream *s) {
  HA_PROTECT({
    HA_CHECK(e != nullptr && s != nullptr, "event or stream is NULL");
    HA_HIP(hipEventRecord(e->raw, s->raw));
  });
}

extern "C" char *hipattn_event_block(hipattn_event *e, hipattn_stream *s) {
  HA_PROTECT({
    HA_CHECK(e != nullptr && s != nullptr, "event or stream is NULL");
    HA_HIP(hipStreamWaitEvent(s->raw, e->raw, 0));
  });
}

extern "C" char *hipattn_event_elapsed_time(hipattn_event *e, hipattn_event *e2, float *elapsed_ms) {
  HA_PROTECT({
    HA_CHECK(e != nullptr && e2 != nullptr && elapsed_ms != nullptr, "event or output is NULL");
    HA_HIP(hipEventElapsedTime(elapsed_ms, e->raw, e2->raw));
  });
}

extern "C" char *hipattn_event_query(hipattn_event *e, int *done) {
  HA_PROTECT({
    HA_CHECK(e != nullptr && done != nullptr, "event or done is NULL");
    hipError_t r = hipEventQuery(e->raw);
    if (r == hipSuccess) *done = 1;
    else if (r == hipErrorNotReady) *done = 0;
    else HA_HIP(r);
  });
}

extern "C" char *hipattn_event_synchronize(hipattn_event *e) {
  HA_PROTECT({
    HA_CHECK(e != nullptr, "event is NULL");
    HA_HIP(hipEventSynchronize(e->raw));
  });
}

extern "C" char *hipattn_event_free(hipattn_event *e) {
  HA_PROTECT({
    if (e == nullptr) return nullptr;
    hipError_t r = hipEventDestroy(e->raw);
    delete e;
    HA_HIP(r);
  });
}
