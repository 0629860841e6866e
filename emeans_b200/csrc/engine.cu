// The C ABI of the engine: engine and buffer management, argument checks that
// mirror the reference's (core/mod.rs:432-439 check_select, assign.rs:121-147
// check_shapes, crates/emeans-cuda/src/lib.rs:1129-1139), and dispatch of the
// layer-1 ops onto the engine's stream.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <string>
#include <unordered_set>

#include "engine.h"

namespace {

thread_local std::string g_last_error;

template <class F>
int guard(F&& f) {
  try {
    f();
    g_last_error.clear();
    return EB_OK;
  } catch (const eb::Error& err) {
    g_last_error = err.what();
    return err.code;
  } catch (const std::bad_alloc&) {
    g_last_error = "host out of memory";
    return EB_ERROR;
  } catch (const std::exception& err) {
    g_last_error = std::string("internal: ") + err.what();
    return EB_INTERNAL;
  }
}

// The same for calls that give something back. One that succeeds leaves the last
// failed call's message: a garbage collector may release objects before the caller
// has read it.
template <class F>
int release(F&& f) {
  std::string kept = std::move(g_last_error);
  const int rc = guard(f);
  if (rc == EB_OK) g_last_error = std::move(kept);
  return rc;
}

// Makes the engine's device current for the duration of a call.
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(const eb_engine* e) {
    cudaGetDevice(&prev);
    if (prev != e->device) EB_CUDA(cudaSetDevice(e->device));
  }
  ~DeviceGuard() {
    int cur = -1;
    cudaGetDevice(&cur);
    if (prev >= 0 && cur != prev) cudaSetDevice(prev);
  }
};

// Messages are put together only when a check fails.
[[noreturn]] void refuse(const char* what, const char* why) {
  throw eb::Error(EB_INVALID_ARGUMENT, std::string(what) + why);
}

void need(const void* p, const char* what) {
  if (!p) refuse(what, " is null");
}

void need_type(const eb_buf* b, int dtype, const char* what) {
  need(b, what);
  if (b->dtype != dtype)
    refuse(what, dtype == EB_F32 ? " must be an f32 buffer" : " must be a u32 buffer");
}

// An op wrote `b` on the device: drop the caches derived from its contents.
void touched(eb_engine* e, eb_buf* b) {
  if (!b) return;
  b->version++;
  eb::drop_f16(b);
  if (b->xnorm) {
    cudaFreeAsync(b->xnorm, e->stream);
    b->xnorm = nullptr;
  }
}

bool is_float(int dtype) { return dtype == EB_F32 || dtype == EB_BF16 || dtype == EB_F16; }

void need_float(const eb_buf* b, const char* what) {
  need(b, what);
  if (!is_float(b->dtype)) refuse(what, " must be an f32, bf16 or f16 buffer");
}

// The row stride of a matrix argument: `ld`, or the row's length for 0; the
// buffer must hold rows x d at that stride.
size_t need_rows(const eb_buf* b, size_t rows, size_t d, size_t ld, const char* what) {
  if (ld == 0) ld = d;
  if (ld < d) refuse(what, ": the row stride is shorter than a row");
  if (rows > 0 && (b->len < d || rows - 1 > (b->len - d) / ld))
    refuse(what, " is too short for its rows");
  return ld;
}

// Buffers over the same memory, in part or whole.
bool overlap(const eb_buf* a, const eb_buf* b) {
  if (!a || !b || a->len == 0 || b->len == 0) return false;
  const char *pa = static_cast<const char*>(a->ptr), *pb = static_cast<const char*>(b->ptr);
  return pa < pb + b->len * eb::dtype_bytes(b->dtype) && pb < pa + a->len * eb::dtype_bytes(a->dtype);
}

// The buffers of a call (null: not given) are on the engine's GPU. Another
// engine's buffers are taken where it shares the GPU: two engines on one stream,
// or a caller who orders their streams.
void need_here(const eb_engine* e, std::initializer_list<const eb_buf*> bufs) {
  for (const eb_buf* b : bufs)
    eb::ensure(!b || b->device == e->device, "a buffer is on another GPU than the engine");
}

// The part of a buffer that a call uses: its first `len` elements, or (rows of d
// elements `ld` apart) up to the last row's end.
struct Part {
  const char* ptr = nullptr;
  size_t bytes = 0;
  Part(const eb_buf* b, size_t len)
      : ptr(b ? static_cast<const char*>(b->ptr) : nullptr),
        bytes(b ? len * eb::dtype_bytes(b->dtype) : 0) {}
  Part(const eb_buf* b, size_t rows, size_t d, size_t ld) : Part(b, rows ? (rows - 1) * ld + d : 0) {}
  bool meets(const Part& o) const {
    return bytes && o.bytes && ptr < o.ptr + o.bytes && o.ptr < ptr + bytes;
  }
};

// The outputs of a call share no memory with one another, nor with its inputs; a
// pair that may (in place) is not among them.
void need_apart(std::initializer_list<Part> outputs, std::initializer_list<Part> inputs) {
  for (auto a = outputs.begin(); a != outputs.end(); ++a) {
    for (auto b = outputs.begin(); b != a; ++b)
      eb::ensure(!a->meets(*b), "an output overlaps another");
    for (const Part& in : inputs) eb::ensure(!a->meets(in), "an output overlaps an input");
  }
}

// check_select (core/mod.rs:432-439).
void check_select(size_t r0, size_t r1, const eb_buf* ids, size_t n) {
  eb::ensure(r0 <= r1, "bad row range");
  if (ids)
    eb::ensure(r1 <= ids->len, "row range past the ids");
  else
    eb::ensure(r1 <= n, "row range past the data");
}

}  // namespace

namespace eb {

eb_buf* new_buf(eb_engine* e, int dtype, size_t len) {
  auto* b = new eb_buf;
  b->dtype = dtype;
  b->device = e->device;
  b->len = len;
  b->owned = true;
  size_t bytes = std::max<size_t>(len * dtype_bytes(dtype), 16);
  cudaError_t st = cudaMallocAsync(&b->ptr, bytes, e->stream);
  e->device_allocs++;
  if (st != cudaSuccess) {
    delete b;
    throw Error(EB_ERROR, std::string("device allocation of ") + std::to_string(bytes) +
                              " bytes failed: " + cudaGetErrorString(st));
  }
  EB_CUDA(cudaMemsetAsync(b->ptr, 0, bytes, e->stream));
  return b;
}

void free_buf(eb_engine* e, eb_buf* b) {
  if (!b) return;
  drop_f16(b);
  if (b->xnorm) cudaFreeAsync(b->xnorm, e->stream);
  if (b->owned && b->ptr) cudaFreeAsync(b->ptr, e->stream);
  delete b;
}

void set_last_error(const std::string& msg) { g_last_error = msg; }

void sync(eb_engine* e) {
  EB_CUDA(cudaMemcpyAsync(e->h_status, e->d_status, 4, cudaMemcpyDeviceToHost, e->stream));
  EB_CUDA(cudaStreamSynchronize(e->stream));
  uint32_t st = *e->h_status;
  if (st) {
    *e->h_status = 0;
    EB_CUDA(cudaMemsetAsync(e->d_status, 0, 4, e->stream));
    EB_CUDA(cudaStreamSynchronize(e->stream));
    if (st & ST_BAD_LABEL) throw Error(EB_INVALID_ARGUMENT, "label out of range");
    if (st & ST_BAD_ROW) throw Error(EB_INVALID_ARGUMENT, "row id out of range");
    if (st & ST_WAIT_TIMEOUT) throw Error(EB_ERROR, "device-side wait timed out");
    if (st & ST_BAD_STATE) throw Error(EB_INTERNAL, "device-side consistency check failed");
    throw Error(EB_INTERNAL, "device reported status " + std::to_string(st));
  }
}

}  // namespace eb

using eb::ensure;

extern "C" {

const char* eb_last_error(void) { return g_last_error.c_str(); }

const char* eb_version(void) { return "emeans_b200 0.1 (sm_100a)"; }

}  // extern "C"

namespace {

// An engine on a stream of its own, or on the caller's.
int create_engine(int device, bool own_stream, cudaStream_t stream, eb_engine** out) {
  return guard([&] {
    need(out, "out");
    *out = nullptr;
    int count = 0;
    cudaError_t st = cudaGetDeviceCount(&count);
    if (st != cudaSuccess || count == 0)
      throw eb::Error(EB_ERROR, std::string("no CUDA device: ") + cudaGetErrorString(st));
    ensure(device >= 0 && device < count, "device index out of range");
    cudaDeviceProp prop{};
    EB_CUDA(cudaGetDeviceProperties(&prop, device));
    if (prop.major != 10)
      throw eb::Error(EB_ERROR, std::string("emeans_b200 needs an sm_100 (B200) device, got ") +
                                    prop.name + " sm_" + std::to_string(prop.major) +
                                    std::to_string(prop.minor));
    auto* e = new eb_engine;
    e->device = device;
    e->num_sms = prop.multiProcessorCount;
    int prev = -1;
    cudaGetDevice(&prev);
    try {
      EB_CUDA(cudaSetDevice(device));
      e->owns_stream = own_stream;
      e->stream = stream;
      if (own_stream) EB_CUDA(cudaStreamCreateWithFlags(&e->stream, cudaStreamNonBlocking));
      EB_CUDA(cudaMalloc(&e->d_status, 16));
      EB_CUDA(cudaMemset(e->d_status, 0, 16));
      EB_CUDA(cudaMallocHost(&e->h_status, 16));
      *e->h_status = 0;
      EB_CUDA(cudaMalloc(&e->d_counters, 4 * sizeof(unsigned long long)));
      EB_CUDA(cudaMemset(e->d_counters, 0, 4 * sizeof(unsigned long long)));
      const char* sc = getenv("EMEANS_B200_SCREEN");
      if (sc && (sc[0] == '0' || sc[0] == '1' || sc[0] == '2') && sc[1] == 0)
        e->screen_mode = sc[0] - '0';
    } catch (...) {
      if (prev >= 0) cudaSetDevice(prev);
      delete e;
      throw;
    }
    if (prev >= 0) cudaSetDevice(prev);
    *out = e;
  });
}

}  // namespace

extern "C" {

int eb_engine_create(int device, eb_engine** out) {
  return create_engine(device, true, nullptr, out);
}

int eb_engine_create_on(int device, void* stream, eb_engine** out) {
  return create_engine(device, false, static_cast<cudaStream_t>(stream), out);
}

int eb_engine_destroy(eb_engine* e) {
  if (!e) return EB_OK;
  return release([&] {
    DeviceGuard g(e);
    cudaStreamSynchronize(e->stream);
    eb::group_leave(e);
    for (auto& ev : e->screen_ev) {
      cudaEventDestroy(ev.first);
      cudaEventDestroy(ev.second);
    }
    if (e->bound) eb::free_buf(e, e->bound);
    for (auto& kv : e->scratch)
      if (kv.second.p) cudaFreeAsync(kv.second.p, e->stream);
    cudaStreamSynchronize(e->stream);
    if (e->copy_stream) cudaStreamSynchronize(e->copy_stream);
    if (e->down_stream) cudaStreamSynchronize(e->down_stream);
    for (cudaEvent_t v : e->stage_ev)
      if (v) cudaEventDestroy(v);
    for (auto& kv : e->pinned)
      if (kv.second.p) cudaFreeHost(kv.second.p);
    cudaFree(e->d_status);
    cudaFree(e->d_counters);
    cudaFreeHost(e->h_status);
    if (e->copy_stream) cudaStreamDestroy(e->copy_stream);
    if (e->down_stream) cudaStreamDestroy(e->down_stream);
    if (e->owns_stream) cudaStreamDestroy(e->stream);
    delete e;
  });
}

int eb_engine_name(eb_engine* e, char* buf, size_t cap) {
  return guard([&] {
    need(e, "engine");
    need(buf, "buf");
    std::string name = e->screen_mode ? "b200-exact" : "b200-exact-simt";
    ensure(cap > name.size(), "name buffer too small");
    std::memcpy(buf, name.c_str(), name.size() + 1);
  });
}

int eb_flush(eb_engine* e) {
  return guard([&] { need(e, "engine"); });
}

int eb_sync(eb_engine* e) {
  return guard([&] {
    need(e, "engine");
    DeviceGuard g(e);
    eb::sync(e);
  });
}

int eb_engine_stream(eb_engine* e, void** stream) {
  return guard([&] {
    need(e, "engine");
    need(stream, "stream");
    *stream = (void*)e->stream;
  });
}

int eb_get_stats(eb_engine* e, eb_stats* out) {
  return guard([&] {
    need(e, "engine");
    need(out, "out");
    DeviceGuard g(e);
    unsigned long long c[4];
    EB_CUDA(cudaMemcpyAsync(c, e->d_counters, sizeof(c), cudaMemcpyDeviceToHost, e->stream));
    eb::sync(e);
    *out = e->stats;
    out->fallback_rows = c[1];
    out->rescored_candidates = c[2];
  });
}

int eb_test_screen_dead_wait(eb_engine* e, int on) {
  return guard([&] {
    need(e, "engine");
    e->screen_dead_wait = on != 0;
  });
}

int eb_device_allocations(eb_engine* e, uint64_t* count) {
  return guard([&] {
    need(e, "engine");
    need(count, "count");
    *count = e->device_allocs;
  });
}

int eb_set_kernel_timing(eb_engine* e, int on) {
  return guard([&] {
    need(e, "engine");
    e->time_screen = on != 0;
  });
}

int eb_screen_timing(eb_engine* e, double* total_ms, uint64_t* launches, uint64_t* rows) {
  return guard([&] {
    need(e, "engine");
    need(total_ms, "total_ms");
    need(launches, "launches");
    need(rows, "rows");
    DeviceGuard g(e);
    eb::sync(e);
    double ms = 0.0;
    uint64_t r = 0;
    for (size_t u = 0; u < e->screen_ev_used; u++) {
      float t = 0.0f;
      EB_CUDA(cudaEventElapsedTime(&t, e->screen_ev[u].first, e->screen_ev[u].second));
      ms += t;
      r += e->screen_ev_rows[u];
    }
    *total_ms = ms;
    *launches = e->screen_ev_used;
    *rows = r;
    e->screen_ev_used = 0;
  });
}

int eb_set_screen_mode(eb_engine* e, int mode) {
  return guard([&] {
    need(e, "engine");
    ensure(mode >= 0 && mode <= 2, "screen mode must be 0 (off), 1 (auto) or 2 (always)");
    e->screen_mode = mode;
  });
}

int eb_buf_alloc(eb_engine* e, int dtype, size_t len, eb_buf** out) {
  return guard([&] {
    need(e, "engine");
    need(out, "out");
    ensure(eb::dtype_bytes(dtype) != 0, "unknown dtype");
    DeviceGuard g(e);
    *out = eb::new_buf(e, dtype, len);
  });
}

int eb_buf_wrap(eb_engine* e, int dtype, void* dev_ptr, size_t len, eb_buf** out) {
  return guard([&] {
    need(e, "engine");
    need(out, "out");
    ensure(eb::dtype_bytes(dtype) != 0, "unknown dtype");
    ensure(dev_ptr != nullptr || len == 0, "null device pointer");
    ensure(((uintptr_t)dev_ptr & 15) == 0, "device pointer must be 16-byte aligned");
    cudaPointerAttributes attr{};
    if (dev_ptr) {
      EB_CUDA(cudaPointerGetAttributes(&attr, dev_ptr));
      ensure(attr.type == cudaMemoryTypeDevice || attr.type == cudaMemoryTypeManaged,
             "pointer is not device memory");
      ensure(attr.type == cudaMemoryTypeManaged || attr.device == e->device,
             "pointer is on another device");
    }
    auto* b = new eb_buf;
    b->ptr = dev_ptr;
    b->len = len;
    b->dtype = dtype;
    b->device = e->device;
    b->owned = false;
    *out = b;
  });
}

int eb_buf_free(eb_engine* e, eb_buf* b) {
  if (!b) return EB_OK;
  return release([&] {
    need(e, "engine");
    DeviceGuard g(e);
    if (e->bound == b) e->bound = nullptr;
    eb::free_buf(e, b);
  });
}

size_t eb_buf_len(const eb_buf* b) { return b ? b->len : 0; }
void* eb_buf_ptr(const eb_buf* b) { return b ? b->ptr : nullptr; }

int eb_buf_write(eb_engine* e, eb_buf* b, size_t offset, const void* host, size_t len) {
  return guard([&] {
    need(e, "engine");
    need(b, "buffer");
    ensure(offset <= b->len && len <= b->len - offset, "write past the buffer");
    if (len == 0) return;
    need(host, "host");
    DeviceGuard g(e);
    const size_t es = eb::dtype_bytes(b->dtype);
    eb::h2d(e, static_cast<char*>(b->ptr) + offset * es, host, len * es, e->stream);
    b->version++;
    eb::drop_f16(b);
    if (b->xnorm) {
      cudaFreeAsync(b->xnorm, e->stream);
      b->xnorm = nullptr;
    }
  });
}

int eb_buf_read(eb_engine* e, const eb_buf* b, size_t lo, size_t hi, void* host) {
  return guard([&] {
    need(e, "engine");
    need(b, "buffer");
    ensure(lo <= hi && hi <= b->len, "read past the buffer");
    DeviceGuard g(e);
    if (hi > lo) {
      need(host, "host");
      const size_t es = eb::dtype_bytes(b->dtype);
      eb::d2h(e, host, static_cast<const char*>(b->ptr) + lo * es, (hi - lo) * es, e->stream);
    }
    eb::sync(e);
  });
}

int eb_buf_upload(eb_engine* e, int dtype, const void* host, size_t len, eb_buf** out) {
  return guard([&] {
    need(e, "engine");
    need(out, "out");
    ensure(eb::dtype_bytes(dtype) != 0, "unknown dtype");
    ensure(host != nullptr || len == 0, "host is null");
    DeviceGuard g(e);
    eb_buf* b = eb::new_buf(e, dtype, len);
    if (len) eb::h2d(e, b->ptr, host, len * eb::dtype_bytes(dtype), e->stream);
    *out = b;
  });
}

int eb_bind(eb_engine* e, const float* x, size_t n, size_t d, eb_buf** out) {
  return guard([&] {
    need(e, "engine");
    need(out, "out");
    ensure(d > 0, "d must be positive");
    ensure(x != nullptr || n == 0, "x is null");
    DeviceGuard g(e);
    eb_buf* b = eb::new_buf(e, EB_F32, n * d);
    if (n) eb::h2d(e, b->ptr, x, n * d * 4, e->stream);
    b->d = d;
    *out = b;
  });
}

int eb_top1(eb_engine* e, const eb_buf* x, size_t d, const eb_buf* ids, size_t r0, size_t r1,
            const eb_buf* centroids, const eb_buf* cnorm, size_t k, int metric, eb_buf* labels,
            eb_buf* scores) {
  return guard([&] {
    need(e, "engine");
    need_type(x, EB_F32, "x");
    ensure(d > 0, "d must be positive");
    ensure(metric == EB_L2 || metric == EB_IP, "unknown metric");
    if (ids) need_type(ids, EB_U32, "ids");
    need_type(centroids, EB_F32, "centroids");
    need_type(labels, EB_U32, "labels");
    need_type(scores, EB_F32, "scores");
    check_select(r0, r1, ids, x->len / d);
    ensure(r1 <= labels->len && r1 <= scores->len, "outputs too short");
    ensure(k > 0 && centroids->len == k * d, "centroids must be k x d");
    ensure(k <= 0xFFFFFFFFull, "k too large");
    if (metric == EB_L2) {
      ensure(cnorm != nullptr && cnorm->len >= k, "L2 needs centroid norms");
      need_type(cnorm, EB_F32, "cnorm");
    }
    if (r0 == r1) return;
    DeviceGuard g(e);
    touched(e, labels);
    touched(e, scores);
    eb::Top1Args a;
    a.x = static_cast<const float*>(x->ptr);
    a.n = x->len / d;
    a.d = d;
    a.ids = ids ? static_cast<const uint32_t*>(ids->ptr) : nullptr;
    a.r0 = r0;
    a.r1 = r1;
    a.c = static_cast<const float*>(centroids->ptr);
    a.cnorm = cnorm ? static_cast<const float*>(cnorm->ptr) : nullptr;
    a.k = k;
    a.metric = metric;
    a.labels = static_cast<uint32_t*>(labels->ptr);
    a.scores = static_cast<float*>(scores->ptr);
    a.xnorm = (x->xnorm && x->d == d) ? x->xnorm : nullptr;
    if (metric == EB_L2 && !a.xnorm && x->d == d) {
      // Bound data: keep its row norms (CPU float order) for every later call.
      float* xn = nullptr;
      EB_CUDA(cudaMallocAsync(&xn, std::max<size_t>(a.n, 1) * 4, e->stream));
      e->device_allocs++;
      eb::row_norms(e, a.x, a.n, d, xn);
      const_cast<eb_buf*>(x)->xnorm = xn;
      a.xnorm = xn;
    }
    eb::top1_dispatch(e, a, const_cast<eb_buf*>(x));
  });
}

int eb_topk(eb_engine* e, const float* queries, size_t m, const float* data, size_t n, size_t d,
            size_t kk, int exclude_self, uint32_t* ids, float* sims) {
  return guard([&] {
    need(e, "engine");
    ensure(d > 0, "d must be positive");
    ensure(kk >= 1 && kk <= 16, "kk must be 1..=16");
    ensure(n > 0, "no data rows");
    ensure(!exclude_self || m == n, "exclude_self needs queries == data");
    ensure(n <= 0xFFFFFFFEull, "too many data rows");
    if (m == 0) return;
    need(queries, "queries");
    need(data, "data");
    need(ids, "ids");
    need(sims, "sims");
    DeviceGuard g(e);
    eb::topk(e, queries, m, data, n, d, kk, exclude_self != 0, ids, sims);
  });
}

int eb_internal_scores(eb_engine* e, const float* x, size_t n, size_t d, const uint32_t* labels,
                       size_t k, eb_internal* out, uint64_t* sizes) {
  return guard([&] {
    need(e, "engine");
    need(out, "out");
    ensure(d > 0, "x must be n x d");  // metrics.rs:116
    ensure(k <= 0x7FFFFFFFull, "k too large");
    if (n > 0) {
      need(x, "x");
      need(labels, "labels");
    }
    uint32_t bad = 0;
    for (size_t i = 0; i < n; i++) bad |= (uint32_t)(labels[i] >= k);
    ensure(bad == 0, "label out of range");  // metrics.rs:119-122
    DeviceGuard g(e);
    eb::internal_scores(e, x, n, d, labels, k, out, sizes);
  });
}

int eb_topk_group(eb_engine* e, const float* queries, size_t m, const float* shard,
                  size_t n_shard, size_t shard_offset, size_t n_total, size_t d, size_t kk,
                  int exclude_self, uint32_t* ids, float* sims) {
  return guard([&] {
    need(e, "engine");
    ensure(d > 0, "d must be positive");
    ensure(kk >= 1 && kk <= 16, "kk must be 1..=16");
    ensure(n_total > 0 && n_total <= 0xFFFFFFFEull, "n_total must be in 1 .. 2^32 - 2");
    ensure(shard_offset + n_shard <= n_total, "shard past the data");
    ensure(!exclude_self || m == n_total, "exclude_self needs queries == data");
    if (m == 0) return;
    need(queries, "queries");
    if (n_shard) need(shard, "shard");
    need(ids, "ids");
    need(sims, "sims");
    DeviceGuard g(e);
    eb::topk(e, queries, m, shard, n_shard, d, kk, exclude_self != 0, ids, sims, shard_offset,
             true);
  });
}

int eb_scatter_add(eb_engine* e, const eb_buf* x, size_t d, const eb_buf* ids, size_t r0,
                   size_t r1, const eb_buf* labels, size_t k, eb_buf* sums, eb_buf* counts,
                   eb_buf* acc) {
  return guard([&] {
    need(e, "engine");
    need_type(x, EB_F32, "x");
    ensure(d > 0, "d must be positive");
    if (ids) need_type(ids, EB_U32, "ids");
    need_type(labels, EB_U32, "labels");
    need_type(sums, EB_F32, "sums");
    need_type(counts, EB_U32, "counts");
    check_select(r0, r1, ids, x->len / d);
    ensure(sums->len == k * d && counts->len == k, "sums k x d, counts k");
    ensure(k > 0, "k must be positive");
    ensure(r1 <= labels->len, "labels too short");
    if (acc) {
      need_type(acc, EB_F32, "acc");
      ensure(acc->len == k * d, "acc must be k x d");
    }
    DeviceGuard g(e);
    touched(e, sums);
    touched(e, counts);
    touched(e, acc);
    eb::scatter_add(e, static_cast<const float*>(x->ptr), x->len / d, d,
                    ids ? static_cast<const uint32_t*>(ids->ptr) : nullptr, r0, r1,
                    static_cast<const uint32_t*>(labels->ptr), k, static_cast<float*>(sums->ptr),
                    static_cast<uint32_t*>(counts->ptr),
                    acc ? static_cast<float*>(acc->ptr) : nullptr);
  });
}

int eb_row_norms(eb_engine* e, const eb_buf* m, size_t rows, size_t d, eb_buf* out) {
  return guard([&] {
    need(e, "engine");
    need_type(m, EB_F32, "m");
    need_type(out, EB_F32, "out");
    ensure(m->len >= rows * d && out->len >= rows, "shapes");
    DeviceGuard g(e);
    touched(e, out);
    eb::row_norms(e, static_cast<const float*>(m->ptr), rows, d, static_cast<float*>(out->ptr));
  });
}

int eb_normalize_rows(eb_engine* e, const eb_buf* src, size_t rows, size_t d, eb_buf* dst) {
  return guard([&] {
    need(e, "engine");
    need_type(src, EB_F32, "src");
    need_type(dst, EB_F32, "dst");
    ensure(src->len >= rows * d && dst->len >= rows * d, "shapes");
    DeviceGuard g(e);
    touched(e, dst);
    eb::normalize_rows(e, static_cast<const float*>(src->ptr), rows, d,
                       static_cast<float*>(dst->ptr));
  });
}

int eb_split(eb_engine* e, eb_buf* positions, eb_buf* usage, const uint32_t* pairs, size_t npairs,
             size_t d) {
  return guard([&] {
    need(e, "engine");
    need_type(positions, EB_F32, "positions");
    need_type(usage, EB_F32, "usage");
    size_t k = usage->len;
    ensure(positions->len == k * d, "positions must be k x d");
    if (npairs == 0) return;
    need(pairs, "pairs");
    std::unordered_set<uint32_t> seen;
    for (size_t i = 0; i < 2 * npairs; i++) {
      ensure(pairs[i] < k, "split ids out of range");
      ensure(seen.insert(pairs[i]).second, "split pairs must not share ids");
    }
    DeviceGuard g(e);
    touched(e, positions);
    touched(e, usage);
    uint32_t* dp = e->scratch_get<uint32_t>("split_pairs", 2 * npairs);
    EB_CUDA(cudaMemcpyAsync(dp, pairs, 2 * npairs * 4, cudaMemcpyHostToDevice, e->stream));
    eb::split(e, static_cast<float*>(positions->ptr), static_cast<float*>(usage->ptr), dp, npairs,
              d);
  });
}

int eb_ema_update(eb_engine* e, eb_buf* positions, eb_buf* usage, const eb_buf* sums,
                  const eb_buf* counts, size_t k, size_t d, float alpha, float decay,
                  int replace) {
  return guard([&] {
    need(e, "engine");
    need_type(positions, EB_F32, "positions");
    need_type(usage, EB_F32, "usage");
    need_type(sums, EB_F32, "sums");
    need_type(counts, EB_U32, "counts");
    ensure(positions->len == k * d && usage->len == k && sums->len == k * d && counts->len == k,
           "shapes");
    DeviceGuard g(e);
    touched(e, positions);
    touched(e, usage);
    eb::ema_update(e, static_cast<float*>(positions->ptr), static_cast<float*>(usage->ptr),
                   static_cast<const float*>(sums->ptr), static_cast<const uint32_t*>(counts->ptr),
                   k, d, alpha, decay, replace != 0);
  });
}

int eb_bind_data(eb_engine* e, const float* data, size_t n, size_t d) {
  return guard([&] {
    need(e, "engine");
    ensure(d > 0, "d must be positive");
    DeviceGuard g(e);
    if (e->bound) {
      eb::free_buf(e, e->bound);
      e->bound = nullptr;
    }
    eb_buf* b = nullptr;
    int rc = eb_bind(e, data, n, d, &b);
    if (rc != EB_OK) throw eb::Error(rc, g_last_error);
    e->bound = b;
    e->bound_host = data;
    e->bound_n = n;
  });
}

int eb_unbind_data(eb_engine* e) {
  return guard([&] {
    need(e, "engine");
    DeviceGuard g(e);
    if (e->bound) eb::free_buf(e, e->bound);
    e->bound = nullptr;
    e->bound_host = nullptr;
    e->bound_n = 0;
  });
}

int eb_assign(eb_engine* e, const float* rows, size_t n, size_t d, const uint32_t* ids, size_t m,
              const float* centroids, size_t k, int metric, uint32_t* labels, float* scores) {
  return guard([&] {
    need(e, "engine");
    // check_shapes (assign.rs:121-147).
    ensure(d > 0, "d must be positive");
    ensure(k > 0 && centroids != nullptr, "centroids must be k x d");
    ensure(k <= 0xFFFFFFFFull, "k too large");
    ensure(metric == EB_L2 || metric == EB_IP, "unknown metric");
    if (ids) {
      for (size_t i = 0; i < m; i++) ensure(ids[i] < n, "row id out of range");
    } else {
      ensure(m == n, "dense rows: m must equal n");
    }
    if (m == 0) return;
    need(rows, "rows");
    need(labels, "labels");
    need(scores, "scores");
    DeviceGuard g(e);
    float* c = e->scratch_get<float>("as_c", k * d);
    eb::h2d(e, c, centroids, k * d * 4, e->stream);
    float* cn = nullptr;
    if (metric == EB_L2) {
      cn = e->scratch_get<float>("as_cn", k);
      eb::row_norms(e, c, k, d, cn);
    }
    uint32_t* lab = e->scratch_get<uint32_t>("as_lab", m);
    float* sco = e->scratch_get<float>("as_sco", m);
    eb_buf cb, cnb, lb, sb;
    cb.ptr = c; cb.len = k * d; cb.dtype = EB_F32;
    cnb.ptr = cn; cnb.len = k; cnb.dtype = EB_F32;
    lb.ptr = lab; lb.len = m; lb.dtype = EB_U32;
    sb.ptr = sco; sb.len = m; sb.dtype = EB_F32;
    int rc;
    if (ids && e->bound && e->bound_host == rows && e->bound_n == n && e->bound->d == d) {
      // Rows::Indexed on the bound data: only the ids travel (core/mod.rs:276-298).
      uint32_t* di = e->scratch_get<uint32_t>("as_ids", m);
      EB_CUDA(cudaMemcpyAsync(di, ids, m * 4, cudaMemcpyHostToDevice, e->stream));
      eb_buf ib;
      ib.ptr = di; ib.len = m; ib.dtype = EB_U32;
      rc = eb_top1(e, e->bound, d, &ib, 0, m, &cb, metric == EB_L2 ? &cnb : nullptr, k, metric,
                   &lb, &sb);
    } else if (ids) {
      // Indexed rows gathered on the host (core/mod.rs:299-325).
      float* xd = e->scratch_get<float>("as_x", m * d);
      std::vector<float> gbuf(m * d);
      for (size_t i = 0; i < m; i++)
        std::memcpy(&gbuf[i * d], rows + (size_t)ids[i] * d, d * 4);
      eb::h2d(e, xd, gbuf.data(), m * d * 4, e->stream);
      eb_buf xb;
      xb.ptr = xd; xb.len = m * d; xb.dtype = EB_F32;
      rc = eb_top1(e, &xb, d, nullptr, 0, m, &cb, metric == EB_L2 ? &cnb : nullptr, k, metric,
                   &lb, &sb);
    } else if (e->bound && e->bound_host == rows && e->bound_n == n && e->bound->d == d) {
      // Dense rows that are the bound data set (the host pointer and shape the
      // binding is served by, as for indexed rows): read in place with the
      // binding's norms and screen copy, so that every fit of a sweep over
      // one bound set assigns without uploading it again.
      rc = eb_top1(e, e->bound, d, nullptr, 0, m, &cb, metric == EB_L2 ? &cnb : nullptr, k,
                   metric, &lb, &sb);
    } else {
      // Dense rows: copied in slices on the copy stream, each slice's top-1
      // queued on the engine's stream behind its own copy, so that the copy
      // of slice j + 1 overlaps the top-1 of slice j. The last slice is
      // small (16,384 rows when there are at least 65,536), so that little
      // compute remains once the last copy has landed; with pinned output
      // buffers each slice's labels and scores go back as soon as they are
      // ready. The centroids' screen copy is made once, by the first slice
      // that takes the screen.
      float* xd = e->scratch_get<float>("as_x", m * d);
      if (!e->copy_stream) EB_CUDA(cudaStreamCreateWithFlags(&e->copy_stream, cudaStreamNonBlocking));
      std::vector<size_t> cut{0};
      if (m >= 65536) {
        const size_t body = m - 16384, third = (body + 2) / 3;
        for (size_t r = third; r < body; r += third) cut.push_back(r);
        cut.push_back(body);
      } else {
        const size_t slice = std::max<size_t>(16384, (m + 3) / 4);
        for (size_t r = slice; r < m; r += slice) cut.push_back(r);
      }
      cut.push_back(m);
      const bool early_out = eb::host_pinned(labels) && eb::host_pinned(scores);
      cudaEvent_t ready;
      EB_CUDA(cudaEventCreateWithFlags(&ready, cudaEventDisableTiming));
      EB_CUDA(cudaEventRecord(ready, e->stream));  // earlier work on the staging buffer
      EB_CUDA(cudaStreamWaitEvent(e->copy_stream, ready, 0));
      EB_CUDA(cudaEventDestroy(ready));
      bool converted = false;
      for (size_t j = 0; j + 1 < cut.size(); j++) {
        const size_t r0 = cut[j], r1 = cut[j + 1];
        if (r1 == r0) continue;
        eb::h2d(e, xd + r0 * d, rows + r0 * d, (r1 - r0) * d * 4, e->copy_stream);
        cudaEvent_t landed;
        EB_CUDA(cudaEventCreateWithFlags(&landed, cudaEventDisableTiming));
        EB_CUDA(cudaEventRecord(landed, e->copy_stream));
        EB_CUDA(cudaStreamWaitEvent(e->stream, landed, 0));
        EB_CUDA(cudaEventDestroy(landed));
        eb::Top1Args a;
        a.x = xd;
        a.n = m;
        a.d = d;
        a.ids = nullptr;
        a.r0 = r0;
        a.r1 = r1;
        a.c = c;
        a.cnorm = cn;
        a.k = k;
        a.metric = metric;
        a.labels = lab;
        a.scores = sco;
        a.xnorm = nullptr;
        a.centroids_ready = converted;
        const bool screened = eb::top1_screen_supported(e, a);
        eb::top1_dispatch(e, a, nullptr);
        converted = converted || screened;
        if (early_out) {
          EB_CUDA(cudaMemcpyAsync(labels + r0, lab + r0, (r1 - r0) * 4, cudaMemcpyDeviceToHost,
                                  e->stream));
          EB_CUDA(cudaMemcpyAsync(scores + r0, sco + r0, (r1 - r0) * 4, cudaMemcpyDeviceToHost,
                                  e->stream));
        }
      }
      if (early_out) {
        eb::sync(e);
        return;
      }
      rc = EB_OK;
    }
    if (rc != EB_OK) throw eb::Error(rc, g_last_error);
    eb::d2h(e, labels, lab, m * 4, e->stream);
    eb::d2h(e, scores, sco, m * 4, e->stream);
    eb::sync(e);
  });
}

int eb_layer_norm(eb_engine* e, const eb_buf* x, size_t rows, size_t d, size_t ldx,
                  const eb_buf* weight, const eb_buf* bias, float eps, eb_buf* y, size_t ldy,
                  eb_buf* mean, eb_buf* rstd) {
  return guard([&] {
    need(e, "engine");
    need_float(x, "x");
    need_float(y, "y");
    ensure(y->dtype == x->dtype, "x and y must have one type");
    ensure(d > 0, "d must be positive");
    ensure(eps >= 0.0f, "eps must not be negative");
    eb::LayerNormArgs a;
    a.ldx = need_rows(x, rows, d, ldx, "x");
    a.ldy = need_rows(y, rows, d, ldy, "y");
    ensure(x->ptr != y->ptr || a.ldx == a.ldy, "y over x needs x's row stride");
    ensure(x->ptr == y->ptr || !overlap(x, y), "y overlaps x");
    a.wtype = EB_F32;
    for (const eb_buf* b : {weight, bias}) {
      if (!b) continue;
      need_float(b, "weight and bias");
      ensure(b->dtype == EB_F32 || b->dtype == x->dtype, "weight and bias must be f32 or of x's type");
      ensure(b->len >= d, "weight and bias must hold d elements");
      a.wtype = b->dtype;
    }
    ensure(!weight || !bias || weight->dtype == bias->dtype, "weight and bias must have one type");
    for (const eb_buf* b : {mean, rstd}) {
      if (!b) continue;
      need_type(b, EB_F32, "mean and rstd");
      ensure(b->len >= rows, "mean and rstd must hold one element a row");
    }
    need_here(e, {x, weight, bias, y, mean, rstd});
    const Part m(mean, rows), r(rstd, rows);
    need_apart({Part(y, rows, d, a.ldy), m, r}, {Part(weight, d), Part(bias, d)});
    need_apart({m, r}, {Part(x, rows, d, a.ldx)});
    DeviceGuard g(e);
    touched(e, y);
    touched(e, mean);
    touched(e, rstd);
    a.x = x->ptr;
    a.rows = rows;
    a.d = d;
    a.weight = weight ? weight->ptr : nullptr;
    a.bias = bias ? bias->ptr : nullptr;
    a.eps = eps;
    a.y = y->ptr;
    a.mean = mean ? static_cast<float*>(mean->ptr) : nullptr;
    a.rstd = rstd ? static_cast<float*>(rstd->ptr) : nullptr;
    a.dtype = x->dtype;
    eb::layer_norm(e, a);
  });
}

int eb_layer_norm_backward(eb_engine* e, const eb_buf* dy, size_t lddy, const eb_buf* x,
                           size_t ldx, size_t rows, size_t d, const eb_buf* weight,
                           const eb_buf* mean, const eb_buf* rstd, eb_buf* dx, size_t lddx,
                           eb_buf* dweight, eb_buf* dbias) {
  return guard([&] {
    need(e, "engine");
    need_float(dy, "dy");
    need_float(x, "x");
    ensure(dy->dtype == x->dtype, "dy and x must have one type");
    ensure(d > 0, "d must be positive");
    eb::LayerNormBackwardArgs a;
    a.lddy = need_rows(dy, rows, d, lddy, "dy");
    a.ldx = need_rows(x, rows, d, ldx, "x");
    a.lddx = d;
    if (dx) {
      need_float(dx, "dx");
      ensure(dx->dtype == x->dtype, "dx and x must have one type");
      a.lddx = need_rows(dx, rows, d, lddx, "dx");
      ensure(dx->ptr != dy->ptr || a.lddx == a.lddy, "dx over dy needs dy's row stride");
      ensure(dx->ptr == dy->ptr || !overlap(dx, dy), "dx overlaps dy");
      ensure(!overlap(dx, x), "dx overlaps x");
    }
    a.wtype = EB_F32;
    if (weight) {
      need_float(weight, "weight");
      ensure(weight->dtype == EB_F32 || weight->dtype == x->dtype,
             "weight must be f32 or of x's type");
      ensure(weight->len >= d, "weight must hold d elements");
      a.wtype = weight->dtype;
    }
    need_type(mean, EB_F32, "mean");
    need_type(rstd, EB_F32, "rstd");
    ensure(mean->len >= rows && rstd->len >= rows, "mean and rstd must hold one element a row");
    for (const eb_buf* b : {dweight, dbias}) {
      if (!b) continue;
      need_float(b, "dweight and dbias");
      ensure(b->dtype == EB_F32 || b->dtype == x->dtype,
             "dweight and dbias must be f32 or of x's type");
      ensure(b->len >= d, "dweight and dbias must hold d elements");
    }
    need_here(e, {dy, x, weight, mean, rstd, dx, dweight, dbias});
    const Part dwp(dweight, d), dbp(dbias, d);
    need_apart({Part(dx, rows, d, a.lddx), dwp, dbp},
               {Part(weight, d), Part(mean, rows), Part(rstd, rows)});
    need_apart({dwp, dbp}, {Part(dy, rows, d, a.lddy), Part(x, rows, d, a.ldx)});
    DeviceGuard g(e);
    touched(e, dx);
    touched(e, dweight);
    touched(e, dbias);
    a.dy = dy->ptr;
    a.x = x->ptr;
    a.rows = rows;
    a.d = d;
    a.weight = weight ? weight->ptr : nullptr;
    a.mean = static_cast<const float*>(mean->ptr);
    a.rstd = static_cast<const float*>(rstd->ptr);
    a.dx = dx ? dx->ptr : nullptr;
    a.dweight = dweight ? dweight->ptr : nullptr;
    a.dbias = dbias ? dbias->ptr : nullptr;
    a.dtype = x->dtype;
    a.dwtype = dweight ? dweight->dtype : EB_F32;
    a.dbtype = dbias ? dbias->dtype : EB_F32;
    eb::layer_norm_backward(e, a);
  });
}

}  // extern "C"

namespace {

// The arguments both passes of the linear cross entropy share.
eb::LinearCeArgs check_linear_ce(eb_engine* e, const eb_buf* x, size_t n, size_t d, size_t ldx,
                                 const eb_buf* w, size_t k, size_t ldw, const eb_buf* targets,
                                 float scale) {
  need(e, "engine");
  need_float(x, "x");
  need_float(w, "w");
  ensure(x->dtype == w->dtype, "x and w must have one type");
  ensure(d > 0 && d <= 0x7FFFFF00ull, "d must be positive and fit 31 bits");
  ensure(k > 0 && k <= 0x7FFFFF00ull, "k must be positive and fit 31 bits");
  ensure(n <= 0x7FFFFF00ull, "n must fit 31 bits");
  // A launch works on a pass of rows or a piece of P, whose tiles are far fewer than 31
  // bits count; a problem whose tiles of 128 x 160 in all are more is refused.
  ensure((n / 128 + 1) * (k / 160 + 1) <= 0x7FFFFFFFull, "n x k is too large");
  ensure(std::isfinite(scale) && scale > 0.0f, "scale must be positive and finite");
  need_type(targets, EB_U32, "targets");
  ensure(targets->len >= n, "targets must hold one element a row");
  eb::LinearCeArgs a;
  a.ldx = need_rows(x, n, d, ldx, "x");
  a.ldw = need_rows(w, k, d, ldw, "w");
  a.x = x->ptr;
  a.n = n;
  a.d = d;
  a.w = w->ptr;
  a.k = k;
  a.targets = static_cast<const uint32_t*>(targets->ptr);
  a.scale = scale;
  a.dtype = x->dtype;
  return a;
}

}  // namespace

extern "C" {

int eb_linear_ce(eb_engine* e, const eb_buf* x, size_t n, size_t d, size_t ldx, const eb_buf* w,
                 size_t k, size_t ldw, const eb_buf* targets, float scale, eb_buf* loss,
                 eb_buf* lse) {
  return guard([&] {
    const eb::LinearCeArgs a = check_linear_ce(e, x, n, d, ldx, w, k, ldw, targets, scale);
    need_type(loss, EB_F32, "loss");
    need_type(lse, EB_F32, "lse");
    ensure(loss->len >= n && lse->len >= n, "loss and lse must hold one element a row");
    need_here(e, {x, w, targets, loss, lse});
    ensure(!overlap(loss, lse), "loss overlaps lse");
    for (const eb_buf* in : {x, w, targets})
      ensure(!overlap(loss, in) && !overlap(lse, in), "an output overlaps an input");
    DeviceGuard g(e);
    touched(e, loss);
    touched(e, lse);
    eb::linear_ce(e, a, static_cast<float*>(loss->ptr), static_cast<float*>(lse->ptr));
  });
}

int eb_linear_ce_backward(eb_engine* e, const eb_buf* x, size_t n, size_t d, size_t ldx,
                          const eb_buf* w, size_t k, size_t ldw, const eb_buf* targets,
                          float scale, const eb_buf* lse, const eb_buf* dloss, eb_buf* dx,
                          size_t lddx, eb_buf* dw, size_t lddw) {
  return guard([&] {
    const eb::LinearCeArgs a = check_linear_ce(e, x, n, d, ldx, w, k, ldw, targets, scale);
    need_type(lse, EB_F32, "lse");
    ensure(lse->len >= n, "lse must hold one element a row");
    need_type(dloss, EB_F32, "dloss");
    ensure(dloss->len == 1 || dloss->len >= n, "dloss must hold one element, or one a row");
    need_here(e, {x, w, targets, lse, dloss, dx, dw});
    eb::LinearCeGrads q{};
    for (const eb_buf* b : {dx, dw}) {
      if (!b) continue;
      need_float(b, "dx and dw");
      ensure(b->dtype == EB_F32 || b->dtype == x->dtype, "dx and dw must be f32 or of x's type");
      for (const eb_buf* in : {x, w, targets, lse, dloss})
        ensure(!overlap(b, in), "an output overlaps an input");
    }
    ensure(!overlap(dx, dw), "dx overlaps dw");
    if (dx) {
      q.lddx = need_rows(dx, n, d, lddx, "dx");
      q.dx = dx->ptr;
      q.dxtype = dx->dtype;
    }
    if (dw) {
      q.lddw = need_rows(dw, k, d, lddw, "dw");
      q.dw = dw->ptr;
      q.dwtype = dw->dtype;
    }
    q.lse = static_cast<const float*>(lse->ptr);
    q.dloss = static_cast<const float*>(dloss->ptr);
    q.one_dloss = dloss->len == 1;
    DeviceGuard g(e);
    touched(e, dx);
    touched(e, dw);
    eb::linear_ce_backward(e, a, q);
  });
}

int eb_adamw_create(eb_engine* e, const eb_adamw_tensor* t, size_t count, eb_adamw** out) {
  return guard([&] {
    need(e, "engine");
    need(out, "out");
    *out = nullptr;
    if (count) need(t, "tensors");
    ensure(count <= 0x7FFFFFFFull, "too many tensors");
    struct Range {
      const char *lo, *hi;
      bool written;
    };
    std::vector<Range> ranges;
    auto use = [&](const eb_buf* b, size_t n, bool written) {
      const char* p = static_cast<const char*>(b->ptr);
      ranges.push_back({p, p + n * eb::dtype_bytes(b->dtype), written});
    };
    auto plan = std::make_unique<eb_adamw>();
    for (size_t i = 0; i < count; i++) {
      need(t[i].p, "p");
      need(t[i].g, "g");
      need(t[i].m, "m");
      need(t[i].v, "v");
      need_here(e, {t[i].p, t[i].g, t[i].m, t[i].v, t[i].m_scale, t[i].v_scale, t[i].copy});
      const size_t len = t[i].p->len;
      for (const eb_buf* b : {(const eb_buf*)t[i].p, t[i].g})
        ensure(b->dtype == EB_F32 || b->dtype == EB_BF16, "p and g must be f32 or bf16 buffers");
      ensure((t[i].m_scale == nullptr) == (t[i].v_scale == nullptr),
             "m_scale and v_scale must be given together");
      const bool eight = t[i].m_scale != nullptr;
      for (const eb_buf* b : {t[i].m, t[i].v})
        ensure(b->dtype == (eight ? EB_F8 : EB_F32),
               eight ? "8-bit m and v must be f8 buffers" : "m and v must be f32 buffers");
      ensure(t[i].g->len == len && t[i].m->len == len && t[i].v->len == len,
             "p, g, m and v must have one length");
      if (eight) {
        const size_t blocks = (len + EB_ADAMW_BLOCK - 1) / EB_ADAMW_BLOCK;
        need_type(t[i].m_scale, EB_F32, "m_scale");
        need_type(t[i].v_scale, EB_F32, "v_scale");
        ensure(t[i].m_scale->len >= blocks && t[i].v_scale->len >= blocks,
               "m_scale and v_scale must hold one element for each 256 of p");
      }
      if (t[i].copy) {
        ensure(t[i].copy->dtype == EB_BF16, "copy must be a bf16 buffer");
        ensure(t[i].copy->len >= len, "copy must be as long as p");
      }
      ensure(std::isfinite(t[i].weight_decay), "weight_decay must be finite");
      if (len == 0) continue;
      for (eb_buf* b : {t[i].p, t[i].m, t[i].v, t[i].m_scale, t[i].v_scale, t[i].copy}) {
        if (!b) continue;
        const bool scale = b == t[i].m_scale || b == t[i].v_scale;
        use(b, scale ? (len + EB_ADAMW_BLOCK - 1) / EB_ADAMW_BLOCK : len, true);
        plan->written.push_back(b);
      }
      use(t[i].g, len, false);
    }
    // Blocks take the tensors in any order: what one writes, no other may touch.
    // Gradients are only read, and may be shared.
    std::sort(ranges.begin(), ranges.end(),
              [](const Range& a, const Range& b) { return a.lo < b.lo; });
    const char *written = nullptr, *read = nullptr;  // ends of the ranges so far
    for (const Range& r : ranges) {
      ensure(r.lo >= written, r.written ? "a buffer is written twice, in part or whole"
                                        : "g overlaps a buffer that is written");
      ensure(!r.written || r.lo >= read, "g overlaps a buffer that is written");
      (r.written ? written : read) = std::max(r.written ? written : read, r.hi);
    }
    DeviceGuard g(e);
    try {
      eb::adamw_create(e, t, count, plan.get());
    } catch (...) {
      if (plan->table) cudaFreeAsync(plan->table, e->stream);
      throw;
    }
    *out = plan.release();
  });
}

int eb_adamw_destroy(eb_engine* e, eb_adamw* plan) {
  if (!plan) return EB_OK;
  return release([&] {
    need(e, "engine");
    DeviceGuard g(e);
    if (plan->table) cudaFreeAsync(plan->table, e->stream);
    delete plan;
  });
}

int eb_adamw_step(eb_engine* e, eb_adamw* plan, double lr, uint64_t step, double beta1,
                  double beta2, double eps, float grad_scale) {
  return guard([&] {
    need(e, "engine");
    need(plan, "plan");
    ensure(step >= 1, "step counts from 1");
    ensure(std::isfinite(lr), "lr must be finite");
    ensure(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "betas must be in [0, 1)");
    ensure(std::isfinite(eps) && eps >= 0.0, "eps must be finite and not negative");
    DeviceGuard g(e);
    for (eb_buf* b : plan->written) touched(e, b);
    eb::adamw_step(e, plan, lr, step, beta1, beta2, eps, grad_scale);
  });
}

}  // extern "C"
