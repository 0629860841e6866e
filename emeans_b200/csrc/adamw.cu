// One AdamW step over many tensors in one kernel.
//
// A plan keeps the tensors' addresses and a table of their pieces (CHUNK
// elements each) on the device; one block takes one piece, so a step is one
// launch however many tensors there are. Every operation is rounded by itself
// (no FMA contraction, IEEE divide and square root): the step's results do
// not depend on how the compiler fuses it.
//
// 8-bit states: 256 elements share a scale, one warp holds them (8 a lane),
// so the new scale is a shuffle maximum over registers and every byte is read
// and written once. The first moment is kept as code x scale with e4m3 codes
// (largest 448); the second as its root, whose range is half as wide in
// exponent and which the update needs anyway. A root above zero keeps at
// least the smallest code: rounded to zero it would leave the moment above it
// divided by eps alone.
//
// Bound by HBM: 28 bytes a parameter (f32), or 16 with bf16 gradients, 8-bit
// states and the bf16 copy.
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cmath>
#include <vector>

#include "elem.h"
#include "engine.h"

namespace eb {

namespace {

constexpr int CHUNK = 2048;
constexpr int THREADS = 256;
constexpr float F8_MAX = 448.0f, F8_MIN = 0.001953125f;  // e4m3: largest, smallest (2^-9)

struct Entry {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* ms;
  float* vs;
  __nv_bfloat16* copy;
  size_t len;
  double decay;
  int ptype, gtype;
};

struct Hyper {
  float b1, c1, b2, c2;  // beta, 1 - beta
  float size, fix, eps, gscale;
  double lr;
};

struct Step {
  float m, root, v, p;
};

// The update of one element.
__device__ __forceinline__ Step step_one(const Hyper& H, float keep, float p, float g, float m,
                                         float v) {
  Step s;
  g = __fmul_rn(g, H.gscale);
  s.m = __fadd_rn(__fmul_rn(m, H.b1), __fmul_rn(g, H.c1));
  s.v = __fadd_rn(__fmul_rn(v, H.b2), __fmul_rn(__fmul_rn(g, g), H.c2));
  s.root = __fsqrt_rn(s.v);
  const float step = __fmul_rn(__fdiv_rn(s.m, __fadd_rn(__fmul_rn(s.root, H.fix), H.eps)), H.size);
  s.p = __fadd_rn(__fmul_rn(p, keep), -step);
  return s;
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  const Pack<T, 4> r = *reinterpret_cast<const Pack<T, 4>*>(p);
#pragma unroll
  for (int u = 0; u < 4; u++) v[u] = to_f32(r.v[u]);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
  Pack<T, 4> r;
#pragma unroll
  for (int u = 0; u < 4; u++) r.v[u] = from_f32<T>(v[u]);
  *reinterpret_cast<Pack<T, 4>*>(p) = r;
}

template <typename PT, typename GT>
__device__ __forceinline__ void piece_f32(const Entry& E, const Hyper& H, float keep, size_t at,
                                          int count) {
  PT* P = static_cast<PT*>(E.p) + at;
  const GT* G = static_cast<const GT*>(E.g) + at;
  float* M = static_cast<float*>(E.m) + at;
  float* V = static_cast<float*>(E.v) + at;
#pragma unroll
  for (int h = 0; h < CHUNK / (4 * THREADS); h++) {
    const int i = (h * THREADS + threadIdx.x) * 4;
    if (i + 4 <= count) {
      float p[4], g[4], m[4], v[4];
      load4(P + i, p);
      load4(G + i, g);
      load4(M + i, m);
      load4(V + i, v);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const Step s = step_one(H, keep, p[u], g[u], m[u], v[u]);
        p[u] = s.p;
        m[u] = s.m;
        v[u] = s.v;
      }
      store4(P + i, p);
      store4(M + i, m);
      store4(V + i, v);
      if (E.copy) store4(E.copy + at + i, p);
    } else {
      for (int j = i; j < count; j++) {
        const Step s = step_one(H, keep, to_f32(P[j]), to_f32(G[j]), M[j], V[j]);
        P[j] = from_f32<PT>(s.p);
        M[j] = s.m;
        V[j] = s.v;
        if (E.copy) E.copy[at + j] = from_f32<__nv_bfloat16>(s.p);
      }
    }
  }
}

__device__ __forceinline__ float f8_value(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}
__device__ __forceinline__ uint8_t f8_code(float v) {
  return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Scale of a block whose largest magnitude is `top`, and its inverse (0 for a
// block of zeros, or of values too small to be scaled up).
__device__ __forceinline__ float f8_scale(float top, bool finite, float& inv) {
  float scale = __fmul_rn(top, 1.0f / F8_MAX);
  inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
  if (!isfinite(inv)) scale = inv = 0.0f;
  return finite ? scale : NAN;
}

template <typename PT, typename GT>
__device__ __forceinline__ void piece_f8(const Entry& E, const Hyper& H, float keep, size_t at,
                                         int count) {
  const int lane = threadIdx.x & 31;
  static_assert(CHUNK == 8 * THREADS, "one block of 256 a warp");
  const int i = (threadIdx.x >> 5) * 256 + lane * 8;
  if (i - lane * 8 >= count) return;  // the whole warp
  const size_t a = at + i, blk = (at + i) / 256;
  const int mine = min(max(count - i, 0), 8);
  PT* P = static_cast<PT*>(E.p) + a;
  const GT* G = static_cast<const GT*>(E.g) + a;
  uint8_t* M = static_cast<uint8_t*>(E.m) + a;
  uint8_t* V = static_cast<uint8_t*>(E.v) + a;
  const float ms = E.ms[blk], vs = E.vs[blk];
  float p[8], g[8];
  Pack<uint8_t, 8> mc, vc;
  if (mine == 8) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float q[4];
      load4(P + 4 * h, q);
#pragma unroll
      for (int u = 0; u < 4; u++) p[4 * h + u] = q[u];
      load4(G + 4 * h, q);
#pragma unroll
      for (int u = 0; u < 4; u++) g[4 * h + u] = q[u];
    }
    mc = *reinterpret_cast<const Pack<uint8_t, 8>*>(M);
    vc = *reinterpret_cast<const Pack<uint8_t, 8>*>(V);
  } else {
#pragma unroll
    for (int u = 0; u < 8; u++) {
      p[u] = u < mine ? to_f32(P[u]) : 0.0f;
      g[u] = u < mine ? to_f32(G[u]) : 0.0f;
      mc.v[u] = u < mine ? M[u] : 0;
      vc.v[u] = u < mine ? V[u] : 0;
    }
  }
  float m[8], r[8], tm = 0.0f, tr = 0.0f;
  bool fine = true;
#pragma unroll
  for (int u = 0; u < 8; u++) {
    const float root = __fmul_rn(f8_value(vc.v[u]), vs);
    const Step s = step_one(H, keep, p[u], g[u], __fmul_rn(f8_value(mc.v[u]), ms),
                            __fmul_rn(root, root));
    p[u] = s.p;
    m[u] = s.m;
    r[u] = s.root;
    if (u < mine) {
      tm = fmaxf(tm, fabsf(s.m));
      tr = fmaxf(tr, s.root);
      fine = fine && isfinite(s.m) && isfinite(s.root);
    }
  }
  fine = __all_sync(0xffffffffu, fine);
  float im, ir;
  const float nms = f8_scale(warp_max(tm), fine, im), nvs = f8_scale(warp_max(tr), fine, ir);
#pragma unroll
  for (int u = 0; u < 8; u++) {
    mc.v[u] = f8_code(__fmul_rn(m[u], im));
    const float q = __fmul_rn(r[u], ir);
    vc.v[u] = f8_code(r[u] > 0.0f && ir > 0.0f ? fmaxf(q, F8_MIN) : q);
  }
  if (lane == 0) {
    E.ms[blk] = nms;
    E.vs[blk] = nvs;
  }
  if (mine == 8) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const float q[4] = {p[4 * h], p[4 * h + 1], p[4 * h + 2], p[4 * h + 3]};
      store4(P + 4 * h, q);
      if (E.copy) store4(E.copy + a + 4 * h, q);
    }
    *reinterpret_cast<Pack<uint8_t, 8>*>(M) = mc;
    *reinterpret_cast<Pack<uint8_t, 8>*>(V) = vc;
  } else {
#pragma unroll
    for (int u = 0; u < 8; u++) {
      if (u < mine) {
        P[u] = from_f32<PT>(p[u]);
        M[u] = mc.v[u];
        V[u] = vc.v[u];
        if (E.copy) E.copy[a + u] = from_f32<__nv_bfloat16>(p[u]);
      }
    }
  }
}

template <typename PT, typename GT>
__device__ __forceinline__ void piece(const Entry& E, const Hyper& H, float keep, size_t at,
                                      int count) {
  if (E.ms)
    piece_f8<PT, GT>(E, H, keep, at, count);
  else
    piece_f32<PT, GT>(E, H, keep, at, count);
}

__global__ void __launch_bounds__(THREADS)
    k_adamw(const Entry* __restrict__ entries, const uint2* __restrict__ pieces, Hyper H) {
  pdl_wait();
  const uint2 w = pieces[blockIdx.x];
  const Entry E = entries[w.x];
  const size_t at = (size_t)w.y * CHUNK;
  const int count = (int)min((size_t)CHUNK, E.len - at);
  const float keep = (float)(1.0 - H.lr * E.decay);
  if (E.ptype == EB_F32) {
    if (E.gtype == EB_F32)
      piece<float, float>(E, H, keep, at, count);
    else
      piece<float, __nv_bfloat16>(E, H, keep, at, count);
  } else {
    if (E.gtype == EB_F32)
      piece<__nv_bfloat16, float>(E, H, keep, at, count);
    else
      piece<__nv_bfloat16, __nv_bfloat16>(E, H, keep, at, count);
  }
}

}  // namespace

void adamw_create(eb_engine* e, const eb_adamw_tensor* t, size_t count, eb_adamw* plan) {
  std::vector<Entry> entries;
  std::vector<uint2> pieces;
  for (size_t i = 0; i < count; i++) {
    Entry E{};
    E.p = t[i].p->ptr;
    E.g = t[i].g->ptr;
    E.m = t[i].m->ptr;
    E.v = t[i].v->ptr;
    E.ms = t[i].m_scale ? static_cast<float*>(t[i].m_scale->ptr) : nullptr;
    E.vs = t[i].v_scale ? static_cast<float*>(t[i].v_scale->ptr) : nullptr;
    E.copy = t[i].copy ? static_cast<__nv_bfloat16*>(t[i].copy->ptr) : nullptr;
    E.len = t[i].p->len;
    E.decay = t[i].weight_decay;
    E.ptype = t[i].p->dtype;
    E.gtype = t[i].g->dtype;
    entries.push_back(E);
    const size_t np = (E.len + CHUNK - 1) / CHUNK;
    ensure(pieces.size() + np <= 0x7FFFFFFFull, "too many elements in one plan");
    for (size_t c = 0; c < np; c++) pieces.push_back(make_uint2((unsigned)i, (unsigned)c));
  }
  plan->pieces = pieces.size();
  if (pieces.empty()) return;
  const size_t eb = entries.size() * sizeof(Entry), pb = pieces.size() * sizeof(uint2);
  const size_t off = (eb + 15) / 16 * 16;
  EB_CUDA(cudaMallocAsync(&plan->table, off + pb, e->stream));
  e->device_allocs++;
  plan->pieces_at = off;
  h2d(e, plan->table, entries.data(), eb, e->stream);
  h2d(e, static_cast<char*>(plan->table) + off, pieces.data(), pb, e->stream);
}

void adamw_step(eb_engine* e, const eb_adamw* plan, double lr, uint64_t step, double b1, double b2,
                double eps, float gscale) {
  if (!plan->pieces) return;
  Hyper H{(float)b1, (float)(1.0 - b1), (float)b2, (float)(1.0 - b2),
          (float)(lr / (1.0 - std::pow(b1, (double)step))),
          (float)(1.0 / std::sqrt(1.0 - std::pow(b2, (double)step))), (float)eps, gscale, lr};
  const char* t = static_cast<const char*>(plan->table);
  launch_pdl(e, k_adamw, dim3((unsigned)plan->pieces), dim3(THREADS), 0,
             reinterpret_cast<const Entry*>(t), reinterpret_cast<const uint2*>(t + plan->pieces_at),
             H);
  e->stats.kernel_launches++;
}

}  // namespace eb
