// One AdamW step over many tensors in one kernel.
//
// A plan keeps the tensors' addresses and a table of their pieces (CHUNK
// elements each) on the device; one block takes one piece, so a step is one
// launch however many tensors there are. Every operation is rounded by itself
// (no FMA contraction, IEEE divide and square root): the step's results do
// not depend on how the compiler fuses it.
//
// 8-bit states: 256 elements share a scale, half a warp holds them (16 a
// lane), so the new scale is a shuffle maximum over registers and every byte
// is read and written once. The first moment is kept as code x scale with e4m3 codes
// (largest 448); the second as its root, whose range is half as wide in
// exponent and which the update needs anyway. A root above zero keeps at
// least the smallest code: rounded to zero it would leave the moment above it
// divided by eps alone.
//
// Bound by HBM: 28 bytes a parameter (f32; 120 M parameters in 160 tensors 488
// us, 6.9 TB/s), or 16 with bf16 gradients, 8-bit states and the bf16 copy (400
// M 1,214 us, 5.3 TB/s: about 70 instructions a parameter, most of them the
// IEEE divide and square root and the code conversions, share the bound).
// Measured and not kept for 8-bit states: longer pieces (4,096 to 32,768
// elements: 1,490 to 1,660 us, their streams lie further apart), elements in
// flight through shared memory (1,476), a warp a block of 256 (1,300).
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cmath>
#include <vector>

#include "elem.h"
#include "engine.h"

namespace eb {

namespace {

constexpr int CHUNK = 2048;  // elements of a piece
constexpr int THREADS = 256, THREADS8 = 128;  // of a block, for 32-bit and 8-bit states
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

// Two codes at a time, each way.
__device__ __forceinline__ float2 f8_values(uint16_t c) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(c, __NV_E4M3)));
}
__device__ __forceinline__ uint16_t f8_codes(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// Larger of two, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Largest over the 16 lanes of a half warp.
__device__ __forceinline__ float half_max(float v) {
#pragma unroll
  for (int o = 8; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
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

// Eight elements as they are loaded.
template <typename PT, typename GT>
struct Raw {
  Pack<PT, 4> p[2];
  Pack<GT, 4> g[2];
  Pack<uint16_t, 4> mc, vc;
};

// Elements i .. i + 8 of the piece at `at`, zeros past `count`.
template <typename PT, typename GT>
__device__ __forceinline__ Raw<PT, GT> load_raw(const Entry& E, size_t at, int i, int count) {
  Raw<PT, GT> r;
  const size_t a = at + i;
  const PT* P = static_cast<const PT*>(E.p) + a;
  const GT* G = static_cast<const GT*>(E.g) + a;
  const uint8_t* M = static_cast<const uint8_t*>(E.m) + a;
  const uint8_t* V = static_cast<const uint8_t*>(E.v) + a;
  if (i + 8 <= count) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      r.p[h] = reinterpret_cast<const Pack<PT, 4>*>(P)[h];
      r.g[h] = reinterpret_cast<const Pack<GT, 4>*>(G)[h];
    }
    r.mc = *reinterpret_cast<const Pack<uint16_t, 4>*>(M);
    r.vc = *reinterpret_cast<const Pack<uint16_t, 4>*>(V);
  } else {
    const int mine = count - i;
#pragma unroll
    for (int u = 0; u < 8; u++) {
      r.p[u / 4].v[u % 4] = u < mine ? P[u] : from_f32<PT>(0.0f);
      r.g[u / 4].v[u % 4] = u < mine ? G[u] : from_f32<GT>(0.0f);
    }
#pragma unroll
    for (int u = 0; u < 8; u += 2) {
      r.mc.v[u / 2] = (uint16_t)((u < mine ? M[u] : 0) | (u + 1 < mine ? M[u + 1] : 0) << 8);
      r.vc.v[u / 2] = (uint16_t)((u < mine ? V[u] : 0) | (u + 1 < mine ? V[u + 1] : 0) << 8);
    }
  }
  return r;
}

// Half a warp a block of 256, 2 x 8 elements a lane: the block's scales, their
// inverses and the addresses are worked out once for 16 elements.
template <typename PT, typename GT>
__device__ __forceinline__ void piece_f8(const Entry& E, const Hyper& H, float keep, size_t at,
                                         int count) {
  static_assert(CHUNK == 16 * THREADS8, "one pass a piece");
  const int lane = threadIdx.x & 15, b = (threadIdx.x >> 4) * 256;
  if ((threadIdx.x >> 5) * 512 >= count) return;  // the whole warp
  const size_t blk = (at + b) / 256;
  const bool some = b < count;
  const float ms = some ? E.ms[blk] : 0.0f, vs = some ? E.vs[blk] : 0.0f;
  Raw<PT, GT> R[2];
#pragma unroll
  for (int h = 0; h < 2; h++) R[h] = load_raw<PT, GT>(E, at, b + h * 128 + lane * 8, count);
  // Elements past the end hold zeros, whose moments stay zero.
  float m[16], r[16], tm = 0.0f, tr = 0.0f;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int i = b + h * 128 + lane * 8;
    const size_t a = at + i;
    float p[8];
#pragma unroll
    for (int u = 0; u < 8; u += 2) {
      const float2 mq = f8_values(R[h].mc.v[u / 2]), rq = f8_values(R[h].vc.v[u / 2]);
#pragma unroll
      for (int w = 0; w < 2; w++) {
        const int q = u + w, k = h * 8 + q;
        const float root = __fmul_rn(w ? rq.y : rq.x, vs);
        const Step s = step_one(H, keep, to_f32(R[h].p[q / 4].v[q % 4]),
                                to_f32(R[h].g[q / 4].v[q % 4]), __fmul_rn(w ? mq.y : mq.x, ms),
                                __fmul_rn(root, root));
        p[q] = s.p;
        m[k] = s.m;
        r[k] = s.root;
        tm = max_nan(tm, fabsf(s.m));
        tr = max_nan(tr, s.root);
      }
    }
    PT* P = static_cast<PT*>(E.p) + a;
    if (i + 8 <= count) {
#pragma unroll
      for (int x = 0; x < 2; x++) {
        const float q[4] = {p[4 * x], p[4 * x + 1], p[4 * x + 2], p[4 * x + 3]};
        store4(P + 4 * x, q);
      }
      if (E.copy) {
        Pack<__nv_bfloat16, 8> c;
#pragma unroll
        for (int u = 0; u < 8; u++) c.v[u] = from_f32<__nv_bfloat16>(p[u]);
        *reinterpret_cast<Pack<__nv_bfloat16, 8>*>(E.copy + a) = c;
      }
    } else {
#pragma unroll
      for (int u = 0; u < 8; u++) {
        if (i + u < count) {
          P[u] = from_f32<PT>(p[u]);
          if (E.copy) E.copy[a + u] = from_f32<__nv_bfloat16>(p[u]);
        }
      }
    }
  }
  tm = half_max(tm);
  tr = half_max(tr);
  const bool fine = isfinite(tm) && isfinite(tr);
  float im, ir;
  const float nms = f8_scale(tm, fine, im), nvs = f8_scale(tr, fine, ir);
  const float least = ir > 0.0f ? F8_MIN : 0.0f;
  if (some && lane == 0) {
    E.ms[blk] = nms;
    E.vs[blk] = nvs;
  }
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int i = b + h * 128 + lane * 8;
    Pack<uint16_t, 4> mc, vc;
#pragma unroll
    for (int u = 0; u < 8; u += 2) {
      const int k = h * 8 + u;
      mc.v[u / 2] = f8_codes(__fmul_rn(m[k], im), __fmul_rn(m[k + 1], im));
      float q[2];
#pragma unroll
      for (int w = 0; w < 2; w++)
        q[w] = r[k + w] > 0.0f ? fmaxf(__fmul_rn(r[k + w], ir), least) : 0.0f;
      vc.v[u / 2] = f8_codes(q[0], q[1]);
    }
    uint8_t* M = static_cast<uint8_t*>(E.m) + at + i;
    uint8_t* V = static_cast<uint8_t*>(E.v) + at + i;
    if (i + 8 <= count) {
      *reinterpret_cast<Pack<uint16_t, 4>*>(M) = mc;
      *reinterpret_cast<Pack<uint16_t, 4>*>(V) = vc;
    } else {
#pragma unroll
      for (int u = 0; u < 8; u++) {
        if (i + u < count) {
          M[u] = (uint8_t)(mc.v[u / 2] >> (u % 2 * 8));
          V[u] = (uint8_t)(vc.v[u / 2] >> (u % 2 * 8));
        }
      }
    }
  }
}

template <bool EIGHT, typename PT, typename GT>
__device__ __forceinline__ void piece(const Entry& E, const Hyper& H, float keep, size_t at,
                                      int count) {
  if constexpr (EIGHT)
    piece_f8<PT, GT>(E, H, keep, at, count);
  else
    piece_f32<PT, GT>(E, H, keep, at, count);
}

// The 8-bit and 32-bit tensors of a plan go to kernels of their own: the
// 32-bit one then keeps six blocks on an SM (120 M f32 parameters: 488 us; four
// blocks, as registers for both allow: 524).
template <bool EIGHT>
__global__ void __launch_bounds__(EIGHT ? THREADS8 : THREADS, 6)
    k_adamw(const Entry* __restrict__ entries, const uint2* __restrict__ pieces, Hyper H) {
  pdl_wait();
  const uint2 w = pieces[blockIdx.x];
  const Entry E = entries[w.x];
  const size_t at = (size_t)w.y * CHUNK;
  const int count = (int)min((size_t)CHUNK, E.len - at);
  const float keep = (float)(1.0 - H.lr * E.decay);
  if (E.ptype == EB_F32) {
    if (E.gtype == EB_F32)
      piece<EIGHT, float, float>(E, H, keep, at, count);
    else
      piece<EIGHT, float, __nv_bfloat16>(E, H, keep, at, count);
  } else {
    if (E.gtype == EB_F32)
      piece<EIGHT, __nv_bfloat16, float>(E, H, keep, at, count);
    else
      piece<EIGHT, __nv_bfloat16, __nv_bfloat16>(E, H, keep, at, count);
  }
}

}  // namespace

void adamw_create(eb_engine* e, const eb_adamw_tensor* t, size_t count, eb_adamw* plan) {
  std::vector<Entry> entries;
  std::vector<uint2> pieces[2];  // of 32-bit states, of 8-bit states
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
    auto& list = pieces[E.ms != nullptr];
    const size_t np = (E.len + CHUNK - 1) / CHUNK;
    ensure(list.size() + np <= 0x7FFFFFFFull, "too many elements in one plan");
    for (size_t c = 0; c < np; c++) list.push_back(make_uint2((unsigned)i, (unsigned)c));
  }
  size_t off = (entries.size() * sizeof(Entry) + 15) / 16 * 16;
  for (int k = 0; k < 2; k++) {
    plan->pieces[k] = pieces[k].size();
    plan->pieces_at[k] = off;
    off += pieces[k].size() * sizeof(uint2);
  }
  if (!plan->pieces[0] && !plan->pieces[1]) return;
  EB_CUDA(cudaMallocAsync(&plan->table, off, e->stream));
  e->device_allocs++;
  char* dst = static_cast<char*>(plan->table);
  h2d(e, dst, entries.data(), entries.size() * sizeof(Entry), e->stream);
  for (int k = 0; k < 2; k++)
    if (plan->pieces[k])
      h2d(e, dst + plan->pieces_at[k], pieces[k].data(), pieces[k].size() * sizeof(uint2),
          e->stream);
}

void adamw_step(eb_engine* e, const eb_adamw* plan, double lr, uint64_t step, double b1, double b2,
                double eps, float gscale) {
  const Hyper H{(float)b1, (float)(1.0 - b1), (float)b2, (float)(1.0 - b2),
                (float)(lr / (1.0 - std::pow(b1, (double)step))),
                (float)(1.0 / std::sqrt(1.0 - std::pow(b2, (double)step))), (float)eps, gscale, lr};
  const char* t = static_cast<const char*>(plan->table);
  for (int k = 0; k < 2; k++) {
    if (!plan->pieces[k]) continue;
    launch_pdl(e, k ? k_adamw<true> : k_adamw<false>, dim3((unsigned)plan->pieces[k]),
               dim3(k ? THREADS8 : THREADS), 0, reinterpret_cast<const Entry*>(t),
               reinterpret_cast<const uint2*>(t + plan->pieces_at[k]), H);
    e->stats.kernel_launches++;
  }
}

}  // namespace eb
