// Layer norm, forward and backward.
//
// y = (x - mean) rstd w + b over each row of d elements. A group of G threads
// holds one row in registers (EPT elements a thread), so the row is read
// once: the mean and then the mean squared deviation come from registers (two
// reductions; no E[x^2] - mean^2, which cancels when a row's offset is large
// against its spread). The backward pass holds x and dy the same way:
//   u = (x - mean) rstd, h = dy w,
//   dx = rstd (h - avg(h) - u avg(h u)), dw += dy u, db += dy.
// Groups stay on the GPU and step through the rows, so that the weights and,
// in the backward pass, each thread's own columns of dw and db stay in
// registers; every block then writes one partial row of each, and a second
// kernel adds the blocks in order (the same bits on every call).
//
// Bound by HBM: forward reads x and writes y, backward reads dy and x and
// writes dx.
#include <cuda_runtime.h>

#include <cmath>

#include "elem.h"
#include "engine.h"

namespace eb {

namespace {

struct NormFwd {
  const void* x;
  const void* w;  // or null
  const void* b;  // or null
  void* y;
  float* mean;  // or null
  float* rstd;  // or null
  long rows, d, ldx, ldy;
  float eps, inv_d;
  int wtype;
};

struct NormBwd {
  const void* dy;
  const void* x;
  const void* w;  // or null
  const float* mean;
  const float* rstd;
  void* dx;       // or null
  float* part_w;  // gridDim.x x d partial sums, or null
  float* part_b;
  long rows, d, lddy, ldx, lddx;
  float inv_d;
  int wtype;
};

constexpr int WARP_BLOCK = 128;  // threads of a block when a group is one warp

// Sum over the group's G threads, in every thread. `slot`: two buffers of
// G / 32 floats used in turn, so that one barrier per sum is enough.
template <int G>
__device__ __forceinline__ float group_sum(float v, float (*slot)[G / 32], int& turn) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (G > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) slot[turn][warp] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < G / 32; i++) v += slot[turn][i];
    turn ^= 1;
  }
  return v;
}

// Two sums at once (one barrier).
template <int G>
__device__ __forceinline__ float2 group_sum2(float a, float b, float2 (*slot)[G / 32], int& turn) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if constexpr (G > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) slot[turn][warp] = make_float2(a, b);
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < G / 32; i++) {
      a += slot[turn][i].x;
      b += slot[turn][i].y;
    }
    turn ^= 1;
  }
  return make_float2(a, b);
}

// Rows in flight: each thread copies its own packs of the next rows to shared
// memory (cp.async, no registers held) and reads them back itself, so no
// barrier is needed. Pack j of a thread covers elements (j G + t) V ...; what
// lies past the row's end is left at zero. Elements of less than four bytes
// (16-bit rows that no 16-byte pack fits) are loaded directly.
constexpr int RING = 2;

template <typename T, int V>
constexpr bool async_copies = V * sizeof(T) >= 4;

template <typename T, int V, int NV, int G>
struct Ring {
  static constexpr int THREADS = G > 32 ? G : WARP_BLOCK;
  static constexpr bool ASYNC = async_copies<T, V>;
  using P = Pack<T, V>;
  static constexpr size_t BYTES = ASYNC ? sizeof(P) * NV * THREADS * RING : 0;
  P* slots;  // [RING][NV][THREADS]
  __device__ __forceinline__ Ring(uint8_t* smem) : slots(reinterpret_cast<P*>(smem)) {}
  __device__ __forceinline__ P* at(int stage, int j) {
    return slots + (stage * NV + j) * THREADS + threadIdx.x;
  }
  __device__ __forceinline__ void clear() {
    if constexpr (ASYNC) {
#pragma unroll
      for (int s = 0; s < RING * NV; s++) {
        P z;
#pragma unroll
        for (int u = 0; u < V; u++) z.v[u] = from_f32<T>(0.0f);
        slots[s * THREADS + threadIdx.x] = z;
      }
    }
  }
  __device__ __forceinline__ void fetch(int stage, const T* row, int t, int packs) {
    if constexpr (ASYNC) {
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const int c = j * G + t;
        if (c < packs) {
          const uint32_t dst = (uint32_t)__cvta_generic_to_shared(at(stage, j));
          if constexpr (sizeof(P) == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst),
                         "l"(reinterpret_cast<const P*>(row) + c)
                         : "memory");
          else
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst),
                         "l"(reinterpret_cast<const P*>(row) + c)
                         : "memory");
        }
      }
    }
  }
  // Pack j of the row in `stage` (ASYNC), or of `row` itself.
  __device__ __forceinline__ P get(int stage, int j, const T* row, int t, int packs) {
    if constexpr (ASYNC) return *at(stage, j);
    P z;
    const int c = j * G + t;
#pragma unroll
    for (int u = 0; u < V; u++) z.v[u] = c < packs ? row[(long)c * V + u] : from_f32<T>(0.0f);
    return z;
  }
};
__device__ __forceinline__ void copies_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
// All but the newest RING - 1 groups of copies have landed.
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
}

template <typename T, int V, int NV, int G>
__global__ void __launch_bounds__(G > 32 ? G : WARP_BLOCK) k_norm_fwd(NormFwd P) {
  pdl_wait();
  constexpr int EPT = NV * V;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float slot[2][G > 32 ? G / 32 : 1];
  int turn = 0;
  const int t = threadIdx.x % G;
  const int packs = (int)(P.d / V);
  const long groups = (long)gridDim.x * (blockDim.x / G);
  long i = (long)blockIdx.x * (blockDim.x / G) + threadIdx.x / G;
  const T* x = static_cast<const T*>(P.x);
  Ring<T, V, NV, G> ring(smem);
  ring.clear();
#pragma unroll
  for (int s = 0; s < RING; s++) {
    if (i + s * groups < P.rows) ring.fetch(s, x + (i + s * groups) * P.ldx, t, packs);
    copies_commit();
  }
  float w[EPT], b[EPT];
#pragma unroll
  for (int j = 0; j < NV; j++) {
#pragma unroll
    for (int u = 0; u < V; u++) {
      const long c = (long)(j * G + t) * V + u;
      w[j * V + u] = P.w && c < P.d ? load_any(P.w, P.wtype, c) : 1.0f;
      b[j * V + u] = P.b && c < P.d ? load_any(P.b, P.wtype, c) : 0.0f;
    }
  }
  for (int stage = 0; i < P.rows; i += groups, stage = stage + 1 == RING ? 0 : stage + 1) {
    copies_wait();
    float v[EPT], s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const Pack<T, V> raw = ring.get(stage, j, x + i * P.ldx, t, packs);
#pragma unroll
      for (int u = 0; u < V; u++) s += v[j * V + u] = to_f32(raw.v[u]);
    }
    if (i + RING * groups < P.rows) ring.fetch(stage, x + (i + RING * groups) * P.ldx, t, packs);
    copies_commit();
    const float mean = group_sum<G>(s, slot, turn) * P.inv_d;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < EPT; k++) {
      v[k] -= mean;
      if ((k / V) * G + t < packs) s = fmaf(v[k], v[k], s);
    }
    const float rstd = 1.0f / sqrtf(group_sum<G>(s, slot, turn) * P.inv_d + P.eps);
    T* out = static_cast<T*>(P.y) + i * P.ldy;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int c = j * G + t;
      if (c < packs) {
        Pack<T, V> o;
#pragma unroll
        for (int u = 0; u < V; u++)
          o.v[u] = from_f32<T>(fmaf(v[j * V + u] * rstd, w[j * V + u], b[j * V + u]));
        reinterpret_cast<Pack<T, V>*>(out)[c] = o;
      }
    }
    if (t == 0) {
      if (P.mean) P.mean[i] = mean;
      if (P.rstd) P.rstd[i] = rstd;
    }
  }
}

// Registers hold each thread's own columns of the two sums; w and the rows'
// elements are read from shared memory where they are needed.
template <typename T, int V, int NV, int G>
__global__ void __launch_bounds__(G > 32 ? G : WARP_BLOCK) k_norm_bwd(NormBwd P) {
  pdl_wait();
  constexpr int EPT = NV * V;
  using R = Ring<T, V, NV, G>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float2 slot[2][G > 32 ? G / 32 : 1];
  __shared__ __align__(16) float ws[EPT * G];
  int turn = 0;
  const int t = threadIdx.x % G;
  const int packs = (int)(P.d / V);
  const long groups = (long)gridDim.x * (blockDim.x / G);
  long i = (long)blockIdx.x * (blockDim.x / G) + threadIdx.x / G;
  const T *x = static_cast<const T*>(P.x), *dy = static_cast<const T*>(P.dy);
  R rx(smem), rg(smem + R::BYTES);
  rx.clear();
  rg.clear();
  auto fetch = [&](int stage, long row) {
    if (row < P.rows) {
      rx.fetch(stage, x + row * P.ldx, t, packs);
      rg.fetch(stage, dy + row * P.lddy, t, packs);
    }
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < RING; s++) fetch(s, i + s * groups);
  for (int c = threadIdx.x; c < EPT * G; c += blockDim.x)
    ws[c] = P.w && c < P.d ? load_any(P.w, P.wtype, c) : 1.0f;
  float dw[EPT], db[EPT];
#pragma unroll
  for (int k = 0; k < EPT; k++) dw[k] = db[k] = 0.0f;
  float mean = 0.0f, rstd = 0.0f;
  if (i < P.rows) {
    mean = P.mean[i];
    rstd = P.rstd[i];
  }
  __syncthreads();
  for (int stage = 0; i < P.rows; i += groups, stage = stage + 1 == RING ? 0 : stage + 1) {
    const float m = mean, r = rstd;
    if (i + groups < P.rows) {
      mean = P.mean[i + groups];
      rstd = P.rstd[i + groups];
    }
    copies_wait();
    const T *xi = x + i * P.ldx, *gi = dy + i * P.lddy;
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const Pack<T, V> xr = rx.get(stage, j, xi, t, packs), gr = rg.get(stage, j, gi, t, packs);
#pragma unroll
      for (int q = 0; q < V; q++) {
        const int k = j * V + q;
        const float g = to_f32(gr.v[q]), u = (to_f32(xr.v[q]) - m) * r;
        dw[k] = fmaf(g, u, dw[k]);
        db[k] += g;
        const float h = g * ws[(j * G + t) * V + q];
        s1 += h;  // elements past d have g = 0
        s2 = fmaf(h, u, s2);
      }
    }
    const float2 c = group_sum2<G>(s1, s2, slot, turn);
    const float c1 = c.x * P.inv_d, c2 = c.y * P.inv_d;
    if (P.dx) {
      T* out = static_cast<T*>(P.dx) + i * P.lddx;
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const int at = j * G + t;
        if (at < packs) {
          const Pack<T, V> xr = rx.get(stage, j, xi, t, packs), gr = rg.get(stage, j, gi, t, packs);
          Pack<T, V> o;
#pragma unroll
          for (int q = 0; q < V; q++) {
            const float h = to_f32(gr.v[q]) * ws[at * V + q], u = (to_f32(xr.v[q]) - m) * r;
            o.v[q] = from_f32<T>(r * (h - c1 - u * c2));
          }
          reinterpret_cast<Pack<T, V>*>(out)[at] = o;
        }
      }
    }
    fetch(stage, i + RING * groups);
  }
  if (!P.part_w) return;
  // The block's groups are added in order, column by column.
  constexpr int GROUPS = (G > 32 ? G : WARP_BLOCK) / G;
  float* pw = P.part_w + (long)blockIdx.x * P.d;
  float* pb = P.part_b + (long)blockIdx.x * P.d;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int k = 0; k < EPT; k++) {
      const long c = (long)((k / V) * G + t) * V + k % V;
      if (c < P.d) {
        pw[c] = dw[k];
        pb[c] = db[k];
      }
    }
  } else {
    __shared__ float acc[2][EPT][G];
    for (int g = 0; g < GROUPS; g++) {
      if ((int)threadIdx.x / G == g) {
#pragma unroll
        for (int k = 0; k < EPT; k++) {
          acc[0][k][t] = g ? acc[0][k][t] + dw[k] : dw[k];
          acc[1][k][t] = g ? acc[1][k][t] + db[k] : db[k];
        }
      }
      __syncthreads();
    }
    for (int q = threadIdx.x; q < EPT * G; q += blockDim.x) {
      const int k = q / G, tt = q % G;
      const long c = (long)((k / V) * G + tt) * V + k % V;
      if (c < P.d) {
        pw[c] = acc[0][k][tt];
        pb[c] = acc[1][k][tt];
      }
    }
  }
}

// Rows too long for registers: one block per row, read again for each pass
// (from L2 for all but the longest rows).
constexpr int LONG_BLOCK = 512;

template <typename T>
__global__ void __launch_bounds__(LONG_BLOCK) k_norm_fwd_long(NormFwd P) {
  pdl_wait();
  __shared__ float slot[2][LONG_BLOCK / 32];
  int turn = 0;
  for (long i = blockIdx.x; i < P.rows; i += gridDim.x) {
    const T* x = static_cast<const T*>(P.x) + i * P.ldx;
    T* y = static_cast<T*>(P.y) + i * P.ldy;
    float s = 0.0f;
    for (long c = threadIdx.x; c < P.d; c += LONG_BLOCK) s += to_f32(x[c]);
    const float mean = group_sum<LONG_BLOCK>(s, slot, turn) * P.inv_d;
    s = 0.0f;
    for (long c = threadIdx.x; c < P.d; c += LONG_BLOCK) {
      const float v = to_f32(x[c]) - mean;
      s = fmaf(v, v, s);
    }
    const float rstd = 1.0f / sqrtf(group_sum<LONG_BLOCK>(s, slot, turn) * P.inv_d + P.eps);
    for (long c = threadIdx.x; c < P.d; c += LONG_BLOCK) {
      const float w = P.w ? load_any(P.w, P.wtype, c) : 1.0f;
      const float b = P.b ? load_any(P.b, P.wtype, c) : 0.0f;
      y[c] = from_f32<T>(fmaf((to_f32(x[c]) - mean) * rstd, w, b));
    }
    if (threadIdx.x == 0) {
      if (P.mean) P.mean[i] = mean;
      if (P.rstd) P.rstd[i] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(LONG_BLOCK) k_norm_bwd_long(NormBwd P) {
  pdl_wait();
  __shared__ float slot[2][LONG_BLOCK / 32];
  int turn = 0;
  float* pw = P.part_w ? P.part_w + (long)blockIdx.x * P.d : nullptr;
  float* pb = P.part_w ? P.part_b + (long)blockIdx.x * P.d : nullptr;
  if (pw)
    for (long c = threadIdx.x; c < P.d; c += LONG_BLOCK) pw[c] = pb[c] = 0.0f;
  for (long i = blockIdx.x; i < P.rows; i += gridDim.x) {
    const T* x = static_cast<const T*>(P.x) + i * P.ldx;
    const T* dy = static_cast<const T*>(P.dy) + i * P.lddy;
    const float mean = P.mean[i], rstd = P.rstd[i];
    float s1 = 0.0f, s2 = 0.0f;
    for (long c = threadIdx.x; c < P.d; c += LONG_BLOCK) {
      const float g = to_f32(dy[c]), u = (to_f32(x[c]) - mean) * rstd;
      const float h = g * (P.w ? load_any(P.w, P.wtype, c) : 1.0f);
      s1 += h;
      s2 = fmaf(h, u, s2);
      if (pw) {  // each thread's own columns of the block's own partial row
        pw[c] = fmaf(g, u, pw[c]);
        pb[c] += g;
      }
    }
    const float c1 = group_sum<LONG_BLOCK>(s1, slot, turn) * P.inv_d;
    const float c2 = group_sum<LONG_BLOCK>(s2, slot, turn) * P.inv_d;
    if (P.dx) {
      T* dx = static_cast<T*>(P.dx) + i * P.lddx;
      for (long c = threadIdx.x; c < P.d; c += LONG_BLOCK) {
        const float u = (to_f32(x[c]) - mean) * rstd;
        const float h = to_f32(dy[c]) * (P.w ? load_any(P.w, P.wtype, c) : 1.0f);
        dx[c] = from_f32<T>(rstd * (h - c1 - u * c2));
      }
    }
  }
}

// Column sums of the blocks' partial rows: 32 columns a block, 32 threads a
// column taking every 32nd partial row, added in order.
__global__ void __launch_bounds__(1024) k_norm_sum(const float* pw, const float* pb, int blocks,
                                                   long d, void* dw, void* db, int wt, int bt) {
  pdl_wait();
  __shared__ float acc[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const long c = (long)blockIdx.x * 32 + cx;
  const float* part = blockIdx.y ? pb : pw;
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  float s = 0.0f;
  if (c < d) {
#pragma unroll 8
    for (int r = ry; r < blocks; r += 32) s += part[(long)r * d + c];
  }
  acc[ry][cx] = s;
  __syncthreads();
  s = acc[cx][ry];  // this warp's column, one partial sum a lane
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (cx == 0 && (long)blockIdx.x * 32 + ry < d)
    store_any(out, blockIdx.y ? bt : wt, (size_t)blockIdx.x * 32 + ry, s);
}

// The grid of a launch whose groups step through the rows: as many blocks as
// stay resident, or fewer when there are fewer rows.
template <typename K>
int resident_blocks(K kern, int threads, size_t smem = 0) {
  int per_sm = 0;
  if (smem)
    EB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  EB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem));
  return per_sm;
}
unsigned resident_grid(eb_engine* e, int per_sm, long rows, int groups) {
  const long need = (rows + groups - 1) / groups;
  return (unsigned)std::max<long>(1, std::min<long>(need, (long)std::max(per_sm, 1) * e->num_sms));
}

// One launch each; by_width picks the template arguments.
template <typename T>
struct FwdLaunch {
  eb_engine* e;
  const NormFwd& P;
  template <int V, int NV, int G>
  void go() {
    constexpr int threads = G > 32 ? G : WARP_BLOCK;
    const auto kern = k_norm_fwd<T, V, NV, G>;
    constexpr size_t smem = Ring<T, V, NV, G>::BYTES;
    static const int per_sm = resident_blocks(kern, threads, smem);
    const unsigned grid = resident_grid(e, per_sm, P.rows, threads / G);
    launch_pdl(e, kern, dim3(grid), dim3(threads), smem, P);
    e->stats.kernel_launches++;
  }
};

// Places the partial rows of dw and db for a grid of that many blocks.
void place_partials(eb_engine* e, NormBwd& P, unsigned grid, bool want) {
  if (!want) return;
  P.part_w = e->scratch_get<float>("norm_part", 2 * (size_t)grid * P.d);
  P.part_b = P.part_w + (size_t)grid * P.d;
}

template <typename T>
struct BwdLaunch {
  eb_engine* e;
  NormBwd& P;
  bool sums;
  unsigned grid;
  template <int V, int NV, int G>
  void go() {
    constexpr int threads = G > 32 ? G : WARP_BLOCK;
    const auto kern = k_norm_bwd<T, V, NV, G>;
    constexpr size_t smem = 2 * Ring<T, V, NV, G>::BYTES;
    static const int per_sm = resident_blocks(kern, threads, smem);
    grid = resident_grid(e, per_sm, P.rows, threads / G);
    place_partials(e, P, grid, sums);
    launch_pdl(e, kern, dim3(grid), dim3(threads), smem, P);
    e->stats.kernel_launches++;
  }
};

// Calls f.go<V, NV, G>() for the smallest group and register
// count that hold a row: one warp up to 1,024 elements, then 128 threads and
// 512 of WIDE elements each. False when a row does not fit.
template <typename T, int WIDE, typename F>
bool by_width(long d, bool packed, F&& f) {
  constexpr int V = 16 / sizeof(T);
  if (packed) {
    const long packs = d / V;
    if (packs <= 32) return f.template go<V, 1, 32>(), true;
    if (packs <= 64) return f.template go<V, 2, 32>(), true;
    if (packs <= 96) return f.template go<V, 3, 32>(), true;
    if (packs <= 128) return f.template go<V, 4, 32>(), true;
    if constexpr (V == 4) {
      if (packs <= 192) return f.template go<V, 6, 32>(), true;
      if (packs <= 256) return f.template go<V, 8, 32>(), true;
    }
    if (packs <= 128 * (32 / V)) return f.template go<V, 32 / V, 128>(), true;
    if (packs <= 512 * (WIDE / V)) return f.template go<V, WIDE / V, 512>(), true;
    return false;
  }
  if (d <= 32 * 4) return f.template go<1, 4, 32>(), true;
  if (d <= 32 * 8) return f.template go<1, 8, 32>(), true;
  if (d <= 32 * 16) return f.template go<1, 16, 32>(), true;
  if (d <= 32 * 32) return f.template go<1, 32, 32>(), true;
  if (d <= 128 * 32) return f.template go<1, 32, 128>(), true;
  if (d <= 512 * WIDE) return f.template go<1, WIDE, 512>(), true;
  return false;
}

template <typename T>
void norm_fwd(eb_engine* e, const NormFwd& P) {
  constexpr int V = 16 / sizeof(T);
  const bool packed = P.d % V == 0 && P.ldx % V == 0 && P.ldy % V == 0;
  if (by_width<T, 32>(P.d, packed, FwdLaunch<T>{e, P})) return;
  static const int per_sm = resident_blocks(k_norm_fwd_long<T>, LONG_BLOCK);
  const unsigned grid = resident_grid(e, per_sm, P.rows, 1);
  launch_pdl(e, k_norm_fwd_long<T>, dim3(grid), dim3(LONG_BLOCK), 0, P);
  e->stats.kernel_launches++;
}

template <typename T>
void norm_bwd(eb_engine* e, NormBwd P, void* dw, void* db, int wt, int bt) {
  constexpr int V = 16 / sizeof(T);
  const bool packed = P.d % V == 0 && P.ldx % V == 0 && P.lddy % V == 0 && P.lddx % V == 0;
  const bool sums = dw || db;
  BwdLaunch<T> one{e, P, sums, 0};
  if (!by_width<T, 16>(P.d, packed, one)) {
    static const int per_sm = resident_blocks(k_norm_bwd_long<T>, LONG_BLOCK);
    one.grid = resident_grid(e, per_sm, P.rows, 1);
    place_partials(e, P, one.grid, sums);
    launch_pdl(e, k_norm_bwd_long<T>, dim3(one.grid), dim3(LONG_BLOCK), 0, P);
    e->stats.kernel_launches++;
  }
  if (sums) {
    launch_pdl(e, k_norm_sum, dim3((unsigned)((P.d + 31) / 32), 2), dim3(1024), 0,
               (const float*)P.part_w, (const float*)P.part_b, (int)one.grid, P.d, dw, db, wt, bt);
    e->stats.kernel_launches++;
  }
}

}  // namespace

void layer_norm(eb_engine* e, const LayerNormArgs& a) {
  if (a.rows == 0) return;
  NormFwd P{a.x, a.weight, a.bias, a.y, a.mean, a.rstd, (long)a.rows, (long)a.d, (long)a.ldx,
            (long)a.ldy, a.eps, 1.0f / (float)a.d, a.wtype};
  if (a.dtype == EB_F32)
    norm_fwd<float>(e, P);
  else if (a.dtype == EB_BF16)
    norm_fwd<__nv_bfloat16>(e, P);
  else
    norm_fwd<__half>(e, P);
}

void layer_norm_backward(eb_engine* e, const LayerNormBackwardArgs& a) {
  if (a.rows == 0) {
    if (a.dweight)
      EB_CUDA(cudaMemsetAsync(a.dweight, 0, a.d * dtype_bytes(a.dwtype), e->stream));
    if (a.dbias) EB_CUDA(cudaMemsetAsync(a.dbias, 0, a.d * dtype_bytes(a.dbtype), e->stream));
    return;
  }
  NormBwd P{a.dy, a.x, a.weight, a.mean, a.rstd, a.dx, nullptr, nullptr, (long)a.rows, (long)a.d,
            (long)a.lddy, (long)a.ldx, (long)(a.dx ? a.lddx : a.ldx), 1.0f / (float)a.d, a.wtype};
  if (a.dtype == EB_F32)
    norm_bwd<float>(e, P, a.dweight, a.dbias, a.dwtype, a.dbtype);
  else if (a.dtype == EB_BF16)
    norm_bwd<__nv_bfloat16>(e, P, a.dweight, a.dbias, a.dwtype, a.dbtype);
  else
    norm_bwd<__half>(e, P, a.dweight, a.dbias, a.dwtype, a.dbtype);
}

}  // namespace eb
