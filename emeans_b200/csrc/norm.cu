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

// This thread's elements of a row: pack j covers elements (j G + t) V ...
template <typename T, int V, int NV, int G>
__device__ __forceinline__ void load_row(const T* row, int t, int packs, Pack<T, V> (&raw)[NV]) {
#pragma unroll
  for (int j = 0; j < NV; j++) {
    const int c = j * G + t;
    if (c < packs) {
      raw[j] = reinterpret_cast<const Pack<T, V>*>(row)[c];
    } else {
#pragma unroll
      for (int u = 0; u < V; u++) raw[j].v[u] = from_f32<T>(0.0f);
    }
  }
}

template <typename T, int V, int NV, int G>
__global__ void __launch_bounds__(G > 32 ? G : WARP_BLOCK) k_norm_fwd(NormFwd P) {
  pdl_wait();
  constexpr int EPT = NV * V;
  __shared__ float slot[2][G > 32 ? G / 32 : 1];
  int turn = 0;
  const int t = threadIdx.x % G;
  const int packs = (int)(P.d / V);
  const long groups = (long)gridDim.x * (blockDim.x / G);
  const long first = (long)blockIdx.x * (blockDim.x / G) + threadIdx.x / G;
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
  for (long i = first; i < P.rows; i += groups) {
    Pack<T, V> raw[NV];
    load_row<T, V, NV, G>(static_cast<const T*>(P.x) + i * P.ldx, t, packs, raw);
    float v[EPT], s = 0.0f;
#pragma unroll
    for (int k = 0; k < EPT; k++) s += v[k] = to_f32(raw[k / V].v[k % V]);
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

template <typename T, int V, int NV, int G>
__global__ void __launch_bounds__(G > 32 ? G : WARP_BLOCK) k_norm_bwd(NormBwd P) {
  pdl_wait();
  constexpr int EPT = NV * V;
  __shared__ float slot[2][G > 32 ? G / 32 : 1];
  int turn = 0;
  const int t = threadIdx.x % G;
  const int packs = (int)(P.d / V);
  const long groups = (long)gridDim.x * (blockDim.x / G);
  const long first = (long)blockIdx.x * (blockDim.x / G) + threadIdx.x / G;
  float w[EPT], dw[EPT], db[EPT];
#pragma unroll
  for (int k = 0; k < EPT; k++) {
    const long c = (long)((k / V) * G + t) * V + k % V;
    w[k] = P.w && c < P.d ? load_any(P.w, P.wtype, c) : 1.0f;
    dw[k] = db[k] = 0.0f;
  }
  for (long i = first; i < P.rows; i += groups) {
    Pack<T, V> xr[NV], gr[NV];
    load_row<T, V, NV, G>(static_cast<const T*>(P.x) + i * P.ldx, t, packs, xr);
    load_row<T, V, NV, G>(static_cast<const T*>(P.dy) + i * P.lddy, t, packs, gr);
    const float mean = P.mean[i], rstd = P.rstd[i];
    float u[EPT], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < EPT; k++) {
      const float g = to_f32(gr[k / V].v[k % V]);
      u[k] = (to_f32(xr[k / V].v[k % V]) - mean) * rstd;
      dw[k] = fmaf(g, u[k], dw[k]);
      db[k] += g;
      const float h = g * w[k];
      s1 += h;  // elements past d have g = 0
      s2 = fmaf(h, u[k], s2);
    }
    const float c1 = group_sum<G>(s1, slot, turn) * P.inv_d;
    const float c2 = group_sum<G>(s2, slot, turn) * P.inv_d;
    if (P.dx) {
      T* out = static_cast<T*>(P.dx) + i * P.lddx;
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const int c = j * G + t;
        if (c < packs) {
          Pack<T, V> o;
#pragma unroll
          for (int q = 0; q < V; q++) {
            const int k = j * V + q;
            o.v[q] = from_f32<T>(rstd * (to_f32(gr[j].v[q]) * w[k] - c1 - u[k] * c2));
          }
          reinterpret_cast<Pack<T, V>*>(out)[c] = o;
        }
      }
    }
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

// Column sums of the blocks' partial rows: 32 columns a block, eight threads a
// column taking every eighth partial row, added in order.
__global__ void __launch_bounds__(256) k_norm_sum(const float* pw, const float* pb, int blocks,
                                                  long d, void* dw, void* db, int wt, int bt) {
  pdl_wait();
  __shared__ float acc[8][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const long c = (long)blockIdx.x * 32 + cx;
  const float* part = blockIdx.y ? pb : pw;
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  float s = 0.0f;
  if (c < d)
    for (int r = ry; r < blocks; r += 8) s += part[(long)r * d + c];
  acc[ry][cx] = s;
  __syncthreads();
  if (ry == 0 && c < d) {
    s = 0.0f;
#pragma unroll
    for (int r = 0; r < 8; r++) s += acc[r][cx];
    store_any(out, blockIdx.y ? bt : wt, c, s);
  }
}

// The grid of a launch whose groups step through the rows: as many blocks as
// stay resident, or fewer when there are fewer rows.
template <typename K>
unsigned resident_grid(eb_engine* e, K kern, int threads, long rows, int groups) {
  int per_sm = 0;
  EB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, 0));
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
    const unsigned grid = resident_grid(e, kern, threads, P.rows, threads / G);
    launch_pdl(e, kern, dim3(grid), dim3(threads), 0, P);
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
    grid = resident_grid(e, kern, threads, P.rows, threads / G);
    place_partials(e, P, grid, sums);
    launch_pdl(e, kern, dim3(grid), dim3(threads), 0, P);
    e->stats.kernel_launches++;
  }
};

// Calls f.go<V, NV, G>() for the smallest group and register
// count that hold a row: one warp up to 1,024 elements, then 128 and 512
// threads. False when a row does not fit.
template <typename T, typename F>
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
    if (packs <= 512 * (32 / V)) return f.template go<V, 32 / V, 512>(), true;
    return false;
  }
  if (d <= 32 * 4) return f.template go<1, 4, 32>(), true;
  if (d <= 32 * 8) return f.template go<1, 8, 32>(), true;
  if (d <= 32 * 16) return f.template go<1, 16, 32>(), true;
  if (d <= 32 * 32) return f.template go<1, 32, 32>(), true;
  if (d <= 128 * 32) return f.template go<1, 32, 128>(), true;
  if (d <= 512 * 32) return f.template go<1, 32, 512>(), true;
  return false;
}

template <typename T>
void norm_fwd(eb_engine* e, const NormFwd& P) {
  constexpr int V = 16 / sizeof(T);
  const bool packed = P.d % V == 0 && P.ldx % V == 0 && P.ldy % V == 0;
  if (by_width<T>(P.d, packed, FwdLaunch<T>{e, P})) return;
  const unsigned grid = resident_grid(e, k_norm_fwd_long<T>, LONG_BLOCK, P.rows, 1);
  launch_pdl(e, k_norm_fwd_long<T>, dim3(grid), dim3(LONG_BLOCK), 0, P);
  e->stats.kernel_launches++;
}

template <typename T>
void norm_bwd(eb_engine* e, NormBwd P, void* dw, void* db, int wt, int bt) {
  constexpr int V = 16 / sizeof(T);
  const bool packed = P.d % V == 0 && P.ldx % V == 0 && P.lddy % V == 0 && P.lddx % V == 0;
  const bool sums = dw || db;
  BwdLaunch<T> one{e, P, sums, 0};
  if (!by_width<T>(P.d, packed, one)) {
    one.grid = resident_grid(e, k_norm_bwd_long<T>, LONG_BLOCK, P.rows, 1);
    place_partials(e, P, one.grid, sums);
    launch_pdl(e, k_norm_bwd_long<T>, dim3(one.grid), dim3(LONG_BLOCK), 0, P);
    e->stats.kernel_launches++;
  }
  if (sums) {
    launch_pdl(e, k_norm_sum, dim3((unsigned)((P.d + 31) / 32), 2), dim3(256), 0,
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
