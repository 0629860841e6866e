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
// writes dx. 200,000 x 768 bf16 forward 100 to 105 us (5.9 TB/s), backward
// 145 (6.4); 131,072 x 1024 bf16 102 and 143 (5.6). (Forward alone read 105 us on
// one GPU and 118 on another.) Rows of odd length keep
// their 16-byte packs: 200,000 x 767 bf16 141 and 196 us (element by element
// 191 and 438; packs rounded outwards and trimmed 201 and 335). Rows of up to 16
// packs share a warp: 200,000 x 64 bf16 13 and 22 us (a warp each: 41 and 55).
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

// Sum over the group's G threads, in every thread. Groups of a warp's part go
// by shuffles among their own lanes; wider ones add their warps' sums through
// `slot`: two buffers used in turn, so that one barrier per sum is enough.
template <int G>
__device__ __forceinline__ uint32_t group_mask() {
  if constexpr (G >= 32) return 0xffffffffu;
  return ((1u << (G & 31)) - 1u) << (threadIdx.x & 31 & ~(G - 1));
}
template <int G>
constexpr int group_warps = G > 32 ? G / 32 : 1;

template <int G>
__device__ __forceinline__ float group_sum(float v, float (*slot)[group_warps<G>], int& turn) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(group_mask<G>(), v, o);
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
__device__ __forceinline__ float2 group_sum2(float a, float b, float2 (*slot)[group_warps<G>],
                                             int& turn) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) {
    a += __shfl_xor_sync(group_mask<G>(), a, o);
    b += __shfl_xor_sync(group_mask<G>(), b, o);
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

// How a group's threads hold a row. Its 16-byte aligned middle is cut into
// packs: pack j of thread t holds the V elements from (j G + t) V of the middle
// on. EDGES: up to V - 1 elements before the middle and after it are held one
// by one, element x of thread t being edge t + x G. A group steps through rows
// whose middles start alike (the number of groups is a multiple of V), so its
// threads keep the same columns throughout. Without EDGES all rows start and
// end on 16 bytes, or V is 1 (tensors whose rows are not aligned alike).
template <typename T, int V_, int NV_, int G_, bool EDGES>
struct Row {
  static constexpr int V = V_, NV = NV_, G = G_;
  static constexpr int NX = EDGES ? (2 * V + G - 1) / G : 0;  // edges a thread
  static constexpr int THREADS = G > 32 ? G : WARP_BLOCK;
  using P = Pack<T, V>;
  int t, head, packs, d;
  __device__ __forceinline__ Row(long row, long ld, long d_)
      : t(threadIdx.x % G), head(0), d((int)d_) {
    if constexpr (EDGES) head = min((int)((V - row * ld % V) % V), d);
    packs = (d - head) / V;
  }
  __device__ __forceinline__ bool live(int j) const { return j * G + t < packs; }  // pack j
  __device__ __forceinline__ int column(int k) const {  // of element k of the packs
    return head + ((k / V) * G + t) * V + k % V;
  }
  // Column of edge element x, or -1: the first V edges are the head's, then
  // the tail's.
  __device__ __forceinline__ int edge(int x) const {
    const int e = t + x * G;
    const int c = e < V ? e : head + packs * V + e - V;
    return (e < V ? e < head : e < 2 * V && c < d) ? c : -1;
  }
};

// Rows in flight: each thread copies its own packs of the next rows to shared
// memory (cp.async, no registers held) and reads them back itself, so no
// barrier is needed. Packs of less than four bytes (V = 1 of 16-bit types) are
// loaded directly. 200,000 x 768 bf16 forward: two stages 105 us, three 107,
// none 123, the next row in registers 137 (they cost more warps than the row
// brings).
constexpr int RING = 2;

template <typename T, typename R>
struct Ring {
  static constexpr int V = R::V, NV = R::NV;
  using P = typename R::P;
  static constexpr bool ASYNC = sizeof(P) >= 4;
  static constexpr size_t BYTES = ASYNC ? sizeof(P) * NV * R::THREADS * RING : 0;
  P* slots;  // [RING][NV][THREADS]
  __device__ __forceinline__ Ring(uint8_t* smem) : slots(reinterpret_cast<P*>(smem)) {}
  __device__ __forceinline__ P* at(int stage, int j) {
    return slots + (stage * NV + j) * R::THREADS + threadIdx.x;
  }
  static __device__ __forceinline__ P zero() {
    P z;
#pragma unroll
    for (int u = 0; u < V; u++) z.v[u] = from_f32<T>(0.0f);
    return z;
  }
  __device__ __forceinline__ void clear() {
    if constexpr (ASYNC) {
#pragma unroll
      for (int s = 0; s < RING * NV; s++) slots[s * R::THREADS + threadIdx.x] = zero();
    }
  }
  __device__ __forceinline__ void fetch(int stage, const T* row, const R& r) {
    if constexpr (ASYNC) {
#pragma unroll
      for (int j = 0; j < NV; j++) {
        if (!r.live(j)) continue;
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(at(stage, j));
        const T* src = row + r.column(j * V);
        if constexpr (sizeof(P) == 16)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
        else
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
      }
    }
  }
  // Pack j of the row in `stage`, or (not ASYNC) of `row` itself.
  __device__ __forceinline__ P get(int stage, int j, const T* row, const R& r) {
    if constexpr (ASYNC) return *at(stage, j);
    return r.live(j) ? *reinterpret_cast<const P*>(row + r.column(j * V)) : zero();
  }
};
__device__ __forceinline__ void copies_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
// All but the newest RING - 1 groups of copies have landed.
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
}

template <typename T, int V, int NV, int G, bool EDGES>
__global__ void __launch_bounds__(G > 32 ? G : WARP_BLOCK) k_norm_fwd(NormFwd P) {
  pdl_wait();
  using R = Row<T, V, NV, G, EDGES>;
  constexpr int EPT = NV * V, NX = R::NX;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float slot[2][group_warps<G>];
  int turn = 0;
  const long groups = (long)gridDim.x * (blockDim.x / G);
  long i = (long)blockIdx.x * (blockDim.x / G) + threadIdx.x / G;
  const R r(i, P.ldx, P.d);
  const T* x = static_cast<const T*>(P.x);
  Ring<T, R> ring(smem);
  ring.clear();
  auto fetch = [&](int stage, long row) {
    if (row < P.rows) ring.fetch(stage, x + row * P.ldx, r);
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < RING; s++) fetch(s, i + s * groups);
  // Elements 0 .. EPT are the packs', then the edges'.
  float w[EPT + NX], b[EPT + NX], edge[NX ? NX : 1];
#pragma unroll
  for (int k = 0; k < EPT + NX; k++) {
    const int c = k < EPT ? (r.live(k / V) ? r.column(k) : -1) : r.edge(k - EPT);
    w[k] = P.w && c >= 0 ? load_any(P.w, P.wtype, c) : 1.0f;
    b[k] = P.b && c >= 0 ? load_any(P.b, P.wtype, c) : 0.0f;
  }
  auto load_edges = [&](long row) {
#pragma unroll
    for (int q = 0; q < NX; q++)
      edge[q] = row < P.rows && r.edge(q) >= 0 ? to_f32(x[row * P.ldx + r.edge(q)]) : 0.0f;
  };
  load_edges(i);
  for (int stage = 0; i < P.rows; i += groups, stage = stage + 1 == RING ? 0 : stage + 1) {
    copies_wait();
    float v[EPT + NX], s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const Pack<T, V> raw = ring.get(stage, j, x + i * P.ldx, r);
#pragma unroll
      for (int u = 0; u < V; u++) s += v[j * V + u] = to_f32(raw.v[u]);
    }
#pragma unroll
    for (int q = 0; q < NX; q++) s += v[EPT + q] = edge[q];
    fetch(stage, i + RING * groups);
    load_edges(i + groups);
    const float mean = group_sum<G>(s, slot, turn) * P.inv_d;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < EPT + NX; k++) {
      v[k] -= mean;
      if (k < EPT ? r.live(k / V) : r.edge(k - EPT) >= 0) s = fmaf(v[k], v[k], s);
    }
    const float rstd = 1.0f / sqrtf(group_sum<G>(s, slot, turn) * P.inv_d + P.eps);
    T* out = static_cast<T*>(P.y) + i * P.ldy;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      if (!r.live(j)) continue;
      Pack<T, V> o;
#pragma unroll
      for (int u = 0; u < V; u++)
        o.v[u] = from_f32<T>(fmaf(v[j * V + u] * rstd, w[j * V + u], b[j * V + u]));
      *reinterpret_cast<Pack<T, V>*>(out + r.column(j * V)) = o;
    }
#pragma unroll
    for (int q = 0; q < NX; q++)
      if (r.edge(q) >= 0)
        out[r.edge(q)] = from_f32<T>(fmaf(v[EPT + q] * rstd, w[EPT + q], b[EPT + q]));
    if (r.t == 0) {
      if (P.mean) P.mean[i] = mean;
      if (P.rstd) P.rstd[i] = rstd;
    }
  }
}

// Registers hold each thread's own columns of the two sums; w (as this group's
// threads read it) and the rows' packs come from shared memory.
template <typename T, int V, int NV, int G, bool EDGES>
__global__ void __launch_bounds__(G > 32 ? G : WARP_BLOCK) k_norm_bwd(NormBwd P) {
  pdl_wait();
  using R = Row<T, V, NV, G, EDGES>;
  constexpr int EPT = NV * V, NX = R::NX, GROUPS = R::THREADS / G;
  constexpr int MOST = EPT * G + (EDGES ? 2 * V : 0);  // columns of a row
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float2 slot[2][group_warps<G>];
  // w of each group, and at the end each column's sums of the block.
  __shared__ __align__(16) float ws[GROUPS == 1 || GROUPS * EPT * G > 2 * MOST ? GROUPS * EPT * G
                                                                              : 2 * MOST];
  int turn = 0;
  const int group = threadIdx.x / G;
  const long groups = (long)gridDim.x * GROUPS;
  long i = (long)blockIdx.x * GROUPS + group;
  const R r(i, P.ldx, P.d);
  const T *x = static_cast<const T*>(P.x), *dy = static_cast<const T*>(P.dy);
  Ring<T, R> rx(smem), rg(smem + Ring<T, R>::BYTES);
  rx.clear();
  rg.clear();
  auto fetch = [&](int stage, long row) {
    if (row < P.rows) {
      rx.fetch(stage, x + row * P.ldx, r);
      rg.fetch(stage, dy + row * P.lddy, r);
    }
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < RING; s++) fetch(s, i + s * groups);
  float* w = ws + group * EPT * G;
  // Elements 0 .. EPT are the packs', then the edges'.
  float dw[EPT + NX], db[EPT + NX], wx[NX ? NX : 1], ex[NX ? NX : 1], eg[NX ? NX : 1];
#pragma unroll
  for (int k = 0; k < EPT + NX; k++) {
    const int c = k < EPT ? (r.live(k / V) ? r.column(k) : -1) : r.edge(k - EPT);
    const float v = P.w && c >= 0 ? load_any(P.w, P.wtype, c) : 1.0f;
    if (k < EPT)
      w[((k / V) * G + r.t) * V + k % V] = v;
    else
      wx[k - EPT] = v;
    dw[k] = db[k] = 0.0f;
  }
  float mean = 0.0f, rstd = 0.0f;
  auto load_edges = [&](long row) {
#pragma unroll
    for (int q = 0; q < NX; q++) {
      const bool is = row < P.rows && r.edge(q) >= 0;
      ex[q] = is ? to_f32(x[row * P.ldx + r.edge(q)]) : 0.0f;
      eg[q] = is ? to_f32(dy[row * P.lddy + r.edge(q)]) : 0.0f;
    }
    if (row < P.rows) {
      mean = P.mean[row];
      rstd = P.rstd[row];
    }
  };
  load_edges(i);
  for (int stage = 0; i < P.rows; i += groups, stage = stage + 1 == RING ? 0 : stage + 1) {
    const float m = mean, rs = rstd;
    float xe[NX ? NX : 1], ge[NX ? NX : 1];
#pragma unroll
    for (int q = 0; q < NX; q++) {
      xe[q] = ex[q];
      ge[q] = eg[q];
    }
    load_edges(i + groups);
    copies_wait();
    const T *xi = x + i * P.ldx, *gi = dy + i * P.lddy;
    float s1 = 0.0f, s2 = 0.0f;
    // Elements outside the row have g = 0 and v = 0. Their mean is 0 as well: (0 -
    // mean) rstd overflows where rows of 1e36 and more have no spread, and 0
    // times it would be NaN.
    auto add = [&](int k, float g, float v, float mean, float wk) {
      const float u = (v - mean) * rs, h = g * wk;
      dw[k] = fmaf(g, u, dw[k]);
      db[k] += g;
      s1 += h;
      s2 = fmaf(h, u, s2);
    };
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const Pack<T, V> xr = rx.get(stage, j, xi, r), gr = rg.get(stage, j, gi, r);
      const float mean_j = r.live(j) ? m : 0.0f;
#pragma unroll
      for (int q = 0; q < V; q++)
        add(j * V + q, to_f32(gr.v[q]), to_f32(xr.v[q]), mean_j, w[(j * G + r.t) * V + q]);
    }
#pragma unroll
    for (int q = 0; q < NX; q++) add(EPT + q, ge[q], xe[q], r.edge(q) >= 0 ? m : 0.0f, wx[q]);
    const float2 c = group_sum2<G>(s1, s2, slot, turn);
    const float c1 = c.x * P.inv_d, c2 = c.y * P.inv_d;
    if (P.dx) {
      T* out = static_cast<T*>(P.dx) + i * P.lddx;
      auto grad = [&](float g, float v, float wk) {
        return from_f32<T>(rs * (g * wk - c1 - (v - m) * rs * c2));
      };
#pragma unroll
      for (int j = 0; j < NV; j++) {
        if (!r.live(j)) continue;
        const Pack<T, V> xr = rx.get(stage, j, xi, r), gr = rg.get(stage, j, gi, r);
        Pack<T, V> o;
#pragma unroll
        for (int q = 0; q < V; q++)
          o.v[q] = grad(to_f32(gr.v[q]), to_f32(xr.v[q]), w[(j * G + r.t) * V + q]);
        *reinterpret_cast<Pack<T, V>*>(out + r.column(j * V)) = o;
      }
#pragma unroll
      for (int q = 0; q < NX; q++)
        if (r.edge(q) >= 0) out[r.edge(q)] = grad(ge[q], xe[q], wx[q]);
    }
    fetch(stage, i + RING * groups);
  }
  if (!P.part_w) return;
  float* pw = P.part_w + (long)blockIdx.x * P.d;
  float* pb = P.part_b + (long)blockIdx.x * P.d;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int k = 0; k < EPT + NX; k++) {
      const int c = k < EPT ? (r.live(k / V) ? r.column(k) : -1) : r.edge(k - EPT);
      if (c < 0) continue;
      pw[c] = dw[k];
      pb[c] = db[k];
    }
  } else {
    // The block's groups are added in order, column by column.
    float *aw = ws, *ab = ws + MOST;
    for (int g = 0; g < GROUPS; g++) {
      __syncthreads();
      if (group != g) continue;
#pragma unroll
      for (int k = 0; k < EPT + NX; k++) {
        const int c = k < EPT ? (r.live(k / V) ? r.column(k) : -1) : r.edge(k - EPT);
        if (c < 0) continue;
        aw[c] = g ? aw[c] + dw[k] : dw[k];
        ab[c] = g ? ab[c] + db[k] : db[k];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < P.d; c += R::THREADS) {
      pw[c] = aw[c];
      pb[c] = ab[c];
    }
  }
}

// Rows too long for registers: one block per row, read again for each pass
// (from L2 for all but the longest rows).
constexpr int LONG_BLOCK = 512;

template <typename T>
__global__ void __launch_bounds__(LONG_BLOCK) k_norm_fwd_long(NormFwd P) {
  pdl_wait();
  __shared__ float slot[2][group_warps<LONG_BLOCK>];
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
  __shared__ float slot[2][group_warps<LONG_BLOCK>];
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
  EB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem));
  return per_sm;
}
// `multiple`: of the number of groups, so that all rows of a group are aligned
// alike.
unsigned resident_grid(eb_engine* e, int per_sm, long rows, int groups, int multiple = 1) {
  const long step = std::max(1, multiple / groups);
  const long most = std::max<long>((long)std::max(per_sm, 1) * e->num_sms / step * step, step);
  const long need = ((rows + groups - 1) / groups + step - 1) / step * step;
  return (unsigned)std::max<long>(step, std::min<long>(need, most));
}

// One launch each; by_width picks the template arguments.
template <typename T>
struct FwdLaunch {
  eb_engine* e;
  const NormFwd& P;
  template <int V, int NV, int G, bool EDGES>
  void go() {
    constexpr int threads = G > 32 ? G : WARP_BLOCK;
    const auto kern = k_norm_fwd<T, V, NV, G, EDGES>;
    constexpr size_t smem = Ring<T, Row<T, V, NV, G, EDGES>>::BYTES;
    static std::atomic<uint64_t> allowed{0};
    if (smem) allow_smem(e, kern, smem, allowed);
    static const int per_sm = resident_blocks(kern, threads, smem);
    const unsigned grid = resident_grid(e, per_sm, P.rows, threads / G, V);
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
  template <int V, int NV, int G, bool EDGES>
  void go() {
    constexpr int threads = G > 32 ? G : WARP_BLOCK;
    const auto kern = k_norm_bwd<T, V, NV, G, EDGES>;
    constexpr size_t smem = 2 * Ring<T, Row<T, V, NV, G, EDGES>>::BYTES;
    static std::atomic<uint64_t> allowed{0};
    if (smem) allow_smem(e, kern, smem, allowed);
    static const int per_sm = resident_blocks(kern, threads, smem);
    grid = resident_grid(e, per_sm, P.rows, threads / G, V);
    place_partials(e, P, grid, sums);
    launch_pdl(e, kern, dim3(grid), dim3(threads), smem, P);
    e->stats.kernel_launches++;
  }
};

// Calls f.go<V, NV, G, EDGES>() for the group that holds a row with the fewest idle
// packs: part of a warp, one warp, then two to sixteen. More packs a thread
// mean fewer rows in flight an SM, fewer mean more threads that wait for one
// another; between them, in us forward and backward:
//   1,025 to 1,536 elements of 16 bits, two warps of 3 packs against four of 4:
//     100,000 x 1536 bf16 114 and 174, 204 and 291 (four of 2: 115 and 211);
//   to 4,096, four warps of 2 or 3 packs against 4 (f32: twice as many):
//     50,000 x 2496 bf16 87 and 157, 112 and 183; 50,000 x 1537 f32 110 and 160,
//     133 and 317;
//   to 6,144, eight warps of 3 (f32: 6) packs: 30,000 x 6144 bf16 122 and 223.
// With edges, whose threads hold one more element and its place, two warps
// already from 24 packed elements a thread (f32: 16): 131,072 x 1023 bf16 105 and
// 180, one warp 129 and 200; 60,000 x 1023 f32 88 and 136, 94 and 155; without
// edges one warp: 131,072 x 1024 bf16 102 and 143, two 101 and 160. `packed`: the
// tensors' rows are aligned alike. False when a row does not fit (past 8,192
// elements).
template <int V, bool EDGES, typename F>
bool by_packs(long packs, F& f) {
  if (packs <= 4) return f.template go<V, 1, 4, EDGES>(), true;
  if (packs <= 8) return f.template go<V, 1, 8, EDGES>(), true;
  if (packs <= 16) return f.template go<V, 1, 16, EDGES>(), true;
  if (packs <= 32) return f.template go<V, 1, 32, EDGES>(), true;
  if (packs <= 64) return f.template go<V, 2, 32, EDGES>(), true;
  if (packs <= 96) return f.template go<V, 3, 32, EDGES>(), true;
  if constexpr (!EDGES || V == 4) {
    if (packs <= 128) return f.template go<V, 4, 32, EDGES>(), true;
  }
  if constexpr (EDGES) {
    if (packs <= 64 * (16 / V)) return f.template go<V, 16 / V, 64, EDGES>(), true;
  } else if constexpr (V == 4) {
    if (packs <= 192) return f.template go<V, 6, 32, EDGES>(), true;
    if (packs <= 256) return f.template go<V, 8, 32, EDGES>(), true;
  }
  if (packs <= 64 * (24 / V)) return f.template go<V, 24 / V, 64, EDGES>(), true;
  if (packs <= 128 * (16 / V)) return f.template go<V, 16 / V, 128, EDGES>(), true;
  if (packs <= 128 * (24 / V)) return f.template go<V, 24 / V, 128, EDGES>(), true;
  if (packs <= 128 * (32 / V)) return f.template go<V, 32 / V, 128, EDGES>(), true;
  if (packs <= 256 * (24 / V)) return f.template go<V, 24 / V, 256, EDGES>(), true;
  if (packs <= 512 * (16 / V)) return f.template go<V, 16 / V, 512, EDGES>(), true;
  return false;
}
template <typename T, typename F>
bool by_width(long d, long ld, bool packed, F& f) {
  constexpr int V = 16 / sizeof(T);
  if (packed) {
    if (d % V == 0 && ld % V == 0) return by_packs<V, false>(d / V, f);
    return by_packs<V, true>(d / V, f);
  }
  if (d <= 32 * 4) return f.template go<1, 4, 32, false>(), true;
  if (d <= 32 * 16) return f.template go<1, 16, 32, false>(), true;
  if (d <= 32 * 32) return f.template go<1, 32, 32, false>(), true;
  if (d <= 128 * 32) return f.template go<1, 32, 128, false>(), true;
  if (d <= 512 * 16) return f.template go<1, 16, 512, false>(), true;
  return false;
}

template <typename T>
void norm_fwd(eb_engine* e, const NormFwd& P) {
  constexpr int V = 16 / sizeof(T);
  const bool packed = P.ldx % V == P.ldy % V;
  FwdLaunch<T> one{e, P};
  if (by_width<T>(P.d, P.ldx, packed, one)) return;
  static const int per_sm = resident_blocks(k_norm_fwd_long<T>, LONG_BLOCK);
  const unsigned grid = resident_grid(e, per_sm, P.rows, 1);
  launch_pdl(e, k_norm_fwd_long<T>, dim3(grid), dim3(LONG_BLOCK), 0, P);
  e->stats.kernel_launches++;
}

template <typename T>
void norm_bwd(eb_engine* e, NormBwd P, void* dw, void* db, int wt, int bt) {
  constexpr int V = 16 / sizeof(T);
  const bool packed = P.ldx % V == P.lddy % V && P.ldx % V == P.lddx % V;
  const bool sums = dw || db;
  BwdLaunch<T> one{e, P, sums, 0};
  if (!by_width<T>(P.d, P.ldx, packed, one)) {
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
