// The linear cross entropy of few rows, in FP32 on the CUDA cores.
//
// On the tensor cores (linear_ce.cu) f32 operands are scaled and split into two
// FP16 terms first (16-bit ones off TMA's alignment copied): w is read twice and
// written once before the products read it again. Up to 16 rows the arithmetic is less than that: 2 n k d operations
// at n = 16 are 8 a byte of w. Here w is read once forward and twice backward.
//
// Scores: x lies in shared memory; a warp takes four prototypes at a time, its
// lanes the columns in turn, and keeps NR x 4 sums a lane, so that each element
// of x read from shared memory serves four products. The sums over the lanes
// are halved from step to step (a lane sends the half that it gives up), 62
// shuffles for 64 sums. Forward, lanes fold their scores into (max, sum of exp);
// backward they write P (k x NR floats). The gradients then read P and w: a
// thread owns a column, keeps x and its part of dx in registers, and writes
// dw as it goes; the blocks' parts of dx are added in order by a second kernel.
// Columns copied ahead by cp.async (16 prototypes deep) instead of four in
// registers: backward 148 us against 156 at 15 x 41,927 x 547, but 154 against 134 at
// 1 x 40,000 x 1024 and 53 against 41 at 8 x 65,536 x 64: not kept.
//
// Bound by reading w (and writing dw): 1 x 40,000 x 1024 forward 43 us, 3.8 TB/s.
#include <cuda_runtime.h>

#include <cmath>
#include <type_traits>

#include "elem.h"
#include "engine.h"
#include "softmax.h"
#include "tc.h"

namespace eb {

namespace {

using tc::pdl_trigger;

constexpr int THREADS = 256;
constexpr long MOST_ROWS = 16, MOST_HALF_ROWS = 4, MOST_COLUMNS = 1024;
constexpr long MOST_PROTOTYPES = 1l << 22;  // P is then at most 256 MB
constexpr int CHUNK = 32;  // prototypes whose P a block holds (128: the same times)

struct Few {
  const void* x;
  const void* w;
  long n, d, k, ldx, ldw;
  const uint32_t* targets;
  float scale;
  // forward: blocks x n (max, sum of exp), and each row's target score
  float2* part;
  float* zt;
  // backward
  const float* lse;
  const float* dloss;
  int one_dloss;
  float* p;     // k x NR
  float* dx;    // blocks x n x d, or null
  void* dw;     // or null
  long lddw;
  int dwtype;
};

template <typename T, int NR, bool BACKWARD>
__global__ void __launch_bounds__(THREADS, 2) k_few_scores(Few F) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ float xs[];  // NR x dp
  __shared__ float2 joint[THREADS / 32][NR];
  constexpr int V = NR * 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int d = (int)F.d, dp = (d + 31) / 32 * 32;
  for (int t = threadIdx.x; t < NR * dp; t += THREADS) {
    const int i = t / dp, c = t % dp;
    xs[t] = i < F.n && c < d ? to_f32(static_cast<const T*>(F.x)[i * F.ldx + c]) : 0.0f;
  }
  __syncthreads();
  // After the halving a lane holds the sums of this row, V / 32 (at least one)
  // of its four prototypes from `q0` on.
  const int i = lane / (32 / NR);
  const int q0 = V == 64 ? (lane & 1) * 2 : V == 32 ? lane & 3 : (lane >> 1) & 3;
  const uint32_t target = i < F.n ? F.targets[i] : EB_IGNORE;
  float m = -INFINITY, s = 0.0f, lse = 0.0f, g = 0.0f;
  if (BACKWARD && i < F.n && (long)target < F.k) {
    lse = F.lse[i];
    g = F.dloss[F.one_dloss ? 0 : i] * F.scale;
  }
  const long step = (long)gridDim.x * (THREADS / 32) * 4;
  for (long p0 = ((long)blockIdx.x * (THREADS / 32) + warp) * 4; p0 < F.k; p0 += step) {
    const T* w[4];
#pragma unroll
    for (int q = 0; q < 4; q++) 
      w[q] = static_cast<const T*>(F.w) + min(p0 + q, F.k - 1) * F.ldw;
    float a[V];
#pragma unroll
    for (int j = 0; j < V; j++) a[j] = 0.0f;
#pragma unroll 4
    for (int c = lane; c < dp; c += 32) {
      float v[4];
#pragma unroll
      for (int q = 0; q < 4; q++) v[q] = c < d ? to_f32(w[q][c]) : 0.0f;
#pragma unroll
      for (int r = 0; r < NR; r++) {
        const float xv = xs[r * dp + c];
#pragma unroll
        for (int q = 0; q < 4; q++) a[r * 4 + q] = fmaf(xv, v[q], a[r * 4 + q]);
      }
    }
#pragma unroll
    for (int o = 16, have = V; o; o >>= 1) {
      if (have > 1) {
        have /= 2;
        const bool upper = lane & o;
#pragma unroll
        for (int j = 0; j < V / 2; j++) {
          if (j >= have) break;
          const float keep = upper ? a[j + have] : a[j], give = upper ? a[j] : a[j + have];
          a[j] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      } else {
        a[0] += __shfl_xor_sync(0xffffffffu, a[0], o);
      }
    }
#pragma unroll
    for (int j = 0; j < (V == 64 ? 2 : 1); j++) {
      const long p = p0 + q0 + j;
      if (p >= F.k) continue;
      const float z = __fmul_rn(a[j], F.scale);  // not fused with what is taken from it
      if constexpr (BACKWARD) {
        // By expm1 at the target: near 1, p's own rounding would be all that is
        // left. Nothing of a row without a gradient, not even its NaN.
        const float v = p == (long)target ? expm1f(z - lse) : ex(z - lse);
        F.p[p * NR + i] = g == 0.0f ? 0.0f : g * v;
      } else {
        fold(m, s, make_float2(z, 1.0f));
        if (p == (long)target) F.zt[i] = z;
      }
    }
  }
  if constexpr (!BACKWARD) {
    // The lanes of a row, then the block's warps in order.
#pragma unroll
    for (int o = V == 16 ? 2 : 1; o < 32 / NR; o <<= 1) {
      const float mo = __shfl_xor_sync(0xffffffffu, m, o), so = __shfl_xor_sync(0xffffffffu, s, o);
      fold(m, s, make_float2(mo, so));
    }
    if (lane % (32 / NR) == 0) joint[warp][i] = make_float2(m, s);
    __syncthreads();
    if (threadIdx.x < F.n) {
      m = -INFINITY, s = 0.0f;
      for (int v = 0; v < THREADS / 32; v++)
        fold(m, s, joint[v][threadIdx.x]);
      F.part[(long)blockIdx.x * F.n + threadIdx.x] = make_float2(m, s);
    }
  }
}

template <typename T, int NR>
__global__ void __launch_bounds__(1024) k_few_grads(Few F, long per) {
  pdl_trigger();
  pdl_wait();
  __shared__ __align__(16) float ps[CHUNK * NR];
  const long c = threadIdx.x;
  const bool has = c < F.d;
  float x[NR], dx[NR];
#pragma unroll
  for (int i = 0; i < NR; i++) {
    x[i] = has && i < F.n ? to_f32(static_cast<const T*>(F.x)[i * F.ldx + c]) : 0.0f;
    dx[i] = 0.0f;
  }
  const long j0 = blockIdx.x * per, j1 = min(j0 + per, F.k);
  // The next four prototypes' elements are on their way while four are used;
  // past the block's last one they are 0.
  T w[4];
  auto fetch = [&](long j) {
#pragma unroll
    for (int q = 0; q < 4; q++)
      w[q] = has && j + q < j1 ? static_cast<const T*>(F.w)[(j + q) * F.ldw + c] : from_f32<T>(0.0f);
  };
  fetch(j0);
  for (long base = j0; base < j1; base += CHUNK) {
    const int count = (int)min((long)CHUNK, j1 - base);
    __syncthreads();
    for (int t = threadIdx.x; t < CHUNK * NR; t += blockDim.x)
      ps[t] = t < count * NR ? F.p[base * NR + t] : 0.0f;
    __syncthreads();
    for (int p = 0; p < count; p += 4) {
      const float now[4] = {to_f32(w[0]), to_f32(w[1]), to_f32(w[2]), to_f32(w[3])};
      fetch(base + p + 4);
#pragma unroll
      for (int q = 0; q < 4; q++) {
        float dw = 0.0f;
#pragma unroll
        for (int i = 0; i < NR; i += 4) {
          const float4 pv = *reinterpret_cast<const float4*>(&ps[(p + q) * NR + i]);
          const float pr[4] = {pv.x, pv.y, pv.z, pv.w};
#pragma unroll
          for (int u = 0; u < 4; u++) {
            dx[i + u] = fmaf(pr[u], now[q], dx[i + u]);
            dw = fmaf(pr[u], x[i + u], dw);
          }
        }
        if (F.dw && has && p + q < count) {
          const size_t at = (size_t)((base + p + q) * F.lddw + c);
          if constexpr (sizeof(T) == 4)
            static_cast<float*>(F.dw)[at] = dw;
          else
            store_any(F.dw, F.dwtype, at, dw);
        }
      }
    }
  }
  if (!F.dx || !has) return;
#pragma unroll
  for (int i = 0; i < NR; i++) {
    if (i >= F.n) break;
    F.dx[((long)blockIdx.x * F.n + i) * F.d + c] = dx[i];
  }
}

// dx: the blocks' parts in order, 32 elements a block of 8 slices.
__global__ void __launch_bounds__(THREADS)
    k_few_sum(const float* __restrict__ part, int blocks, long total, long d, void* dx, long lddx,
              int type) {
  pdl_trigger();
  pdl_wait();
  __shared__ float joint[8][33];
  const int c = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const long t = (long)blockIdx.x * 32 + c;
  float s = 0.0f;
  if (t < total) {
#pragma unroll 8
    for (int b = slice; b < blocks; b += 8) s += part[b * total + t];
  }
  joint[slice][c] = s;
  __syncthreads();
  if (slice || t >= total) return;
  s = 0.0f;
#pragma unroll
  for (int v = 0; v < 8; v++) s += joint[v][c];
  store_any(dx, type, (size_t)(t / d * lddx + t % d), s);
}

Few few(const LinearCeArgs& a) {
  Few F{};
  F.x = a.x;
  F.w = a.w;
  F.n = (long)a.n;
  F.d = (long)a.d;
  F.k = (long)a.k;
  F.ldx = (long)a.ldx;
  F.ldw = (long)a.ldw;
  F.targets = a.targets;
  F.scale = a.scale;
  return F;
}

template <typename T, int NR, bool BACKWARD>
void scores(eb_engine* e, const Few& F, unsigned grid) {
  const size_t smem = (size_t)NR * ((F.d + 31) / 32 * 32) * 4;
  const auto kern = k_few_scores<T, NR, BACKWARD>;
  static std::atomic<uint64_t> allowed{0};
  allow_smem(e, kern, (size_t)NR * MOST_COLUMNS * 4, allowed);
  launch_pdl(e, kern, dim3(grid), dim3(THREADS), smem, F);
  e->stats.kernel_launches++;
}
template <typename T, int NR>
void grads(eb_engine* e, const Few& F, unsigned grid, unsigned threads, long per) {
  launch_pdl(e, k_few_grads<T, NR>, dim3(grid), dim3(threads), 0, F, per);
  e->stats.kernel_launches++;
}
// Calls f(T{}, NR) for x's type and the padded number of rows.
template <typename F>
void by_type(int dtype, long n, F&& f) {
  if (dtype == EB_BF16) return f(__nv_bfloat16{}, std::integral_constant<int, 4>{});
  if (dtype == EB_F16) return f(__half{}, std::integral_constant<int, 4>{});
  if (n <= 4) return f(float{}, std::integral_constant<int, 4>{});
  if (n <= 8) return f(float{}, std::integral_constant<int, 8>{});
  f(float{}, std::integral_constant<int, 16>{});
}
unsigned scores_grid(eb_engine* e, const LinearCeArgs& a) {
  return (unsigned)std::min<size_t>((a.k + 31) / 32, (size_t)e->num_sms * 2);
}

}  // namespace

// f32 up to 16 rows; forward and backward in us, in loops of one call, here and on the
// tensor cores:
//   1 x 40,000 x 1024 43 and 134, 152 and 244; 16 x 40,000 x 1024 77 and 214, 151 and 240;
//   15 x 41,927 x 547 48 and 156, 102 and 190; 5 x 7,689 x 807 13 and 30, 34 and 58;
//   16 x 60,000 x 8 16 and 47, 41 and 51; 1 x 760 x 506 8 and 12, 18 and 25.
// With more rows the backward pass would lose: at 16 it is bound by its 4 n k d
// operations in FP32 as much as by memory. 16-bit types whose prototypes TMA
// cannot read as they lie (a copy of w, not a split) up to 4 rows:
//   1 x 41,524 x 420 bf16 17 and 59, 31 and 71; 4 x 40,000 x 1023 34 and 122, 62 and 135;
//   2 x 410 x 924 10 and 14, 12 and 16; with more: 9 x 16,885 x 535 22 and 62, 22 and 48.
bool linear_ce_is_few(const LinearCeArgs& a) {
  const bool few = a.dtype == EB_F32 ? (long)a.n <= MOST_ROWS
                                     : a.ldw % 8 && (long)a.n <= MOST_HALF_ROWS;
  return few && (long)a.d <= MOST_COLUMNS && (long)a.k <= MOST_PROTOTYPES;
}

int linear_ce_few_parts(eb_engine* e, const LinearCeArgs& a) { return (int)scores_grid(e, a); }

void linear_ce_few(eb_engine* e, const LinearCeArgs& a, float2* part, float* zt) {
  Few F = few(a);
  F.part = part;
  F.zt = zt;
  by_type(a.dtype, F.n, [&](auto t, auto rows) {
    scores<decltype(t), decltype(rows)::value, false>(e, F, scores_grid(e, a));
  });
}

void linear_ce_few_backward(eb_engine* e, const LinearCeArgs& a, const LinearCeGrads& g) {
  Few F = few(a);
  const int nr = F.n <= 4 ? 4 : F.n <= 8 ? 8 : 16;
  F.lse = g.lse;
  F.dloss = g.dloss;
  F.one_dloss = g.one_dloss;
  F.p = e->scratch_get<float>("ce_p", a.k * nr);
  by_type(a.dtype, F.n, [&](auto t, auto rows) {
    scores<decltype(t), decltype(rows)::value, true>(e, F, scores_grid(e, a));
  });
  const unsigned threads = (unsigned)((a.d + 31) / 32 * 32);  // a column each
  const long most = (long)e->num_sms * (1024 / std::max(threads, 64u));
  const long per = std::max<long>((F.k + most - 1) / most, 4);
  const unsigned grid = (unsigned)((F.k + per - 1) / per);
  F.dx = g.dx ? e->scratch_get<float>("ce_dx", (size_t)grid * a.n * a.d) : nullptr;
  F.dw = g.dw;
  F.lddw = (long)g.lddw;
  F.dwtype = g.dwtype;
  by_type(a.dtype, F.n, [&](auto t, auto rows) {
    grads<decltype(t), decltype(rows)::value>(e, F, grid, threads, per);
  });
  if (!g.dx) return;
  const long total = F.n * F.d;
  launch_pdl(e, k_few_sum, dim3((unsigned)((total + 31) / 32)), dim3(THREADS), 0,
             (const float*)F.dx, (int)grid, total, F.d, g.dx, (long)g.lddx, g.dxtype);
  e->stats.kernel_launches++;
}

}  // namespace eb
