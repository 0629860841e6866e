// The linear cross entropy of small problems, in FP32 on the CUDA cores.
//
// Up to 64 prototypes of up to 64 columns, what a call costs on the tensor
// cores (linear_ce.cu) is its launches: operand preparation, scores, join, P,
// products, sums. Where the operands would need preparation, one kernel here
// does the forward pass and one the backward pass (a second adds the blocks'
// dw): 1,000 x 32 x 64 f32 forward 5.9 us and backward 11.1 (tensor cores 13.9
// and 19.0), 60,000 x 64 x 64 23.8 and 63.2 (51.1 and 85.2). With 128
// prototypes or columns the two are even, and operands that TMA reads as they
// lie take 9.1 and 10.8 there (1,000 x 32 x 64 bf16). (In loops of one call;
// a step of 1,000 x 32 x 64, forward and then backward, takes 12.)
//
// A block of 256 threads holds all prototypes and 16 R rows of x in shared
// memory; a thread keeps R x 4 scores in registers, and the 16 threads of a
// row add up its (max, sum) by shuffles. Backward, P goes to shared memory and
// feeds dx (R x 4 outputs a thread) and the block's own partial dw (4 x 4).
//
// Bound by latency: one round of loads, then d and 64 steps from shared memory
// between barriers.
#include <cuda_runtime.h>

#include <cmath>

#include "elem.h"
#include "engine.h"
#include "softmax.h"
#include "tc.h"

namespace eb {

namespace {

using tc::pdl_trigger;

constexpr int THREADS = 256;
constexpr int MOST = 64;           // prototypes, and columns
constexpr size_t MOST_ROWS = 1 << 19;  // the blocks' partial dw are then at most 256 MB
constexpr int STRIDE = MOST + 4;   // floats of a shared-memory row

struct Small {
  const void* x;
  const void* w;
  long n, ldx, ldw;
  int k, d;
  const uint32_t* targets;
  float scale;
  uint32_t* status;
  // forward
  float* loss;
  float* lse;
  // backward (reads lse)
  const float* dloss;
  int one_dloss;
  void* dx;  // or null
  long lddx;
  int dxtype;
  void* dw;  // or null
  long lddw;
  int dwtype;
  float* part;  // blocks x k x d, or null with one block
};

// COUNT rows of a matrix from row r0 on (zeros past `rows` and past d) into
// shared memory: a warp takes every eighth row, all of them in flight at once.
template <typename T, int COUNT>
__device__ __forceinline__ void load_rows(const void* src, long r0, long rows, long ld, int d,
                                          float* dst) {
  constexpr int EACH = COUNT / (THREADS / 32);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* at = static_cast<const T*>(src) + (r0 + warp) * ld;
  const int live = (int)min((long)EACH, max((rows - r0 - warp + 7) / 8, 0l));
  float v[MOST / 32][EACH];
#pragma unroll
  for (int h = 0; h < MOST / 32; h++)
#pragma unroll
    for (int i = 0; i < EACH; i++)
      v[h][i] = i < live && h * 32 + lane < d ? to_f32(at[i * 8 * ld + h * 32 + lane]) : 0.0f;
#pragma unroll
  for (int h = 0; h < MOST / 32; h++)
#pragma unroll
    for (int i = 0; i < EACH; i++) dst[(warp + i * 8) * STRIDE + h * 32 + lane] = v[h][i];
}

// This thread's scores, rows R ty .. + R against prototypes tx + 16 c; rounded, so
// that none is above its row's log-sum.
template <int R>
__device__ __forceinline__ void scores(const Small& P, const float* xs, const float* ws, int ty,
                                       int tx, float (&z)[R][4]) {
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int c = 0; c < 4; c++) z[r][c] = 0.0f;
  const int groups = (P.d + 3) / 4;
#pragma unroll 4
  for (int q = 0; q < groups; q++) {
    float4 x[R];
#pragma unroll
    for (int r = 0; r < R; r++)
      x[r] = *reinterpret_cast<const float4*>(xs + (R * ty + r) * STRIDE + q * 4);
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const float4 w = *reinterpret_cast<const float4*>(ws + (tx + 16 * c) * STRIDE + q * 4);
#pragma unroll
      for (int r = 0; r < R; r++)
        z[r][c] = fmaf(x[r].w, w.w, fmaf(x[r].z, w.z, fmaf(x[r].y, w.y, fmaf(x[r].x, w.x, z[r][c]))));
    }
  }
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int c = 0; c < 4; c++)
      z[r][c] = __fmul_rn(z[r][c], P.scale);  // not fused with what is taken from it
}

template <typename T, int R>
__global__ void __launch_bounds__(THREADS) k_ce_small(Small P) {
  pdl_trigger();
  pdl_wait();
  constexpr int ROWS = 16 * R;
  __shared__ __align__(16) float xs[ROWS * STRIDE], ws[MOST * STRIDE];
  __shared__ float zt[ROWS];
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const long row0 = (long)blockIdx.x * ROWS;
  load_rows<T, ROWS>(P.x, row0, P.n, P.ldx, P.d, xs);
  load_rows<T, MOST>(P.w, 0, P.k, P.ldw, P.d, ws);
  uint32_t t[R];
#pragma unroll
  for (int r = 0; r < R; r++)
    t[r] = row0 + R * ty + r < P.n ? P.targets[row0 + R * ty + r] : EB_IGNORE;
  __syncthreads();
  float z[R][4];
  scores<R>(P, xs, ws, ty, tx, z);
#pragma unroll
  for (int r = 0; r < R; r++) {
    float m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const int j = tx + 16 * c;
      if (j >= P.k) z[r][c] = -INFINITY;
      if ((uint32_t)j == t[r]) zt[R * ty + r] = z[r][c];
      m = fmaxf(m, z[r][c]);
    }
    // The maximum passes over NaN scores; they reach the sum.
    const float off = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int c = 0; c < 4; c++) sum += ex(z[r][c] - off);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m, o);
      const float os = __shfl_xor_sync(0xffffffffu, sum, o);
      fold(m, sum, make_float2(om, os));
    }
    __syncwarp();
    const long i = row0 + R * ty + r;
    if (tx == 0 && i < P.n) {
      const float l = m + logf(sum);
      P.lse[i] = l;
      if (t[r] >= (uint32_t)P.k) {
        P.loss[i] = 0.0f;
        if (t[r] != EB_IGNORE) atomicOr(P.status, ST_BAD_LABEL);
      } else {
        P.loss[i] = l - zt[R * ty + r];
      }
    }
  }
}

template <typename T, int R>
__global__ void __launch_bounds__(THREADS) k_ce_small_grad(Small P) {
  pdl_trigger();
  pdl_wait();
  constexpr int ROWS = 16 * R;
  __shared__ __align__(16) float xs[ROWS * STRIDE], ws[MOST * STRIDE], ps[ROWS * STRIDE];
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const long row0 = (long)blockIdx.x * ROWS;
  load_rows<T, ROWS>(P.x, row0, P.n, P.ldx, P.d, xs);
  load_rows<T, MOST>(P.w, 0, P.k, P.ldw, P.d, ws);
  uint32_t t[R];
  float g[R], lse[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const long i = row0 + R * ty + r;
    t[r] = i < P.n ? P.targets[i] : EB_IGNORE;
    const bool live = t[r] < (uint32_t)P.k;
    g[r] = live ? P.dloss[P.one_dloss ? 0 : i] * P.scale : 0.0f;
    lse[r] = live ? P.lse[i] : 0.0f;
  }
  __syncthreads();
  float z[R][4];
  scores<R>(P, xs, ws, ty, tx, z);
#pragma unroll
  for (int r = 0; r < R; r++) {
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const int j = tx + 16 * c;
      const float e = z[r][c] - lse[r];
      // The target's p - 1 by expm1: near 1, p's own rounding would be all that
      // is left.
      const float p = (uint32_t)j == t[r] ? expm1f(e) : ex(e);
      ps[(R * ty + r) * STRIDE + j] = g[r] != 0.0f && j < P.k ? p * g[r] : 0.0f;
    }
  }
  __syncthreads();
  const int c0 = tx * 4;
  if (c0 >= P.d) return;
  if (P.dx) {
    float o[R][4] = {};
#pragma unroll 4
    for (int j = 0; j < P.k; j += 4) {
      float4 p[R];
#pragma unroll
      for (int r = 0; r < R; r++)
        p[r] = *reinterpret_cast<const float4*>(ps + (R * ty + r) * STRIDE + j);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const float4 w = *reinterpret_cast<const float4*>(ws + (j + u) * STRIDE + c0);
#pragma unroll
        for (int r = 0; r < R; r++) {
          const float q = u == 0 ? p[r].x : u == 1 ? p[r].y : u == 2 ? p[r].z : p[r].w;
          o[r][0] = fmaf(q, w.x, o[r][0]);
          o[r][1] = fmaf(q, w.y, o[r][1]);
          o[r][2] = fmaf(q, w.z, o[r][2]);
          o[r][3] = fmaf(q, w.w, o[r][3]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
      const long i = row0 + R * ty + r;
#pragma unroll
      for (int v = 0; v < 4; v++)
        if (i < P.n && c0 + v < P.d)
          store_any(P.dx, P.dxtype, (size_t)(i * P.lddx + c0 + v), o[r][v]);
    }
  }
  if (P.dw && ty * 4 < P.k) {
    // Prototypes 4 ty .. + 4.
    float o[4][4] = {};
#pragma unroll 8
    for (int r = 0; r < ROWS; r++) {
      const float4 p4 = *reinterpret_cast<const float4*>(ps + r * STRIDE + ty * 4);
      const float4 x4 = *reinterpret_cast<const float4*>(xs + r * STRIDE + c0);
      const float p[4] = {p4.x, p4.y, p4.z, p4.w}, x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int v = 0; v < 4; v++) o[u][v] = fmaf(p[u], x[v], o[u][v]);
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int j = ty * 4 + u;
#pragma unroll
      for (int v = 0; v < 4; v++) {
        if (j >= P.k || c0 + v >= P.d) continue;
        if (P.part)
          P.part[((long)blockIdx.x * P.k + j) * P.d + c0 + v] = o[u][v];
        else
          store_any(P.dw, P.dwtype, (size_t)j * P.lddw + c0 + v, o[u][v]);
      }
    }
  }
}

// dw from the blocks' partial sums: 32 elements a block, 32 threads an element
// taking every 32nd block, added in order.
__global__ void __launch_bounds__(1024) k_ce_small_sum(const float* __restrict__ part, int blocks,
                                                       Small P) {
  pdl_trigger();
  pdl_wait();
  __shared__ float acc[32][33];
  const int e = threadIdx.x & 31, b0 = threadIdx.x >> 5;
  const int total = P.k * P.d, i = blockIdx.x * 32 + e;
  float s = 0.0f;
  if (i < total) {
#pragma unroll 8
    for (int b = b0; b < blocks; b += 32) s += part[(long)b * total + i];
  }
  acc[b0][e] = s;
  __syncthreads();
  s = acc[e][b0];  // this warp's element, one partial sum a lane
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int q = blockIdx.x * 32 + b0;
  if (e == 0 && q < total) store_any(P.dw, P.dwtype, (size_t)(q / P.d) * P.lddw + q % P.d, s);
}

// Rows a thread: one while 16-row blocks leave an SM at most two.
int rows_a_thread(eb_engine* e, size_t n) { return n <= (size_t)e->num_sms * 32 ? 1 : 2; }

Small base(eb_engine* e, const LinearCeArgs& a) {
  Small P{};
  P.x = a.x;
  P.w = a.w;
  P.n = (long)a.n;
  P.ldx = (long)a.ldx;
  P.ldw = (long)a.ldw;
  P.k = (int)a.k;
  P.d = (int)a.d;
  P.targets = a.targets;
  P.scale = a.scale;
  P.status = e->d_status;
  return P;
}

template <typename T>
void launch(eb_engine* e, const Small& P, int r, bool grad) {
  const auto kern = grad ? (r == 1 ? k_ce_small_grad<T, 1> : k_ce_small_grad<T, 2>)
                         : (r == 1 ? k_ce_small<T, 1> : k_ce_small<T, 2>);
  launch_pdl(e, kern, dim3((unsigned)((P.n + 16 * r - 1) / (16 * r))), dim3(THREADS), 0, P);
  e->stats.kernel_launches++;
}

void launch(eb_engine* e, const Small& P, int dtype, int r, bool grad) {
  if (dtype == EB_F32)
    launch<float>(e, P, r, grad);
  else if (dtype == EB_BF16)
    launch<__nv_bfloat16>(e, P, r, grad);
  else
    launch<__half>(e, P, r, grad);
}

}  // namespace

bool linear_ce_is_small(const LinearCeArgs& a) {
  const bool prepared = a.dtype == EB_F32 || a.ldx % 8 || a.ldw % 8;
  return prepared && a.k <= MOST && a.d <= MOST && a.n <= MOST_ROWS;
}

void linear_ce_small(eb_engine* e, const LinearCeArgs& a, float* loss, float* lse) {
  Small P = base(e, a);
  P.loss = loss;
  P.lse = lse;
  launch(e, P, a.dtype, rows_a_thread(e, a.n), false);
}

void linear_ce_small_backward(eb_engine* e, const LinearCeArgs& a, const LinearCeGrads& g) {
  Small P = base(e, a);
  P.lse = const_cast<float*>(g.lse);
  P.dloss = g.dloss;
  P.one_dloss = g.one_dloss;
  P.dx = g.dx;
  P.lddx = (long)g.lddx;
  P.dxtype = g.dxtype;
  P.dw = g.dw;
  P.lddw = (long)g.lddw;
  P.dwtype = g.dwtype;
  const int r = rows_a_thread(e, a.n);
  const size_t blocks = (a.n + 16 * r - 1) / (16 * r);
  if (g.dw && blocks > 1) P.part = e->scratch_get<float>("ce_small", blocks * a.k * a.d);
  launch(e, P, a.dtype, r, true);
  if (P.part) {
    launch_pdl(e, k_ce_small_sum, dim3((unsigned)((a.k * a.d + 31) / 32)), dim3(1024), 0,
               (const float*)P.part, (int)blocks, P);
    e->stats.kernel_launches++;
  }
}

}  // namespace eb
