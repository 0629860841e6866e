// Softmax cross entropy of rows x (n x d) against prototypes w (k x d), and
// its gradients, without keeping the n x k scores.
//
//   z_ij = scale x_i . w_j,  lse_i = log sum_j exp z_ij,  loss_i = lse_i - z_i,t(i)
//   P_ij = g_i scale (exp(z_ij - lse_i) - [j = t(i)]),  dx = P w,  dw = P^T x
//
// All products run in one persistent tcgen05 kernel (k_gemm) with three
// epilogues. Forward: the tile of scores stays in TMEM; its epilogue reduces
// each row's 128 columns to (max, sum of exp) and k_ce_join adds those up.
// Backward, a piece of the prototypes at a time: the scores again, turned
// into P (16-bit terms, engine scratch), then dx += P w and dw = P^T x read that
// piece. Operands are K-major or MN-major as they lie in memory (w is the
// K-major operand of the scores and the MN-major one of dx), so nothing is
// transposed.
//
// P is kept as (g_i / max|g|) (p - [j = t]), whose largest entries are
// rounded with the least error (with one g for all rows they are near -1),
// and max|g| scale multiplies the products in FP32. bf16 keeps P as bf16; f16
// keeps it times 2^14 (probabilities down to 2^-28 stay normal); f32 keeps
// two FP16 terms of P times 2^14. Where a gradient of 16-bit rows is wanted in f32,
// P is three bf16 or two f16 terms and its sums are chained, so that no rounding but
// FP32's is left (with 16-bit gradients P's own rounding adds 15 to 24 % to the
// outputs'): 16,384 x 1,024 x 768 bf16 backward 161 us, 73 with bf16 gradients.
//
// f32 operands: scaled by a power of two so that the largest is below 2^15
// and split into two FP16 terms (22 bits, absolute floor 2^-39 of the
// largest); three products hi.hi + hi.lo + lo.hi add into one FP32
// accumulator. The dropped lo.lo term is 2^-22 of the product. That floor is the
// matrix's, so rows, columns or loss gradients far below the largest would lose
// their last bits, or all of them. Where the smallest row's or column's largest
// element (of those that are not 0) is below 2^-12 of the largest, the operands and
// P are instead split into three bf16 terms each (24 bits, FP32's own range, no
// scale) and multiplied in six products. Where only the rows' loss gradients lie
// that far apart, P and the gradients' products are: the scores again stay the
// forward pass's, to the last bit. The preparation decides it on the device, and
// the same kernels read it. Forward and backward, one way and the other: 3,001 x 5,003
// x 385 62 and 152 us, 83 and 238; 8,192 x 8,192 x 1024 291 and 909, 506 and 1,867.
//
// Bound by the tensor cores, 2 n k d operations forward and 6 n k d backward
// (three times that for f32); for few rows by reading w once. 16,384 x 65,536 x
// 1024 bf16, under the power cap: in loops of one call forward 1.46 ms (1,510
// TFLOP/s) and backward 4.75 ms (1,390), a step of both 7.0 ms; 16,384 x 8,192 x 1024:
// forward 179 us, its kernel's tensor cores active 82 % of the time, the scores
// again 79 %, the gradients 92 %; 8 x 65,536 x 1024 forward 30 us (4.5 TB/s of w).
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cfloat>
#include <cmath>
#include <type_traits>

#include "elem.h"
#include "engine.h"
#include "softmax.h"
#include "tc.h"

namespace eb {

namespace {

using tc::pdl_trigger;

constexpr int BM = 128;   // rows of a tile a CTA holds (TMEM lanes)
constexpr int BN = 256;   // most columns of a tile (TMEM columns of one accumulator)
constexpr int BK = 64;    // k-elements a stage: one 128-byte swizzle row
constexpr int NTHREADS = 384;  // warp 0 loads, warp 1 issues products, warps 4-11 epilogue
constexpr float PSCALE = 16384.0f;  // f16 and f32: P is kept times 2^14

enum Epi { LSE, PROB, OUT };

// Words shared by a call's kernels (device scratch): bits of max|x| and max|w| over
// the finite elements (f32 operands) and of max|dloss| over the rows with a target;
// whether f32 operands, and whether P and the gradients' operands are three bf16
// terms.
enum { S_X, S_W, S_G, S_WIDE, S_WIDE_P, S_WORDS };

// Words that an f32 call's first kernels raise, zero between calls: the same
// magnitudes; the complements of the smallest row's max|x| and max|w| and of the
// smallest |dloss| that are not 0; then, for x and for w, each column's largest, and
// for each range of columns what no column's largest is below. The first product
// kernel zeroes them.
enum { R_X, R_W, R_G, R_X_LOW, R_W_LOW, R_G_LOW, R_COLUMNS };
constexpr int RANGE = 1024;  // columns of a range
__host__ __device__ constexpr long range_count(long d) { return (d + RANGE - 1) / RANGE; }
__host__ __device__ constexpr long found_count(long d) {
  return R_COLUMNS + 2 * (d + range_count(d));
}

// Whether a largest and a smallest magnitude (bits, and the smallest's complement;
// 0: none) lie more than 2^12 apart: two FP16 terms then leave the smallest fewer
// than 26 bits.
__device__ __forceinline__ bool apart(uint32_t top, uint32_t low) {
  return low && __uint_as_float(top) * 0x1p-12f > __uint_as_float(~low);
}

// The power of two that brings a largest magnitude (its bits) below 2^15, as
// its exponent.
__device__ __forceinline__ int split_exp(uint32_t bits) {
  if (bits == 0) return 0;
  const int e = max((int)(bits >> 23), 1) - 127;  // 2^e <= max < 2^(e+1)
  return min(max(14 - e, -126), 126);
}

// Division of 0 <= n < 2^31 by d >= 1 through a multiplication: q = (n + floor(n m /
// 2^32)) >> l with l = ceil(log2 d), m = floor(2^32 (2^l - d) / d) + 1 (Granlund and
// Montgomery, 1994).
struct Divisor {
  uint32_t m, l;
  __host__ static Divisor of(long d) {
    uint32_t l = 0;
    while ((1l << l) < d) l++;
    return {(uint32_t)((((uint64_t)((1l << l) - d)) << 32) / (uint64_t)d + 1), l};
  }
  __device__ __forceinline__ int operator()(int n) const {
    return (int)(((uint32_t)n + __umulhi((uint32_t)n, m)) >> l);
  }
};

// One product D = A B^T of a launch, cut into units: tiles of CG * 128 rows by
// `bn` columns, times splits of k.
struct Prob {
  long M, N, K;
  int bn;           // columns of a tile: a multiple of 32, at most BN
  int mtiles, ntiles, kblocks, kb_split, splits, units;
  int group;        // row tiles that pass over the column tiles together
  Divisor tiles, whole, rows, last;  // by a split's units, a group's, and its row tiles
  int a_mn;         // A is K x M (MN-major) rather than M x K
  // OUT: v = acc scale max|dloss| / pscale, to `out`, or through FP32 sums
  int unscale;      // scal slot of the second operand's largest (f32 operands)
  void* out;
  int otype, ovec;  // ovec: rows of `out` keep 16-byte alignment
  long ldo;
  float* accum;     // M x ldacc (+ split * M * ldacc)
  long ldacc;       // a multiple of 4
  int read_acc, write_acc;
};

struct GemmParams {
  Prob q[2];        // the second only with OUT, after the first's (longer) units
  int skip;         // rounds of the second's units ahead of those for all clusters
  int more, ahead;  // clusters with a first unit more; units in those rounds
  uint32_t fmt;     // operand format of the instruction (0 f16, 1 bf16)
  uint32_t* status;
  int split;        // f32 operands
  int p_terms;      // 16-bit operands: P's terms
  const uint32_t* scal;
  uint32_t* found;  // f32 operands: words to zero for the next call, or null
  long found_words;
  float scale;      // of the scores
  // LSE
  float2* part;     // [2 ntiles][M]: (max, sum) of a half tile's columns
  float* zt;        // M: target scores
  const uint32_t* targets;
  // PROB
  long col0;        // first column of the piece
  const float* lse;
  const float* dloss;
  int one_dloss;
  long k;           // columns in all
  float pscale;     // what P is kept times: 1 (bf16) or PSCALE
};

// CG CTAs a tile, columns up to WIDTH a tile; TERMS: operands of several 16-bit
// terms.
template <int EPI, int CG, bool TERMS, int WIDTH, bool CHAINED>
struct Shape {
  static constexpr int A_ROWS = BM;
  static constexpr int B_ROWS = WIDTH / CG;
  static constexpr int HALF = WIDTH / 2;  // columns an epilogue warp takes
  static constexpr int A_BYTES = A_ROWS * BK * 2;
  static constexpr int B_BYTES = B_ROWS * BK * 2;
  static constexpr int RING = 196608, MOST_STAGES = 8;
  // Operand ring, each epilogue warp's 32 x 32 block, and barriers.
  static constexpr size_t SMEM = 1024 + RING + 8 * 4096 + 256;
  // k-blocks summed in one TMEM accumulator. The tensor cores' FP32 sums are
  // cut, not rounded, at every step of 16 (about 2^-26 of the sum a product,
  // always towards zero): 5.6e-6 of dx at k = 5,003 in one chain of three
  // products a step. CHAINED products end a chain after CHAIN blocks and add it
  // to the epilogue's registers, rounded. Operands of several terms, which aim
  // at FP32's own error, take two: gradients 6e-7 (four: 1.1e-6 and 4 % less time),
  // or with three terms each one (24 products). Scores of 16-bit rows past 768
  // columns: eight (loss 3e-7; unchained 7e-7).
  static constexpr int CHAIN = !CHAINED ? 1 << 28 : TERMS ? 2 : 8;
};

// A launch's tensor maps, one a term: A, B, and C: the second product's B (OUT) or
// P (PROB). Operands that are kept both ways have f16 terms 0 and 1 and bf16 terms 2
// to 4.
template <int T>
struct Maps {
  CUtensorMap a[T], b[T], c[T];
};

// A place of the operand ring, and the parity its barriers have there.
struct Place {
  int s;
  uint32_t parity;
  __device__ __forceinline__ Place next(int stages) const {
    return s + 1 == stages ? Place{0, parity ^ 1} : Place{s + 1, parity};
  }
};

// The softmax of rows whose largest score is past this size goes by rounded scores:
// half their last bit is 2^-14 and more, and the exact products of fmaf would leave a
// row's largest score that much, or (past 2^24) whole units, above or below an lse
// that is that score rounded.
constexpr float STEEP = 1024.0f;

// A warp's 32 x 32 block in shared memory: row r's four-column group g is
// kept at group g ^ (r & 7), so that rows are written by their own threads
// and read across lanes without bank conflicts.
__device__ __forceinline__ float4& block4(float* blk, int r, int g) {
  return reinterpret_cast<float4*>(blk)[r * 8 + (g ^ (r & 7))];
}
// Eight values rounded to 16 bits (bf16, or f16); with REST, what that left of
// them stays in f (exact), for the next term.
template <bool F16, bool REST>
__device__ __forceinline__ uint4 pack8(float (&f)[8]) {
  uint32_t h[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float2 v = make_float2(f[2 * j], f[2 * j + 1]);
    float2 b;
    if constexpr (F16) {
      const __half2 q = __float22half2_rn(v);
      h[j] = *reinterpret_cast<const uint32_t*>(&q);
      b = __half22float2(q);
    } else {
      const __nv_bfloat162 q = __float22bfloat162_rn(v);
      h[j] = *reinterpret_cast<const uint32_t*>(&q);
      b = __bfloat1622float2(q);
    }
    if constexpr (REST) f[2 * j] = v.x - b.x, f[2 * j + 1] = v.y - b.y;
  }
  return make_uint4(h[0], h[1], h[2], h[3]);
}

// The tile and k-range of unit u: within a split, groups of row tiles pass
// over all column tiles, row tile fastest, so that the tiles in flight share
// operands in L2.
struct Unit {
  int prob, mt, nt, split, kb0, kb1;
};
template <int EPI>
__device__ __forceinline__ Unit unit_at(const GemmParams& P, int u) {
  Unit r;
  r.prob = EPI == OUT && u >= P.q[0].units;
  const Prob& q = P.q[r.prob];
  if (r.prob) u -= P.q[0].units;
  r.split = q.tiles(u);
  const int t = u - r.split * q.mtiles * q.ntiles;
  const int g = q.whole(t), w = t - g * q.group * q.ntiles;
  const int gm = min(q.group, q.mtiles - g * q.group);
  r.nt = gm == q.group ? q.rows(w) : q.last(w);
  r.mt = g * q.group + w - r.nt * gm;
  r.kb0 = r.split * q.kb_split;
  r.kb1 = min(r.kb0 + q.kb_split, q.kblocks);
  return r;
}

// A warp's 32 x 32 block of a product, times `factor`, to the output or the
// FP32 sums (at `sums`, the block's first row). Whole blocks go in 16-byte
// groups; what is cut off by the matrix's edge, or whose rows keep no 16-byte
// alignment, a row at a time, a column a lane.
__device__ __forceinline__ void store_block(const Prob& q, float* sums, float* blk, int lane,
                                            long row0, int rows, long col, int cols,
                                            float factor) {
  const bool whole = rows == 32 && cols >= 32;
  if (whole && (q.write_acc || (q.ovec && q.otype == EB_F32))) {
    // Eight lanes a row, four columns each.
    const int g = lane & 7, r = lane >> 3;
    const float* in = sums + r * q.ldacc + col + g * 4;
    const long ld = q.write_acc ? q.ldacc : q.ldo;
    float* out = q.write_acc ? sums + r * ld + col + g * 4
                             : static_cast<float*>(q.out) + (row0 + r) * ld + col + g * 4;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float4 v[4];
#pragma unroll
      for (int t = 0; t < 4; t++) {
        v[t] = block4(blk, r + (h * 4 + t) * 4, g);
        v[t] = make_float4(v[t].x * factor, v[t].y * factor, v[t].z * factor, v[t].w * factor);
      }
      if (q.read_acc) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
          const float4 o = *reinterpret_cast<const float4*>(in + (h * 4 + t) * 4 * q.ldacc);
          v[t] = make_float4(v[t].x + o.x, v[t].y + o.y, v[t].z + o.z, v[t].w + o.w);
        }
      }
#pragma unroll
      for (int t = 0; t < 4; t++) *reinterpret_cast<float4*>(out + (h * 4 + t) * 4 * ld) = v[t];
    }
  } else if (whole && q.ovec) {
    // Four lanes a row, eight columns each.
    const int g = (lane & 3) * 2, r = lane >> 2;
    const float* in = sums + r * q.ldacc + col + g * 4;
    uint16_t* out = static_cast<uint16_t*>(q.out) + (row0 + r) * q.ldo + col + g * 4;
#pragma unroll
    for (int t = 0; t < 4; t++) {
      float4 a = block4(blk, r + t * 8, g), b = block4(blk, r + t * 8, g + 1);
      a = make_float4(a.x * factor, a.y * factor, a.z * factor, a.w * factor);
      b = make_float4(b.x * factor, b.y * factor, b.z * factor, b.w * factor);
      if (q.read_acc) {
        const float4* o = reinterpret_cast<const float4*>(in + t * 8 * q.ldacc);
        a = make_float4(a.x + o[0].x, a.y + o[0].y, a.z + o[0].z, a.w + o[0].w);
        b = make_float4(b.x + o[1].x, b.y + o[1].y, b.z + o[1].z, b.w + o[1].w);
      }
      float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      *reinterpret_cast<uint4*>(out + t * 8 * q.ldo) =
          q.otype == EB_BF16 ? pack8<false, false>(f) : pack8<true, false>(f);
    }
  } else if (lane < cols) {
    float* at = sums + col + lane;
    const size_t out = (size_t)(row0 * q.ldo + col + lane);
    auto value = [&](int r) {
      return reinterpret_cast<const float*>(&block4(blk, r, lane >> 2))[lane & 3] * factor;
    };
    if (q.read_acc) {
#pragma unroll 4
      for (int r = 0; r < rows; r++) {
        const float v = value(r) + at[r * q.ldacc];
        if (q.write_acc)
          at[r * q.ldacc] = v;
        else
          store_any(q.out, q.otype, out + r * q.ldo, v);
      }
    } else if (q.write_acc) {
#pragma unroll 8
      for (int r = 0; r < rows; r++) at[r * q.ldacc] = value(r);
    } else if (q.otype == EB_F32) {
#pragma unroll 8
      for (int r = 0; r < rows; r++) static_cast<float*>(q.out)[out + r * q.ldo] = value(r);
    } else if (q.otype == EB_BF16) {
#pragma unroll 8
      for (int r = 0; r < rows; r++)
        static_cast<__nv_bfloat16*>(q.out)[out + r * q.ldo] = __float2bfloat16_rn(value(r));
    } else {
#pragma unroll 8
      for (int r = 0; r < rows; r++)
        static_cast<__half*>(q.out)[out + r * q.ldo] = __float2half_rn(value(r));
    }
  }
}

// Every operand arrives in boxes of 64 columns by 64 rows (8 KB, 128-byte
// swizzle): a K-major operand's boxes follow one another down its rows, an
// MN-major one's along its columns, so one tensor map serves either reading.
// LSE and PROB: A = x, B = w, both K-major. OUT: A = P, K-major for dx
// (B = w) and MN-major for dw (B = x), B MN-major. With TERMS each operand is
// several 16-bit terms (f32: two f16 or three bf16 ones), or (OUT of 16-bit rows) A
// alone; FINE, PROB leaves several terms of 16-bit rows' P; CHAINED, sums are kept in
// registers between chains.
template <int EPI, int CG, bool TERMS, int WIDTH, bool CHAINED, bool FINE>
__global__ void __launch_bounds__(NTHREADS, 1)
    k_gemm(const __grid_constant__ Maps<TERMS || FINE ? 5 : 1> maps,
           const __grid_constant__ GemmParams P) {
  using S = Shape<EPI, CG, TERMS, WIDTH, CHAINED>;
  constexpr int HALF = S::HALF;
  using namespace tc;
  extern __shared__ uint8_t smem_raw[];
  // Aligned by an offset, not by rounding the pointer: the compiler then knows
  // that it points to shared memory (with generic accesses the step of 16,384
  // x 65,536 x 1024 bf16 took 6.5 ms instead of 6.1).
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  uint64_t* full = (uint64_t*)(smem + S::RING + 8 * 4096);
  uint64_t* empty = full + S::MOST_STAGES;
  uint64_t* tfull = empty + S::MOST_STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* done = tempty + 2;
  uint32_t* tmem_slot = (uint32_t*)(done + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cta_rank() : 0;
  const int units = P.q[0].units + (EPI == OUT ? P.q[1].units : 0);
  // Units go to the clusters in turn. With OUT, `more` clusters get one more of
  // the first product's than the rest, which meanwhile take `skip` rounds of the
  // second's among themselves; what is left goes to all, those first.
  const int cluster = blockIdx.x / CG, step = gridDim.x / CG;
  auto after_long = [&] {
    const int c = cluster - P.more;
    return P.q[0].units + (c < 0 ? P.ahead + c + step : c);
  };
  auto next_unit = [&](int u) {
    if (EPI != OUT) return u + step;
    if (u < P.q[0].units) return u + step < P.q[0].units ? u + step : after_long();
    if (u - P.q[0].units >= P.ahead) return u + step;
    u += step - P.more;
    return u - P.q[0].units < P.ahead ? u : P.q[0].units + P.ahead + cluster - P.more;
  };
  const int first = EPI != OUT || cluster < P.q[0].units ? cluster : after_long();

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::MOST_STAGES; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 8 * CG);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc<CG>(tmem_slot, 512);
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  // Terms of the operands, and what follows from them. A stage holds A's terms,
  // then B's.
  const bool split = TERMS && (EPI != OUT || P.split);
  const bool wide_p = split && EPI != LSE && P.scal[S_WIDE_P];
  const bool wide = EPI == OUT ? wide_p : split && P.scal[S_WIDE];
  const int bf16_at = EPI == OUT && wide && !P.scal[S_WIDE] ? 2 : 0;  // of B's terms
  const int terms = !TERMS ? 1 : !split ? P.p_terms : wide ? 3 : 2;  // of A
  const int b_terms = split ? terms : 1;
  const int stage_bytes = terms * S::A_BYTES + b_terms * S::B_BYTES;
  const int stages = min(S::RING / stage_bytes, S::MOST_STAGES);
  const int chain = wide ? 1 : S::CHAIN;
  auto stage_at = [&](int s) { return smem + s * stage_bytes; };

  // With the sums in registers, the first warpgroup gives some of its own to
  // the epilogue (128 x 72 + 256 x 216 = 384 x 168).
  if (warp < 4) {
    if constexpr (CHAINED) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      const bool one = elect_one();
      int it = 0;
      Place at = {0, 1};
      bool stop = false;
      for (int u = first; u < units && !stop; u = next_unit(u)) {
        const Unit q = unit_at<EPI>(P, u);
        const int am = (q.mt * CG + (int)rank) * BM, bn = q.nt * P.q[q.prob].bn + (int)rank * (P.q[q.prob].bn / CG);
        // Boxes of 64 of each CTA's rows and columns; those past the matrix are
        // left out (what their shared memory holds reaches only rows and
        // columns that are not stored).
        const Prob& pr = P.q[q.prob];
        int a_boxes = 0, b_boxes = 0, all = 0;  // all: of both CTAs and all terms
#pragma unroll
        for (int c = 0; c < CG; c++) {
          const long m = pr.M - (long)(q.mt * CG + c) * BM;
          const long n = min((long)(pr.bn / CG), pr.N - (long)q.nt * pr.bn - c * (pr.bn / CG));
          const int a = (int)min(max(m + 63, 0l) / 64, (long)(S::A_ROWS / 64));
          const int b = (int)(max(n + 63, 0l) / 64);
          if (c == (int)rank) a_boxes = a, b_boxes = b;
          all += terms * a + b_terms * b;
        }
        for (int kb = q.kb0; kb < q.kb1; kb++, it++, at = at.next(stages)) {
          const int s = at.s;
          if (!warp_wait(&empty[s], at.parity, abort_flag)) {
            stop = true;
            break;
          }
          if (!one) continue;
          if (rank == 0) mbar_expect_tx(&full[s], all * 8192);
          const uint32_t bar = CG == 2 ? map_rank(smem_u32(&full[s]), 0) : smem_u32(&full[s]);
          uint8_t* st = stage_at(s);
          const bool a_mn = EPI == OUT && P.q[q.prob].a_mn;
#pragma unroll
          for (int p = 0; p < (TERMS ? 3 : 1); p++) {
            if (p >= terms) break;
#pragma unroll
            for (int c = 0; c < S::A_ROWS / 64; c++, st += 8192) {
              const int m = am + c * 64;
              if (c < a_boxes)
                tma_load<CG>(st, &maps.a[p], bar, a_mn ? m : kb * BK, a_mn ? kb * BK : m);
            }
          }
#pragma unroll
          for (int p = 0; p < (TERMS ? 3 : 1); p++) {
            if (p >= b_terms) break;
            const CUtensorMap* mb = q.prob ? &maps.c[p + bf16_at] : &maps.b[p + bf16_at];
#pragma unroll
            for (int c = 0; c < S::B_ROWS / 64; c++, st += 8192) {
              const int n = bn + c * 64;
              if (c < b_boxes)
                tma_load<CG>(st, mb, bar, EPI == OUT ? n : kb * BK, EPI == OUT ? kb * BK : n);
            }
          }
        }
      }
      // No copy may still be landing when the CTA exits: the first CTA's full
      // barriers count both CTAs' bytes (on the normal path these waits
      // return at once).
      if (rank == 0) {
        for (int j = it > stages ? it - stages : 0; j < it; j++) {
          const uint64_t t0 = now_ns();
          while (!mbar_try(&full[j % stages], (j / stages) & 1) && now_ns() - t0 < WAIT_NS) {
          }
        }
      }
    }
    // The warp walks the loop together and one elected lane issues: as one
    // thread's branch, its addresses came from vector registers and took it longer
    // than the products take the tensor cores (16,384 x 8,192 x 1024 bf16 forward
    // 202 us, 177 now; 512 columns 108 and 97).
    if (warp == 1 && rank == 0) {
      const bool one = elect_one();
      const uint32_t fmt = wide ? 1u : P.fmt;
      Place at = {0, 0};
      int tc = 0;  // counts chains
      bool stop = false;
      for (int u = first; u < units && !stop; u = next_unit(u)) {
        const Unit q = unit_at<EPI>(P, u);
        const bool a_mn = EPI == OUT && P.q[q.prob].a_mn;
        const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((a_mn ? 1u : 0u) << 15) |
                               ((EPI == OUT ? 1u : 0u) << 16) |
                               ((uint32_t)(P.q[q.prob].bn >> 3) << 17) |
                               ((uint32_t)(CG * BM >> 4) << 24);
        for (int k0 = q.kb0; k0 < q.kb1 && !stop; k0 += chain, tc++) {
          const int k1 = min(k0 + chain, q.kb1);
          const uint32_t d = tmem + (tc & 1) * BN;
          if (!warp_wait(&tempty[tc & 1], ((tc >> 1) & 1) ^ 1, abort_flag)) {
            stop = true;
            break;
          }
          fence_after();
          // The products of one stage: of the operands' terms a and b.
          auto multiply = [&](int s, int pa, int pb, uint32_t first) {
            const uint32_t a = smem_u32(stage_at(s)) + pa * S::A_BYTES;
            const uint32_t b = smem_u32(stage_at(s)) + terms * S::A_BYTES + pb * S::B_BYTES;
#pragma unroll
            for (int kk = 0; kk < BK / 16; kk++)
              mma_f16<CG>(d, a_mn ? desc_mn(a + kk * 2048, 8192) : desc_k(a + kk * 32),
                          EPI == OUT ? desc_mn(b + kk * 2048, 8192) : desc_k(b + kk * 32), idesc,
                          kk == 0 ? first : 1u);
          };
          // All of them but the largest, the smallest first.
          auto small = [&](int s, uint32_t first) {
            if (EPI == OUT && !split) {
              if (terms == 3) multiply(s, 2, 0, first);
              multiply(s, 1, 0, terms == 3 ? 1u : first);
              return;
            }
            if (wide) {
              multiply(s, 0, 2, first);
              multiply(s, 1, 1, 1u);
              multiply(s, 2, 0, 1u);
              first = 1u;
            }
            multiply(s, 0, 1, first);
            multiply(s, 1, 0, 1u);
          };
          // Two-term scores take two stages together, the small products of both
          // first: sums are then cut at their full size eight times in the two
          // blocks, not 24. Gradients take a stage at a time (the ring's three
          // stages are held longer otherwise: 8 % of the time), and so do three
          // terms, whose ring has two.
          constexpr int MOST = TERMS && EPI != OUT ? 2 : 1;
          const int together = wide ? 1 : MOST;
          for (int kb = k0; kb < k1 && !stop; kb += together) {
            const int n = min(together, k1 - kb);
            Place p = at;
#pragma unroll
            for (int g = 0; g < MOST; g++) {
              if (g >= n) break;
              if (!warp_wait(&full[p.s], p.parity, abort_flag)) {
                stop = true;
                break;
              }
              fence_after();
              if constexpr (TERMS) {
                if (one) small(p.s, (kb > k0 || g > 0) ? 1u : 0u);
              }
              p = p.next(stages);
            }
            if (stop) break;
#pragma unroll
            for (int g = 0; g < MOST; g++) {
              if (g >= n) break;
              if (one) {
                multiply(at.s, 0, 0, (TERMS || kb > k0) ? 1u : 0u);
                mma_commit<CG>(&empty[at.s]);
              }
              at = at.next(stages);
            }
          }
          if (!stop && one) mma_commit<CG>(&tfull[tc & 1]);
        }
      }
      // Every product this thread issued is complete once `done` flips.
      if (one) mma_commit<CG>(done);
      const uint64_t t0 = now_ns();
      while (!mbar_try(done, 0) && now_ns() - t0 < WAIT_NS) {
      }
    }
  } else {
    if constexpr (CHAINED) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    if constexpr (TERMS && EPI != OUT) {
      if (blockIdx.x == 0)
        for (long t = threadIdx.x - 128; t < P.found_words; t += NTHREADS - 128) P.found[t] = 0;
    }
    // Epilogue: warp w reads TMEM lanes 32 (w % 4) .. + 31, one row a thread,
    // and half (w - 4) / 4 of the tile's columns.
    const int hf = (warp - 4) >> 2;
    const int r = (warp & 3) * 32 + lane;
    float* blk = (float*)(smem + S::RING) + (warp - 4) * 1024;
    const uint32_t base = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(hf * HALF);
    float sc = P.scale, gmax = 0.0f;
    // Kept finite and above 0: products below or past FP32's range leave scores of 0
    // or infinities, not 0 x infinity.
    if (EPI != OUT && TERMS && !wide)
      sc = fminf(fmaxf(ldexpf(sc, -(split_exp(P.scal[S_X]) + split_exp(P.scal[S_W]))), FLT_MIN),
                 FLT_MAX);
    if constexpr (EPI != LSE) {
      gmax = P.one_dloss ? fabsf(P.dloss[0]) : __uint_as_float(P.scal[S_G]);
      // Nothing to be relative to: P takes the rows' own (a non-finite one stays with
      // the rows that have a target).
      // Three bf16 terms of P have FP32's range: they too take the rows' own.
      if (wide_p || !(gmax > 0.0f && gmax < INFINITY)) gmax = 1.0f;
    }
    // What sums become in the outputs. Of several terms: the operand's power of two,
    // the scores' scale and the loss gradients at once where that keeps well within
    // FP32's range (for both products), else one after the other.
    float factors[2] = {P.scale / P.pscale * gmax, P.scale / P.pscale * gmax}, scales[2] = {1.0f, 1.0f};
    bool fine = true;
    if constexpr (EPI == OUT && TERMS) {
#pragma unroll
      for (int r = 0; r < 2; r++) {
        if (!split || wide)
          scales[r] = split ? 1.0f : 1.0f / P.pscale;
        else
          scales[r] = ldexpf(1.0f / P.pscale, -split_exp(P.scal[P.q[r].unscale]));
        const float two = scales[r] * P.scale;
        factors[r] = two * gmax;
        fine = fine && two > 0x1p-90f && two < 0x1p90f && factors[r] > 0x1p-90f && factors[r] < 0x1p90f;
      }
      if (!fine) factors[0] = factors[1] = gmax;
    }
    const uint32_t release = CG == 2 ? map_rank(smem_u32(tempty), 0) : smem_u32(tempty);
    int tc = 0, stores = 0;
    bool stop = false;
    // A tile's row of this thread. The next tile's is fetched while the current
    // one is worked on: with few k-blocks a tile, these loads' latency would be
    // most of its time.
    struct Row {
      uint32_t t;
      float lse, g;
    };
    auto row_of = [&](int u, const Unit& q) {
      Row n = {EB_IGNORE, 0.0f, 0.0f};
      if constexpr (EPI != OUT) {
        if (u < units) {
          const long i = (long)(q.mt * CG + (int)rank) * BM + r;
          if (i < P.q[0].M) {
            n.t = P.targets[i];
            if constexpr (EPI == PROB) {
              n.lse = P.lse[i];
              n.g = P.dloss[P.one_dloss ? 0 : i];
            }
          }
        }
      }
      return n;
    };
    Unit after = unit_at<EPI>(P, first);  // the next tile's
    Row next = row_of(first, after);
    for (int u = first; u < units && !stop; u = next_unit(u)) {
      const Unit q = EPI == OUT ? unit_at<EPI>(P, u) : after;
      if constexpr (EPI != OUT) after = unit_at<EPI>(P, next_unit(u));
      const Prob& pr = P.q[q.prob];
      const long i = (long)(q.mt * CG + (int)rank) * BM + r;
      const bool live = i < pr.M;
      const long c0 = (long)q.nt * pr.bn + hf * HALF;
      const int cols = (int)min((long)min(HALF, pr.bn - hf * HALF), pr.N - c0);  // may be negative
      float m2 = -INFINITY, sum = 0.0f, zt = 0.0f, lse = 0.0f, gr = 0.0f;
      int tcol = -1;  // the target's column among this warp's, if it is one of them
      if constexpr (EPI != OUT) {
        const Row row = next;
        if (row.t != EB_IGNORE) {
          const long rel = (long)row.t - (EPI == PROB ? P.col0 : 0l) - c0;
          if (rel >= 0 && rel < cols) tcol = (int)rel;
          if (EPI == PROB && (long)row.t < P.k) {
            lse = row.lse;
            gr = row.g / gmax;
          }
        }
        next = row_of(next_unit(u), after);
      }
      // exp(v psc + poff) is p.
      const bool steep = EPI == PROB && __any_sync(0xffffffffu, fabsf(lse) > STEEP);
      const float psc = steep ? 1.0f : sc, poff = steep ? 0.0f : -lse;
      // Waits for the next chain; then its TMEM columns are this warp's.
      auto wait_chain = [&] {
        stop = !mbar_wait(&tfull[tc & 1], (tc >> 1) & 1, abort_flag);
        fence_after();
        return !stop;
      };
      auto release_chain = [&] {
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_at(release + (tc & 1) * 8);
        tc++;
      };
      float acc[CHAINED ? HALF : 1];
      if constexpr (CHAINED) {
#pragma unroll
        for (int j = 0; j < HALF; j++) acc[j] = 0.0f;
        for (int k0 = q.kb0; k0 < q.kb1; k0 += chain) {
          if (!wait_chain()) break;
#pragma unroll
          for (int h = 0; h < HALF / 16; h++) {
            if (h * 16 >= cols) break;
            uint32_t raw[16];
            tmem_ld16(base + (tc & 1) * BN + h * 16, raw);
            ld_wait(raw);
#pragma unroll
            for (int j = 0; j < 16; j++) acc[h * 16 + j] += __uint_as_float(raw[j]);
          }
          release_chain();
        }
      } else {
        wait_chain();
      }
      if (stop) break;
      const float factor = q.prob ? factors[1] : factors[0];
      uint32_t raw[CHAINED ? 1 : 32];
      if constexpr (!CHAINED) tmem_ld32(base + (tc & 1) * BN, raw);
#pragma unroll
      for (int h = 0; h < HALF / 32; h++) {
        float v[32];
        if constexpr (CHAINED) {
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = acc[h * 32 + j];
        } else {
          ld_wait(raw);
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = __uint_as_float(raw[j]);
          // The next columns are on their way while these are worked on.
          if (h + 1 < HALF / 32)
            tmem_ld32(base + (tc & 1) * BN + (h + 1) * 32, raw);
          else
            release_chain();
        }
        if (EPI != LSE && h * 32 >= cols) continue;
        const int left = cols - h * 32;
        if constexpr (EPI == LSE) {
          if (left < 32) {
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = j < left ? v[j] : -INFINITY;
          }
          if (tcol >> 5 == h) {  // through shared memory: registers have no index
#pragma unroll
            for (int g = 0; g < 8; g++)
              block4(blk, lane, g) = make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
            zt = reinterpret_cast<const float*>(&block4(blk, lane, (tcol & 31) >> 2))[tcol & 3];
          }
          // The maximum passes over NaN scores; they reach the sum.
          float top[4] = {m2, v[0], v[1], v[2]};
#pragma unroll
          for (int j = 3; j < 32; j++) top[j & 3] = fmaxf(top[j & 3], v[j]);
          const float m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
          const float off = m == -INFINITY ? 0.0f : -m * sc;
          float part[4] = {sum * ex(fmaf(m2, sc, off)), 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < 32; j++) part[j & 3] += ex(fmaf(v[j], sc, off));
          sum = (part[0] + part[1]) + (part[2] + part[3]);
          m2 = m;
        } else if constexpr (EPI == PROB) {
          const bool target = tcol >> 5 == h;
          const int e = tcol & 31;
          float at_target = 0.0f;
          if (steep) {  // no score is above lse (a NaN stays one)
#pragma unroll
            for (int j = 0; j < 32; j++) {
              v[j] = __fmul_rn(v[j], sc) - lse;
              v[j] = v[j] > 0.0f ? 0.0f : v[j];
            }
          }
          if (target) {  // by expm1: near 1, p's own rounding would be all that is left
            float z = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; j++) z = j == e ? v[j] : z;
            at_target = gr * expm1f(fmaf(z, psc, poff));
          }
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = ex(fmaf(v[j], psc, poff)) * gr;
          if (gr == 0.0f) {  // nothing of a row without a gradient, not even its NaN
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = 0.0f;
            at_target = 0.0f;
          }
          // A row a thread, 64 bytes a term, 16-byte groups placed by the 64-byte
          // swizzle; a tile store takes the block to P and cuts it at P's
          // edges. One-term blocks go through two buffers in turn, two terms
          // through both, and three through them in turn again. (Transposed
          // in shared memory as FP32 and stored by four lanes a row: backward
          // 16,384 x 8,192 x 256 bf16 221 us, 211 now, x 1,024 x 768 78 and 74,
          // 8,192 x 8,192 x 256 f32 272 and 263.)
          const int turn = (lane >> 1) & 3;
          constexpr bool SEVERAL = TERMS || FINE;
          const bool bf = TERMS ? wide_p : P.fmt;
          if (!bf) {
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] *= PSCALE;
            at_target *= PSCALE;
          }
          // One round: a term of the block to `box` (and the next to what follows it),
          // then to P; v and at_target keep the rest.
          auto round = [&](uint8_t* box, int term, auto as_f16, auto both) {
            constexpr bool F16 = decltype(as_f16)::value, BOTH = decltype(both)::value;
            uint8_t* row = box + lane * 64;
            __syncwarp();
#pragma unroll
            for (int g = 0; g < 4; g++) {
              float f[8];
#pragma unroll
              for (int j = 0; j < 8; j++) f[j] = v[8 * g + j];
              uint8_t* at = row + ((g ^ turn) << 4);
              *reinterpret_cast<uint4*>(at) = pack8<F16, SEVERAL>(f);
              if constexpr (BOTH) *reinterpret_cast<uint4*>(at + 2048) = pack8<F16, false>(f);
              if constexpr (SEVERAL && !BOTH) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[8 * g + j] = f[j];
              }
            }
            if (target) {
              float f[8] = {at_target};
              uint8_t* at = row + (((e >> 3) ^ turn) << 4) + (e & 7) * 2;
              *reinterpret_cast<uint16_t*>(at) = (uint16_t)pack8<F16, SEVERAL>(f).x;
              if constexpr (BOTH)
                *reinterpret_cast<uint16_t*>(at + 2048) = (uint16_t)pack8<F16, false>(f).x;
              at_target = f[0];
            }
            store_fence();
            __syncwarp();
            if (lane == 0) {
              const int row0 = (int)i, col = (int)c0 + h * 32;
              if (row0 < pr.M) {
                tma_store(&maps.c[term], box, col, row0);
                if constexpr (BOTH) tma_store(&maps.c[term + 1], box + 2048, col, row0);
              }
              stores_commit();
            }
          };
          constexpr std::true_type yes{};
          constexpr std::false_type no{};
          uint8_t* boxes = (uint8_t*)blk;
          if constexpr (!SEVERAL) {
            if (lane == 0) stores_read<1>();
            uint8_t* box = boxes + (stores++ & 1) * 2048;
            if (bf)
              round(box, 0, no, no);
            else
              round(box, 0, yes, no);
          } else if (!bf) {
            if (lane == 0) stores_read<0>();
            round(boxes, 0, yes, yes);
          } else {
#pragma unroll 1
            for (int p = 0; p < 3; p++, stores++) {
              if (lane == 0) stores_read<1>();
              round(boxes + (stores & 1) * 2048, p, no, no);
            }
          }
        } else {
          if (TERMS && !fine) {
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = v[j] * (q.prob ? scales[1] : scales[0]) * P.scale;
          }
          __syncwarp();
#pragma unroll
          for (int g = 0; g < 8; g++)
            block4(blk, lane, g) = make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
          __syncwarp();
          const long row0 = i - lane, col = c0 + h * 32;
          store_block(pr, pr.accum + ((long)q.split * pr.M + row0) * pr.ldacc, blk, lane, row0,
                      (int)min(32l, pr.M - row0), col, min(left, 32), factor);
        }
      }
      if constexpr (EPI == LSE) {
        if (live) {
          // Past STEEP the sum goes by the largest score itself, not its rounded value,
          // as P will: 1 where the others are nothing beside it.
          const float top = m2 * sc, off = fmaf(m2, sc, -top);
          if (fabsf(top) > STEEP && top > -INFINITY)
            sum = fabsf(off) < 60.0f || isnan(sum) ? sum * ex(-off) : 1.0f;
          P.part[(long)(q.nt * 2 + hf) * pr.M + i] = make_float2(top, sum);
          if (tcol >= 0) P.zt[i] = zt * sc;
        }
      }
    }
    if (EPI == PROB && lane == 0) stores_done();
  }

  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  if (warp == 1) {
    fence_after();
    tmem_free<CG>(tmem, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(P.status, ST_WAIT_TIMEOUT);
}

// One row's lse and loss from its (max, sum).
__device__ __forceinline__ void finish_row(long i, float m, float s, long k, const float* zt,
                                           const uint32_t* targets, float* loss, float* lse,
                                           uint32_t* status) {
  const float l = m + logf(s);
  lse[i] = l;
  const uint32_t t = targets[i];
  if (t == EB_IGNORE || (long)t >= k) {
    loss[i] = 0.0f;
    if (t != EB_IGNORE) atomicOr(status, ST_BAD_LABEL);
  } else {
    loss[i] = l - zt[i];
  }
}

// lse and loss of 32 rows from their half tiles' (max, sum): 32 threads a row
// take every 32nd half tile, then the row's thread adds the 32 in order.
__global__ void __launch_bounds__(1024)
    k_ce_join(const float2* __restrict__ part, int parts, long n, long k,
              const float* __restrict__ zt, const uint32_t* __restrict__ targets, float* loss,
              float* lse, uint32_t* status) {
  pdl_trigger();
  pdl_wait();
  __shared__ float2 acc[32][33];
  const int rx = threadIdx.x & 31, py = threadIdx.x >> 5;
  const long i = (long)blockIdx.x * 32 + rx;
  float m = -INFINITY, s = 0.0f;
  if (i < n) {
#pragma unroll 4
    for (int p = py; p < parts; p += 32) fold(m, s, part[(long)p * n + i]);
  }
  acc[py][rx] = make_float2(m, s);
  __syncthreads();
  if (py || i >= n) return;
  for (int p = 1; p < 32; p++) fold(m, s, acc[p][rx]);
  finish_row(i, m, s, k, zt, targets, loss, lse, status);
}

// The same for few rows: a block a row, so that its half tiles are one round of
// loads (8 rows of 592: 2 us less than 32 rows a block).
__global__ void __launch_bounds__(256)
    k_ce_join_row(const float2* __restrict__ part, int parts, long n, long k,
                  const float* __restrict__ zt, const uint32_t* __restrict__ targets, float* loss,
                  float* lse, uint32_t* status) {
  pdl_trigger();
  pdl_wait();
  __shared__ float2 acc[8];
  const long i = blockIdx.x;
  float m = -INFINITY, s = 0.0f;
#pragma unroll 4
  for (int p = threadIdx.x; p < parts; p += 256) fold(m, s, part[(long)p * n + i]);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
    fold(m, s, make_float2(om, os));
  }
  if ((threadIdx.x & 31) == 0) acc[threadIdx.x >> 5] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x) return;
  for (int p = 1; p < 8; p++) fold(m, s, acc[p]);
  finish_row(i, m, s, k, zt, targets, loss, lse, status);
}

// The same for few half tiles: one thread a row.
__global__ void __launch_bounds__(128)
    k_ce_join_few(const float2* __restrict__ part, int parts, long n, long k,
                  const float* __restrict__ zt, const uint32_t* __restrict__ targets, float* loss,
                  float* lse, uint32_t* status) {
  pdl_trigger();
  pdl_wait();
  const long i = (long)blockIdx.x * 128 + threadIdx.x;
  if (i >= n) return;
  float m = -INFINITY, s = 0.0f;
#pragma unroll 8
  for (int p = 0; p < parts; p++) fold(m, s, part[(long)p * n + i]);
  finish_row(i, m, s, k, zt, targets, loss, lse, status);
}

// Rows of an operand on their way to rows of dp 16-bit elements (zeros past
// d): f32 as two or three terms (`term` elements apart), 16-bit types as they are.
// `blocks` of a launch work on it.
struct Prep {
  const void* x;
  long rows, d, ld, dp;
  uint16_t* out;
  long term;
  unsigned blocks;
};
constexpr int PREP_BLOCKS = 1024;  // most blocks of a launch for one operand

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}
__device__ __forceinline__ uint32_t block_max(uint32_t m) {
  __shared__ uint32_t all[8];
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) all[threadIdx.x >> 5] = m;
  __syncthreads();
  m = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) m = max(m, all[i]);
  return m;
}

// Eight elements of a matrix from element `at` on, of which the first `live` are
// wanted (the others come as zeros); `end`: elements the matrix holds. Where
// `at` is not on 16 bytes, the aligned groups around them are loaded and
// shifted.
__device__ __forceinline__ void load8(const float* x, long at, int live, long end, float (&f)[8]) {
  const int s = (int)(at & 3);
  if (at - s + 12 <= end) {
    float v[12];
#pragma unroll
    for (int g = 0; g < 3; g++) {
      if (g == 2 && s == 0) continue;
      const float4 q = *reinterpret_cast<const float4*>(x + at - s + 4 * g);
      v[4 * g] = q.x, v[4 * g + 1] = q.y, v[4 * g + 2] = q.z, v[4 * g + 3] = q.w;
    }
    if (s == 0) v[8] = v[9] = v[10] = v[11] = 0.0f;
#pragma unroll
    for (int j = 0; j < 10; j++) v[j] = s & 2 ? v[j + 2] : v[j];
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = s & 1 ? v[j + 1] : v[j];
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = j < live ? f[j] : 0.0f;
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = j < live ? x[at + j] : 0.0f;
  }
}
__device__ __forceinline__ uint4 load8(const uint16_t* x, long at, int live, long end) {
  const int s = (int)(at & 7);
  uint32_t w[8];
  if (at - s + 16 <= end) {
    const uint4* p = reinterpret_cast<const uint4*>(x + at - s);
    const uint4 a = p[0], b = p[1];
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
#pragma unroll
    for (int j = 0; j < 6; j++) w[j] = s & 4 ? w[j + 2] : w[j];
#pragma unroll
    for (int j = 0; j < 5; j++) w[j] = s & 2 ? w[j + 1] : w[j];
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = s & 1 ? __funnelshift_r(w[j], w[j + 1], 16) : w[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t lo = 2 * j < live ? x[at + 2 * j] : 0, hi = 2 * j + 1 < live ? x[at + 2 * j + 1] : 0;
      w[j] = lo | hi << 16;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if (2 * j >= live)
      w[j] = 0;
    else if (2 * j + 1 >= live)
      w[j] &= 0xFFFFu;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Calls f(row, column, elements left in the row) for each group of eight
// columns of the operand's rows, consecutive threads taking consecutive
// groups whatever the rows' length.
template <typename F>
__device__ __forceinline__ void for_groups(const Prep& q, unsigned block, F&& f) {
  const unsigned groups = (unsigned)(q.dp / 8);
  const long total = q.rows * groups, step = (long)q.blocks * 256;
#pragma unroll 2
  for (long t = (long)block * 256 + threadIdx.x; t < total; t += step) {
    const long i = total <= 0xFFFFFFFFl ? (long)((unsigned)t / groups) : t / groups;
    const long c = (t - i * groups) * 8;
    f(i, c, (int)min(8l, q.d - c));
  }
}

// Whether a matrix's columns lie too far apart, for all of a block's 256 threads: no
// column of a range is below its word (some block saw every column that large), or,
// where there is none, as every block had columns of zeros or far smaller ones, from the
// columns' own words.
__device__ __forceinline__ bool columns_apart(const uint32_t* found, long d, uint32_t top) {
  bool far = false, by_column = false;
  uint32_t low = 0;
  for (long r = 0; r < range_count(d); r++) {
    const uint32_t least = found[d + r];
    if (least) {
      far |= apart(top, ~least);
      continue;
    }
    by_column = true;
#pragma unroll 4
    for (long c = r * RANGE + threadIdx.x; c < min((r + 1) * RANGE, d); c += 256) {
      const uint32_t m = found[c];
      if (m) low = max(low, ~m);
    }
  }
  return by_column ? __syncthreads_or(far || apart(top, low)) : far;
}

// The magnitudes of both operands' finite elements: the largest, the
// smallest row's largest (of its part in a range of columns) and each column's. L
// lanes take a row, eight columns at a time; a block keeps to one range, whose
// largest elements a lane keeps in registers. A block all of whose columns come
// within 2^-12 of its largest element leaves their smallest largest, as any other
// block's can only be added to it; only one that finds columns of zeros or far
// smaller ones leaves each column's (all blocks: 10 us of atomics at 4,096 x 768). 3,001
// x 5,003 x 385: 10 us.
template <int L, int PASSES>
__global__ void __launch_bounds__(256, 2)
    k_ce_max(Prep X, Prep W, uint32_t* found) {
  constexpr int COLS = 8 * L * PASSES;
  static_assert(COLS <= RANGE, "a block's columns are one range's");
  __shared__ uint32_t cols[COLS], rows[3];
  pdl_trigger();
  pdl_wait();
  const bool second = blockIdx.x >= X.blocks;
  const Prep& q = second ? W : X;
  const int ranges = (int)range_count(q.d);
  const unsigned block = blockIdx.x - (second ? X.blocks : 0), range = block % ranges;
  const long c0 = (long)range * RANGE, end = (q.rows - 1) * q.ld + q.d;
  const long last_c = min(c0 + COLS, q.dp) - 8;  // the last eight columns
  const int lane = threadIdx.x % L;
  const float* x = static_cast<const float*>(q.x);
  for (int t = threadIdx.x; t < COLS; t += 256) cols[t] = 0;
  if (threadIdx.x < 3) rows[threadIdx.x] = threadIdx.x < 2 ? 0 : ~0u;
  uint32_t top = 0, low = 0, col[PASSES][8] = {};
  const long step = (long)(q.blocks / ranges) * (256 / L);
  for (long r0 = (long)(block / ranges) * (256 / L); r0 < q.rows; r0 += step) {
    const long i = r0 + threadIdx.x / L;
    const int s = (int)(i * q.ld & 3);
    uint32_t m = 0;
    auto add = [&](int p, const float (&f)[8]) {
      const long live = q.d - (c0 + (p * L + lane) * 8);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const uint32_t b = j < live ? finite_bits(f[j]) : 0;
        col[p][j] = max(col[p][j], b);
        m = max(m, b);
      }
    };
    if (i < q.rows && i * q.ld + last_c + 12 <= end) {
      // All loads of the row first: the aligned groups around eight columns (a
      // lane past the row takes its last ones), shifted as in load8.
      float4 v[PASSES][3];
      const float* row = x + (i * q.ld - s);
#pragma unroll
      for (int p = 0; p < PASSES; p++) {
        if (c0 + p * L * 8 > last_c) break;
        const float* at = row + min(c0 + (p * L + lane) * 8, last_c);
#pragma unroll
        for (int g = 0; g < 3; g++) v[p][g] = reinterpret_cast<const float4*>(at)[g];
      }
#pragma unroll
      for (int p = 0; p < PASSES; p++) {
        if (c0 + p * L * 8 > last_c) break;
        float f[12];
#pragma unroll
        for (int g = 0; g < 3; g++)
          f[4 * g] = v[p][g].x, f[4 * g + 1] = v[p][g].y, f[4 * g + 2] = v[p][g].z, f[4 * g + 3] = v[p][g].w;
#pragma unroll
        for (int j = 0; j < 10; j++) f[j] = s & 2 ? f[j + 2] : f[j];
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = s & 1 ? f[j + 1] : f[j];
        add(p, e);
      }
    } else if (i < q.rows) {  // the matrix's end
#pragma unroll 1
      for (int p = 0; p < PASSES; p++) {
        const long c = c0 + (p * L + lane) * 8;
        if (c >= q.d) break;
        float f[8];
        load8(x, i * q.ld + c, (int)min(8l, q.d - c), end, f);
#pragma unroll
        for (int u = 0; u < PASSES; u++)
          if (u == p) add(u, f);
      }
    }
#pragma unroll
    for (int o = L / 2; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    top = max(top, m);
    if (m) low = max(low, ~m);
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < PASSES; p++)
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (col[p][j]) atomicMax(&cols[(p * 8 + j) * L + lane], col[p][j]);
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_max_sync(0xffffffffu, low);
  if (threadIdx.x % 32 == 0) {
    atomicMax(&rows[0], top);
    atomicMax(&rows[1], low);
  }
  __syncthreads();
  auto column = [&](int t) { return c0 + (t / (8 * L) * L + t % L) * 8 + t / L % 8; };
  uint32_t least = ~0u;
#pragma unroll
  for (int t = threadIdx.x; t < COLS; t += 256)
    if (column(t) < q.d) least = min(least, cols[t]);
  least = __reduce_min_sync(0xffffffffu, least);
  if (threadIdx.x % 32 == 0) atomicMin(&rows[2], least);
  __syncthreads();
  least = rows[2];
  uint32_t* mine = found + R_COLUMNS + (second ? q.d + ranges : 0);
  const bool by_column = !least || apart(rows[0], ~least);
  if (by_column) {
#pragma unroll
    for (int t = threadIdx.x; t < COLS; t += 256)
      if (column(t) < q.d && cols[t]) atomicMax(mine + column(t), cols[t]);
  }
  if (threadIdx.x == 0) {
    atomicMax(found + (second ? R_W : R_X), rows[0]);
    atomicMax(found + (second ? R_W_LOW : R_X_LOW), rows[1]);
    if (!by_column) atomicMax(mine + q.d + range, least);
  }
}

// The operands' 16-bit rows; with SPLIT, in two f16 terms scaled by the largest
// element, or, where rows or columns lie too far apart for that, in three bf16
// terms, or both ways where the loss gradients do; the first block leaves what the
// products need in `scal`.
template <bool SPLIT>
__global__ void __launch_bounds__(256)
    k_ce_rows(Prep X, Prep W, const uint32_t* __restrict__ found, uint32_t* scal) {
  pdl_trigger();
  pdl_wait();
  const bool second = blockIdx.x >= X.blocks;
  const Prep& q = second ? W : X;
  bool wide = false, wide_p = false;
  float s = 1.0f;
  if constexpr (SPLIT) {
    uint32_t word[R_COLUMNS];
#pragma unroll
    for (int t = 0; t < R_COLUMNS; t++) word[t] = found[t];
    const uint32_t x = word[R_X], w = word[R_W], g = word[R_G];
    const bool far_x = columns_apart(found + R_COLUMNS, q.d, x);
    const bool far_w = columns_apart(found + R_COLUMNS + q.d + range_count(q.d), q.d, w);
    wide = apart(x, word[R_X_LOW]) || apart(w, word[R_W_LOW]) || far_x || far_w;
    wide_p = wide || apart(g, word[R_G_LOW]);
    s = ldexpf(1.0f, split_exp(second ? w : x));
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      scal[S_X] = x;
      scal[S_W] = w;
      scal[S_G] = g;
      scal[S_WIDE] = wide;
      scal[S_WIDE_P] = wide_p;
    }
  }
  const long end = (q.rows - 1) * q.ld + q.d;
  for_groups(q, blockIdx.x - (second ? X.blocks : 0), [&](long i, long c, int live) {
    uint16_t* out = q.out + i * q.dp + c;
    auto put = [&](int term, const uint4& v) { *reinterpret_cast<uint4*>(out + term * q.term) = v; };
    if constexpr (SPLIT) {
      float f[8];
      load8(static_cast<const float*>(q.x), i * q.ld + c, live, end, f);
#pragma unroll
      for (int j = 0; j < 8; j++) f[j] = isfinite(f[j]) ? f[j] : NAN;
      if (!wide) {
        float h[8];
#pragma unroll
        for (int j = 0; j < 8; j++) h[j] = f[j] * s;
#pragma unroll
        for (int j = 0; j < 2; j++) put(j, pack8<true, true>(h));
      }
      if (wide_p) {
#pragma unroll
        for (int j = 0; j < 3; j++) put(wide ? j : j + 2, pack8<false, true>(f));
      }
    } else {
      put(0, load8(static_cast<const uint16_t*>(q.x), i * q.ld + c, live, end));
    }
  });
}

// Largest and smallest magnitude of the rows' loss gradients (finite ones that
// are not 0, of rows with a target: what the others hold is not used), into
// zeroed words; `least` may be null.
__global__ void __launch_bounds__(256)
    k_ce_gmax(const float* __restrict__ g, const uint32_t* __restrict__ targets, long n, long k,
              uint32_t* most, uint32_t* least) {
  pdl_trigger();
  pdl_wait();
  uint32_t top = 0, low = 0;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const uint32_t m = (long)targets[i] < k ? finite_bits(g[i]) : 0;
    top = max(top, m);
    if (m) low = max(low, ~m);
  }
  top = block_max(top);
  __syncthreads();
  low = block_max(low);
  if (threadIdx.x == 0 && top) {
    atomicMax(most, top);
    if (least) atomicMax(least, low);
  }
}

// The outputs of a product that ran in splits of k: the sum of the splits'
// partial products (M x ld each), plus the FP32 sums so far. A group of four
// outputs is a thread's; with `slices` as many threads', each taking every
// slices-th split, joined in order: 105 groups in 74 splits (the gradient of 1 x
// 420 from 41,524 prototypes) are otherwise one block's, a load at a time.
__global__ void __launch_bounds__(256)
    k_ce_reduce(const float* __restrict__ part, int splits, int slices, Prob q) {
  __shared__ float4 joint[256];
  pdl_trigger();
  pdl_wait();
  const int each = 256 / slices, lane = threadIdx.x % each, slice = threadIdx.x / each;
  const long groups = q.ldacc / 4, total = q.M * groups;
  for (long t0 = (long)blockIdx.x * each; t0 < total; t0 += (long)gridDim.x * each) {
    const long t = t0 + lane;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](const float4& v) { s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w); };
    if (t < total) {
#pragma unroll 4
      for (int p = slice; p < splits; p += slices)
        add(reinterpret_cast<const float4*>(part)[(long)p * total + t]);
    }
    if (slices > 1) {
      __syncthreads();
      joint[threadIdx.x] = s;
      __syncthreads();
      for (int j = 1; j < slices && slice == 0; j++) add(joint[j * each + lane]);
    }
    if (slice || t >= total) continue;
    if (q.read_acc) add(reinterpret_cast<const float4*>(q.accum)[t]);
    if (q.write_acc) {
      reinterpret_cast<float4*>(q.accum)[t] = s;
    } else {
      const long i = t / groups, c = t % groups * 4;
      const float f[4] = {s.x, s.y, s.z, s.w};
      const size_t at = (size_t)(i * q.ldo + c);
      if (q.ovec && c + 4 <= q.N) {
        if (q.otype == EB_F32) {
          *reinterpret_cast<float4*>(static_cast<float*>(q.out) + at) = s;
        } else {
          Pack<uint16_t, 4> h;
#pragma unroll
          for (int j = 0; j < 4; j++)
            h.v[j] = q.otype == EB_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f[j]))
                                        : __half_as_ushort(__float2half_rn(f[j]));
          *reinterpret_cast<Pack<uint16_t, 4>*>(static_cast<uint16_t*>(q.out) + at) = h;
        }
      } else {
        for (int j = 0; j < 4 && c + j < q.N; j++) store_any(q.out, q.otype, at + j, f[j]);
      }
    }
  }
}

// ---------------------------------------------------------------- host side

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    EB_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q));
    if (q != cudaDriverEntryPointSuccess || !p)
      throw Error(EB_ERROR, "cuTensorMapEncodeTiled is not available from the driver");
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// A 16-bit operand: rows x cols, row stride ld (a multiple of 8), and the room
// of one, three or five terms, `term` elements apart.
struct Operand {
  const uint16_t* at;
  long term;
  int terms;
  long rows, cols, ld;
};

// Read in boxes of 64 columns (128 bytes) by 64 rows, 128-byte swizzle; P is
// written in boxes of 32 by 32, 64-byte swizzle. Every box's first column is a
// multiple of 64, or 32.
CUtensorMap make_map(const Operand& o, int term, bool store = false) {
  CUtensorMap m;
  cuuint64_t dims[2] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows};
  cuuint64_t strides[1] = {(cuuint64_t)o.ld * 2};
  cuuint32_t box[2] = {store ? 32u : 64u, store ? 32u : 64u};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2,
                           const_cast<uint16_t*>(o.at + term * o.term), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE,
                           store ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error(EB_ERROR, "cuTensorMapEncodeTiled failed: " + std::to_string(r));
  return m;
}

template <int EPI, int CG, bool TERMS, int WIDTH, bool CHAINED = TERMS, bool FINE = false>
void launch_gemm(eb_engine* e, const Operand& A, const Operand& B, const Operand& C,
                 GemmParams P) {
  using S = Shape<EPI, CG, TERMS, WIDTH, CHAINED>;
  const auto kern = k_gemm<EPI, CG, TERMS, WIDTH, CHAINED, FINE>;
  static std::atomic<uint64_t> allowed{0};
  allow_smem(e, kern, S::SMEM, allowed);
  Maps<TERMS || FINE ? 5 : 1> maps;
  for (int t = 0; t < (TERMS || FINE ? 5 : 1); t++) {  // what an operand lacks is not read
    maps.a[t] = t < A.terms ? make_map(A, t) : maps.a[0];
    maps.b[t] = t < B.terms ? make_map(B, t) : maps.b[0];
    maps.c[t] = EPI == LSE || t >= C.terms ? maps.b[0] : make_map(C, t, EPI == PROB);
  }
  const int units = P.q[0].units + P.q[1].units;
  const int clusters = std::min(units, e->num_sms / CG);
  P.more = P.q[0].units % clusters;
  P.ahead = P.skip * (clusters - P.more);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * CG));
  cfg.blockDim = dim3(NTHREADS);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = e->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = EB_PDL;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 ? 2 : 1;
  cuda_check(cudaLaunchKernelEx(&cfg, kern, maps, P), "linear cross entropy");
  e->stats.kernel_launches++;
}

// A tile's shape: CTAs that share it (128 rows each) and its most columns.
enum Tile { PAIR, SINGLE, NARROW };  // 256 x 256, 128 x 256 (f32: 128), 128 x 64
struct TileCost {
  int ctas, width;
  double block_us, tile_us;  // a k-block of 64, and what the last tile adds
};
TileCost tile_cost(Tile t, int parts) {
  if (t == PAIR) return {2, 256, parts == 2 ? 0.84 : 0.28, 3.0};
  if (t == SINGLE) return {1, parts == 2 ? 128 : 256, parts == 2 ? 0.45 : 0.28, 2.5};
  return {1, 64, parts == 2 ? 0.3 : 0.15, 1.2};
}

// The product in tiles of at most `width` columns, all of one width: as few
// tiles as that allows (385 columns of 256: two of 224, a fifth less work than
// two of 256), or with `clusters` the width from 5/8 of the most up whose
// rounds of that many tiles take least (65,536 columns of one row tile: 224
// wide, two full rounds of 148).
Prob make_prob(long M, long N, long K, const TileCost& t, int clusters = 0) {
  Prob q{};
  q.M = M;
  q.N = N;
  q.K = K;
  q.mtiles = (int)((M + t.ctas * BM - 1) / (t.ctas * BM));
  const long few = (N + t.width - 1) / t.width;
  q.bn = (int)(((N + few - 1) / few + 31) / 32 * 32);
  if (clusters && few > 1) {
    long best = -1;
    for (int w = t.width; w >= t.width * 5 / 8; w -= 32) {
      const long tiles = q.mtiles * ((N + w - 1) / w);
      const long cost = (tiles + clusters - 1) / clusters * (w + 32);
      if (best < 0 || cost < best) {
        best = cost;
        q.bn = w;
      }
    }
  }
  q.ntiles = (int)((N + q.bn - 1) / q.bn);
  q.kblocks = (int)((K + BK - 1) / BK);
  q.kb_split = q.kblocks;
  q.splits = 1;
  q.units = q.mtiles * q.ntiles;
  q.group = std::min(q.mtiles, 8);
  return q;
}

// The scores' tiles: by rounds of tiles. A narrow tile spreads a small problem
// over more SMs and holds more k-blocks in flight; where the rows' count of 128
// is odd a pair's second half would stand idle in the last.
Tile score_tile(eb_engine* e, long M, long N, long K, int parts) {
  Tile best = PAIR;
  double least = 1e300;
  for (Tile t : {PAIR, SINGLE, NARROW}) {
    if (t == SINGLE && (M + BM - 1) / BM % 2 == 0) continue;
    const TileCost c = tile_cost(t, parts);
    const int clusters = e->num_sms / c.ctas;
    const Prob q = make_prob(M, N, K, c, clusters);
    const long rounds = (q.units + clusters - 1) / clusters;
    const double us = (double)rounds * q.kblocks * c.block_us * q.bn / c.width + c.tile_us * rounds;
    if (us < least) {
      least = us;
      best = t;
    }
  }
  return best;
}

template <int EPI, bool TERMS, bool CHAINED, bool FINE>
void launch_tile(eb_engine* e, const Operand& A, const Operand& B, const Operand& C, Tile t,
                 const GemmParams& P) {
  if (t == NARROW)
    launch_gemm<EPI, 1, TERMS, 64, CHAINED, FINE>(e, A, B, C, P);
  else if (t == SINGLE)
    launch_gemm<EPI, 1, TERMS, TERMS ? 128 : 256, CHAINED, FINE>(e, A, B, C, P);
  else
    launch_gemm<EPI, 2, TERMS, 256, CHAINED, FINE>(e, A, B, C, P);
}

template <int EPI>
void gemm(eb_engine* e, const Operand& A, const Operand& B, const Operand& C, Tile t,
          GemmParams P) {
  P.status = e->d_status;
  for (Prob& q : P.q) {
    if (!q.units) continue;
    q.tiles = Divisor::of((long)q.mtiles * q.ntiles);
    q.whole = Divisor::of((long)q.group * q.ntiles);
    q.rows = Divisor::of(q.group);
    q.last = Divisor::of(std::max(q.mtiles % q.group, 1));
  }
  if (A.terms > 1) return launch_tile<EPI, true, true, false>(e, A, B, C, t, P);
  // The same chains in both passes: the scores again are the forward pass's, to the
  // last bit.
  const bool chained = EPI != OUT && P.q[0].kblocks > 12;
  if constexpr (EPI == PROB) {
    if (C.terms > 1)
      return chained ? launch_tile<EPI, false, true, true>(e, A, B, C, t, P)
                     : launch_tile<EPI, false, false, true>(e, A, B, C, t, P);
  }
  if constexpr (EPI != OUT) {
    if (chained) return launch_tile<EPI, false, true, false>(e, A, B, C, t, P);
  }
  launch_tile<EPI, false, false, false>(e, A, B, C, t, P);
}

// The words that f32 calls raise, zero between them: a call that failed before its
// products left them as they were.
uint32_t* found_words(eb_engine* e, const LinearCeArgs& a) {
  uint32_t* found = e->scratch_get<uint32_t>("ce_found", found_count(a.d), true);
  if (e->ce_found_raised) {
    auto& all = e->scratch["ce_found"];
    EB_CUDA(cudaMemsetAsync(all.p, 0, all.bytes, e->stream));
    e->ce_found_raised = false;
  }
  return found;
}

// The 16-bit operands of x and w: each itself where TMA can read it (16-bit,
// row stride a multiple of 16 bytes), else a copy in scratch; f32 split into two or
// three terms, or (`both`: the loss gradients may ask for it) five.
void operands(eb_engine* e, const LinearCeArgs& a, uint32_t* found, uint32_t* scal, Operand& X,
              Operand& W, bool both = false) {
  const bool split = a.dtype == EB_F32;
  Prep prep[2] = {};
  const void* src[2] = {a.x, a.w};
  const size_t rows[2] = {a.n, a.k}, ld[2] = {a.ldx, a.ldw};
  Operand* out[2] = {&X, &W};
  for (int i = 0; i < 2; i++) {
    Operand& o = *out[i];
    o = Operand{static_cast<const uint16_t*>(src[i]), 0, 1, (long)rows[i], (long)a.d, (long)ld[i]};
    if (!split && ld[i] % 8 == 0) continue;
    o.ld = ((long)a.d + 7) / 8 * 8;
    o.term = (long)rows[i] * o.ld;
    o.terms = !split ? 1 : both ? 5 : 3;
    uint16_t* c = e->scratch_get<uint16_t>(i ? "ce_w" : "ce_x", (size_t)(o.term * o.terms));
    o.at = c;
    prep[i] = Prep{src[i], (long)rows[i], (long)a.d, (long)ld[i], o.ld, c, o.term,
                   (unsigned)std::min<size_t>((rows[i] * (size_t)(o.ld / 8) + 255) / 256, PREP_BLOCKS)};
  }
  const unsigned grid = prep[0].blocks + prep[1].blocks;
  if (!grid) return;
  if (split) {
    // Lanes of a row, and blocks: each takes its share of the rows of one range.
    e->ce_found_raised = true;
    const int lanes = a.d <= 64 ? 8 : a.d <= 128 ? 16 : 32;
    const int passes = (int)std::min<size_t>((a.d + 255) / 256, 4);
    const auto kern = lanes == 8    ? k_ce_max<8, 1>
                      : lanes == 16 ? k_ce_max<16, 1>
                      : passes == 1 ? k_ce_max<32, 1>
                      : passes == 2 ? k_ce_max<32, 2>
                      : passes == 3 ? k_ce_max<32, 3>
                                    : k_ce_max<32, 4>;
    const long resident = (passes == 1 ? 4 : passes == 2 ? 3 : 2) * (long)e->num_sms;
    Prep m[2] = {prep[0], prep[1]};
    for (Prep& q : m) {
      const long each = 256 / lanes, ranges = range_count(q.d);
      const long most = (resident * q.rows / (long)(a.n + a.k) + ranges) / ranges;
      q.blocks = (unsigned)(ranges * std::min((q.rows + each - 1) / each, most));
    }
    launch_pdl(e, kern, dim3(m[0].blocks + m[1].blocks), dim3(256), 0, m[0], m[1], found);
    launch_pdl(e, k_ce_rows<true>, dim3(grid), dim3(256), 0, prep[0], prep[1],
               (const uint32_t*)found, scal);
    e->stats.kernel_launches += 2;
  } else {
    launch_pdl(e, k_ce_rows<false>, dim3(grid), dim3(256), 0, prep[0], prep[1],
               (const uint32_t*)nullptr, scal);
    e->stats.kernel_launches++;
  }
}

Operand rows_of(const Operand& o, long r0, long r1) {
  Operand p = o;
  p.at += r0 * o.ld;
  p.rows = r1 - r0;
  return p;
}

GemmParams base_params(const LinearCeArgs& a, uint32_t* found, const uint32_t* scal) {
  GemmParams P{};
  P.split = a.dtype == EB_F32;
  P.found = found;
  P.found_words = found ? found_count((long)a.d) : 0;
  P.scal = scal;
  P.scale = a.scale;
  P.fmt = a.dtype == EB_BF16 ? 1u : 0u;
  P.targets = a.targets;
  P.k = (long)a.k;
  P.pscale = a.dtype == EB_BF16 ? 1.0f : PSCALE;
  return P;
}

// Splits of k for the products of one launch, chosen over a few counts by an
// estimate (returned, us) of its last cluster's end: units go to the clusters in
// turn, the longer product's first, and clusters with one of those less go
// ahead with `skip` rounds of the other's (16,384 x 8,192 x 1024 bf16: 128 units of
// 256 k-blocks on 74 clusters and 256 of 128, backward 580 us -> 546). A split product also
// writes and reads its partial sums again in a launch of its own.
double choose_splits(Prob* q, int count, int clusters, const TileCost& t, int* skip) {
  static const int tries[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64};
  auto len = [](const Prob& p, int s) { return (p.kblocks + s - 1) / s; };
  double best = 1e300;
  int pick[2] = {1, 1};
  for (int s0 : tries) {
    if (s0 > 1 && len(q[0], s0) < 2) break;
    for (int s1 : tries) {
      if (s1 > 1 && (count < 2 || len(q[1], s1) < 2)) break;
      const int s[2] = {s0, s1};
      double extra_us = 0;
      long units[2] = {0, 0}, l[2] = {0, 0};
      for (int i = 0; i < count; i++) {
        l[i] = len(q[i], s[i]);
        units[i] = (long)q[i].mtiles * q[i].ntiles * ((q[i].kblocks + l[i] - 1) / l[i]);
        if (s[i] > 1) extra_us += 3.0 + (double)q[i].M * q[i].ldacc * 4 * (s[i] + 1) / 4e6;
      }
      const int a = l[0] >= l[1] ? 0 : 1;
      auto unit_us = [&](int i) {  // a narrower tile's blocks take that much less
        return std::max(l[i] * t.block_us * std::max(q[i].bn, 96) / std::max(t.width, 96),
                        t.tile_us * q[i].bn / t.width);
      };
      const double ua = unit_us(a), ub = units[1 - a] ? unit_us(1 - a) : 0.0;
      const long ra = (units[a] + clusters - 1) / clusters, rest = units[a] % clusters;
      const long free = clusters - rest;
      const int rounds = rest && ub > 0.0 ? (int)(ua / ub) : 0;  // ahead of the others
      double us = ra * ua;
      if (units[1 - a] > 0 && units[1 - a] <= rounds * free) {
        us = std::max(us, (ra - 1) * ua + (units[1 - a] + free - 1) / free * ub);
      } else if (units[1 - a] > 0) {
        const long left = units[1 - a] - rounds * free, rb = (left + clusters - 1) / clusters;
        const bool free_last = rest && left - (rb - 1) * clusters <= free;
        us = std::max(ra * ua + (rb - free_last) * ub,
                      (ra - (rest > 0)) * ua + (rounds + rb) * ub);
      }
      us += t.tile_us + extra_us;
      if (us < best) {
        best = us;
        pick[0] = s0;
        pick[1] = s1;
        *skip = rounds;
      }
    }
  }
  for (int i = 0; i < count; i++) {
    q[i].kb_split = len(q[i], pick[i]);
    q[i].splits = (q[i].kblocks + q[i].kb_split - 1) / q[i].kb_split;
    q[i].units = q[i].mtiles * q[i].ntiles * q[i].splits;
  }
  return best;
}

// One or both of a piece's gradient products in one launch: A = P; B of the
// first product, C of the second.
void products(eb_engine* e, const Operand& A, Operand B, Operand C, GemmParams P, int count) {
  Tile tile = PAIR;
  double least = 1e300;
  Prob chosen[2] = {};
  for (Tile t : {PAIR, SINGLE, NARROW}) {
    if (t == SINGLE && (P.q[0].M > BM || (count == 2 && P.q[1].M > BM))) continue;
    const TileCost c = tile_cost(t, A.terms > 1 ? 2 : 1);
    Prob q[2] = {P.q[0], P.q[1]};
    for (int i = 0; i < count; i++) {
      const Prob m = make_prob(q[i].M, q[i].N, q[i].K, c);
      q[i].mtiles = m.mtiles, q[i].ntiles = m.ntiles, q[i].bn = m.bn, q[i].group = m.group;
    }
    int skip = 0;
    const double us = choose_splits(q, count, e->num_sms / c.ctas, c, &skip);
    if (us < least) {
      least = us;
      P.skip = skip;
      tile = t;
      chosen[0] = q[0];
      chosen[1] = q[1];
    }
  }
  for (int i = 0; i < count; i++) P.q[i] = chosen[i];
  if (count == 2 && P.q[1].kb_split > P.q[0].kb_split) {
    std::swap(P.q[0], P.q[1]);
    std::swap(B, C);
  }
  const Prob whole[2] = {P.q[0], P.q[1]};
  size_t room = 0, at[2] = {0, 0};
  for (int i = 0; i < count; i++) {
    at[i] = room;
    if (P.q[i].splits > 1) room += (size_t)(P.q[i].splits * P.q[i].M * P.q[i].ldacc);
  }
  float* part = room ? e->scratch_get<float>("ce_splits", room) : nullptr;
  for (int i = 0; i < count; i++) {
    if (P.q[i].splits == 1) continue;
    P.q[i].accum = part + at[i];
    P.q[i].read_acc = 0;
    P.q[i].write_acc = 1;
  }
  gemm<OUT>(e, A, B, count == 2 ? C : B, tile, P);
  for (int i = 0; i < count; i++) {
    if (P.q[i].splits == 1) continue;
    const long groups = whole[i].M * whole[i].ldacc / 4;
    const int slices = P.q[i].splits >= 16 && groups < 64l * e->num_sms ? 16 : 1;
    const unsigned grid = (unsigned)std::min<long>((groups * slices + 255) / 256, (long)e->num_sms * 8);
    launch_pdl(e, k_ce_reduce, dim3(grid), dim3(256), 0, (const float*)(part + at[i]),
               P.q[i].splits, slices, whole[i]);
    e->stats.kernel_launches++;
  }
}

// Losses and lse of n rows from their parts.
void join(eb_engine* e, const float2* part, int parts, long n, long k, const float* zt,
          const uint32_t* targets, float* loss, float* lse) {
  const bool few = parts <= 32, row = !few && n <= 1024;
  launch_pdl(e, few ? k_ce_join_few : row ? k_ce_join_row : k_ce_join,
             dim3((unsigned)(few ? (n + 127) / 128 : row ? n : (n + 31) / 32)),
             dim3(few ? 128 : row ? 256 : 1024), 0, part, parts, n, k, zt, targets, loss, lse,
             e->d_status);
  e->stats.kernel_launches++;
}

}  // namespace

void linear_ce(eb_engine* e, const LinearCeArgs& a, float* loss, float* lse) {
  if (a.n == 0) return;
  if (linear_ce_is_small(a)) return linear_ce_small(e, a, loss, lse);
  if (linear_ce_is_few(a)) {
    const int parts = linear_ce_few_parts(e, a);
    float2* part = e->scratch_get<float2>("ce_part", (size_t)parts * a.n);
    float* zt = e->scratch_get<float>("ce_zt", a.n);
    linear_ce_few(e, a, part, zt);
    return join(e, part, parts, (long)a.n, (long)a.k, zt, a.targets, loss, lse);
  }
  uint32_t* scal = e->scratch_get<uint32_t>("ce_scalars", S_WORDS);
  uint32_t* found = a.dtype == EB_F32 ? found_words(e, a) : nullptr;
  Operand X, W;
  operands(e, a, found, scal, X, W);
  // Rows a pass: all, or a multiple of 256 that keeps the half tiles' (max, sum) to 256
  // MB (or 256 where those are more); all passes in tiles of one width.
  const int terms = a.dtype == EB_F32 ? 2 : 1;
  constexpr size_t ROOM = ((size_t)256 << 20) / sizeof(float2);
  size_t rows = a.n;
  Tile tile;
  Prob whole;
  while (true) {
    tile = score_tile(e, (long)rows, (long)a.k, (long)a.d, terms);
    const TileCost cost = tile_cost(tile, terms);
    whole = make_prob((long)rows, (long)a.k, (long)a.d, cost, e->num_sms / cost.ctas);
    const size_t most = ROOM / (2 * (size_t)whole.ntiles);
    if (rows <= std::max<size_t>(most, 256)) break;
    rows = std::max<size_t>(std::min(most, rows - 1) / 256 * 256, 256);
  }
  const TileCost cost = tile_cost(tile, terms);
  for (size_t r0 = 0; r0 < a.n; r0 += rows) {
    const long n = (long)std::min(a.n - r0, rows);
    GemmParams P = base_params(a, found, scal);
    P.q[0] = make_prob(n, (long)a.k, (long)a.d, cost, e->num_sms / cost.ctas);
    P.q[0].bn = whole.bn;
    P.q[0].ntiles = whole.ntiles;
    P.q[0].units = P.q[0].mtiles * whole.ntiles;
    const int parts = 2 * whole.ntiles;
    float2* part = e->scratch_get<float2>("ce_part", (size_t)parts * n);
    P.part = part;
    P.zt = e->scratch_get<float>("ce_zt", (size_t)n);
    P.targets = a.targets + r0;
    gemm<LSE>(e, rows_of(X, (long)r0, (long)r0 + n), W, W, tile, P);
    e->ce_found_raised = false;
    join(e, part, parts, n, (long)a.k, P.zt, P.targets, loss + r0, lse + r0);
  }
}

void linear_ce_backward(eb_engine* e, const LinearCeArgs& a, const LinearCeGrads& g) {
  if (!g.dx && !g.dw) return;
  if (a.n == 0) {
    if (g.dw)
      EB_CUDA(cudaMemset2DAsync(g.dw, g.lddw * dtype_bytes(g.dwtype), 0,
                                a.d * dtype_bytes(g.dwtype), a.k, e->stream));
    return;
  }
  if (linear_ce_is_small(a)) return linear_ce_small_backward(e, a, g);
  if (linear_ce_is_few(a)) return linear_ce_few_backward(e, a, g);
  uint32_t* scal = e->scratch_get<uint32_t>("ce_scalars", S_WORDS);
  uint32_t* found = a.dtype == EB_F32 ? found_words(e, a) : nullptr;
  if (!g.one_dloss) {
    uint32_t *most = scal + S_G, *least = nullptr;
    if (found) {
      e->ce_found_raised = true;
      most = found + R_G;
      least = found + R_G_LOW;
    } else {
      EB_CUDA(cudaMemsetAsync(most, 0, 4, e->stream));
    }
    const unsigned grid = (unsigned)std::min<size_t>((a.n + 255) / 256, (size_t)e->num_sms);
    launch_pdl(e, k_ce_gmax, dim3(grid), dim3(256), 0, g.dloss, a.targets, (long)a.n, (long)a.k,
               most, least);
    e->stats.kernel_launches++;
  }
  Operand X, W;
  operands(e, a, found, scal, X, W, !g.one_dloss);
  // Pieces of P, as many elements as the scratch holds: the shorter side of
  // P whole where at least 2,048 of the longer then fit (the sums that run
  // over pieces are the shorter side's gradient), else pieces of both sides.
  const int parts = a.dtype == EB_F32 ? 2 : 1;
  const bool fine = (g.dx && g.dxtype == EB_F32) || (g.dw && g.dwtype == EB_F32);
  const int terms = a.dtype == EB_F32 ? 3 : !fine ? 1 : a.dtype == EB_BF16 ? 3 : 2;
  const size_t room = ((size_t)512 << 20) / 2 / terms;  // elements of P
  const size_t npad = (a.n + 255) / 256 * 256, kpad = (a.k + 255) / 256 * 256;
  const size_t side = std::min(std::min(npad, kpad), room / 2048 / 256 * 256);
  const size_t other = std::max<size_t>(room / side / 256 * 256, 256);
  const size_t rows = std::min(npad, npad <= kpad ? side : other);
  const size_t cols = std::min(kpad, npad <= kpad ? other : side);
  uint16_t* p = e->scratch_get<uint16_t>("ce_p", rows * cols * terms);
  const bool many_cols = cols < a.k, many_rows = rows < a.n;
  const long ldacc = ((long)a.d + 3) / 4 * 4;
  float* dxacc = g.dx && many_cols ? e->scratch_get<float>("ce_dx", std::min(rows, a.n) * ldacc) : nullptr;
  float* dwacc = g.dw && many_rows ? e->scratch_get<float>("ce_dw", a.k * ldacc) : nullptr;
  auto vec = [](int type, size_t ld) { return ld * dtype_bytes(type) % 16 == 0; };
  for (size_t r0 = 0; r0 < a.n; r0 += rows) {
    const size_t r1 = std::min(a.n, r0 + rows);
    const Operand Xr = rows_of(X, (long)r0, (long)r1);
    for (size_t v0 = 0; v0 < a.k; v0 += cols) {
      const size_t v1 = std::min(a.k, v0 + cols);
      const Operand Wv = rows_of(W, (long)v0, (long)v1);
      const long pr = (long)(r1 - r0), pc = (long)(v1 - v0);
      GemmParams P = base_params(a, found, scal);
      const Tile tile = score_tile(e, pr, pc, (long)a.d, parts);
      const TileCost cost = tile_cost(tile, parts);
      P.q[0] = make_prob(pr, pc, (long)a.d, cost, e->num_sms / cost.ctas);
      P.targets = a.targets + r0;
      P.lse = g.lse + r0;
      P.dloss = g.one_dloss ? g.dloss : g.dloss + r0;
      P.one_dloss = g.one_dloss;
      P.col0 = (long)v0;
      P.p_terms = terms;
      const Operand Pm{p, (long)(rows * cols), terms, pr, pc, (pc + 7) / 8 * 8};
      gemm<PROB>(e, Xr, Wv, Pm, tile, P);
      e->ce_found_raised = false;
      int count = 0;
      Operand B[2];
      if (g.dx) {
        Prob& q = P.q[count];
        q = make_prob(pr, (long)a.d, pc, cost);
        q.unscale = S_W;
        q.out = static_cast<char*>(g.dx) + r0 * g.lddx * dtype_bytes(g.dxtype);
        q.otype = g.dxtype;
        q.ldo = (long)g.lddx;
        q.ovec = vec(g.dxtype, g.lddx);
        q.accum = dxacc;
        q.ldacc = ldacc;
        q.read_acc = v0 > 0;
        q.write_acc = v1 < a.k;
        B[count++] = Wv;
      }
      if (g.dw) {
        Prob& q = P.q[count];
        q = make_prob(pc, (long)a.d, pr, cost);
        q.a_mn = 1;
        q.unscale = S_X;
        q.out = static_cast<char*>(g.dw) + v0 * g.lddw * dtype_bytes(g.dwtype);
        q.otype = g.dwtype;
        q.ldo = (long)g.lddw;
        q.ovec = vec(g.dwtype, g.lddw);
        q.accum = dwacc ? dwacc + v0 * ldacc : nullptr;
        q.ldacc = ldacc;
        q.read_acc = r0 > 0;
        q.write_acc = r1 < a.n;
        B[count++] = Xr;
      }
      products(e, Pm, B[0], B[1], P, count);
    }
  }
}

}  // namespace eb
