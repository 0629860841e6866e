// Pieces of a softmax's arithmetic that the linear cross entropy's kernels share.
#pragma once

#include <cuda_runtime.h>

#include <cmath>

namespace eb {

constexpr float LOG2E = 1.4426950408889634f;

// exp of a difference of scores (inputs <= 0 but for rounding; relative error
// 2^-22 and 2^-24 of the input). Differences are formed in natural units,
// where the scores' scale needs no rounding (a power of two apart), and only
// then scaled to base 2.
__device__ __forceinline__ float ex(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * LOG2E));
  return r;
}

// Folds (m', s') into a running (max, sum of exp(z - max)); (-inf, 0) is empty.
// NaN scores are in the sums, not in the maxima.
__device__ __forceinline__ void fold(float& m, float& s, float2 v) {
  const float top = fmaxf(m, v.x), off = top == -INFINITY ? 0.0f : top;
  s = s * ex(m - off) + v.y * ex(v.x - off);
  m = top;
}

}  // namespace eb
