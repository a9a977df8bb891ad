// What the kernels of products of mx4 rows share: one step of the matrix cores and the way out of a sum.
#pragma once

#include "mx4.h"

namespace krm {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// 128 codes of 16 rows of w times those of 16 rows of x: lane l has the 32 codes (16 bytes) of row l % 16 that block
// l / 16 holds, and their scale in byte SELECT of its word.  Sum (4 (l / 16) + i, l % 16) = (row of w, row of x) is
// element i.  Products are exact, sums f32; scales apply to a block's sum; 255 gives NaN.
template <int WSEL = 0, int XSEL = 0>
__device__ inline v4f mx4_step(v4i w, uint32_t w_scale, v4i x, uint32_t x_scale, v4f sum) {
  const v8i a = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, b = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, sum, 4, 4, WSEL, (int)w_scale, XSEL, (int)x_scale);
}

struct Mx4Out {
  const float* bias;     // [n] or 0
  const void* residual;  // [m, n_out] or 0; may be out
  void* out;             // [m, n_out]
  uint32_t m, n;
  bool wide;             // four (pairs: two) neighbouring results of a row are stored at once
};

__device__ inline float mx4_silu(float g) {
  const float t = expf(-fabsf(g));
  return g * (g < 0.f ? t / (1.0f + t) : 1.0f / (1.0f + t));
}
__device__ inline float mx4_load(const float* p) { return *p; }
__device__ inline float mx4_load(const __half* p) { return __half2float(*p); }
__device__ inline void mx4_store(float* p, float v) { *p = v; }
__device__ inline void mx4_store(__half* p, float v) { *p = __float2half_rn(v); }

// The sums of row `row` and columns col .. col + 3 (col a multiple of 4): bias, silu(gate) * up where the columns are
// such pairs, residual, one rounding to the stored type.
template <typename OT, bool PAIRS>
__device__ inline void mx4_finish(const Mx4Out& o, uint32_t row, uint32_t col, v4f sum) {
  if (row >= o.m || col >= o.n) return;
  constexpr int kCount = PAIRS ? 2 : 4;
  if (o.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += o.bias[min(col + i, o.n - 1)];
  }
  float v[kCount];
  if constexpr (PAIRS) {
    v[0] = mx4_silu(sum[0]) * sum[1];
    v[1] = mx4_silu(sum[2]) * sum[3];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = sum[i];
  }
  const uint32_t width = PAIRS ? o.n / 2 : o.n, first = PAIRS ? col / 2 : col;
  const size_t at = (size_t)row * width + first;
  OT* out = static_cast<OT*>(o.out) + at;
  const OT* residual = static_cast<const OT*>(o.residual) + at;
  if (o.wide) {  // (the width is a multiple of kCount)
    struct alignas(kCount * sizeof(OT)) Pack { OT e[kCount]; } pack;
    if (o.residual) {
      pack = *reinterpret_cast<const Pack*>(residual);
#pragma unroll
      for (int i = 0; i < kCount; ++i) v[i] += mx4_load(&pack.e[i]);
    }
#pragma unroll
    for (int i = 0; i < kCount; ++i) mx4_store(&pack.e[i], v[i]);
    *reinterpret_cast<Pack*>(out) = pack;
    return;
  }
#pragma unroll
  for (int i = 0; i < kCount; ++i)
    if (first + i < width) mx4_store(out + i, o.residual ? v[i] + mx4_load(residual + i) : v[i]);
}

}  // namespace
}  // namespace krm
