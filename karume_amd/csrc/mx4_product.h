// What the kernels of products of mx4 rows share: one step of the matrix cores and the way out of a sum.
#pragma once

#include "mx4.h"

#include <initializer_list>
#include <type_traits>

namespace krm {
namespace {

__device__ inline uint32_t least(uint32_t a, uint32_t b) { return a < b ? a : b; }

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
  uint32_t pack;         // bytes of a lane's neighbouring results that are stored at once: 16, 8, or one result's
};

// silu(g) * up, g times its logistic 1 / (1 + e^-g), on the exponential and reciprocal of the hardware, off by a step each.
// fp16 results: as written; 1 + e^-g is infinite or its reciprocal flushed from g = -87.4 down, where silu is zero then
// (2^-119: an fp16 result would need an up past 2^94).  The exponent's rounding makes the exponential off by |g| 2^-23, 2^-18
// where a result of such an up as models have is not zero, which moves one rounding in a hundred.
// f32 results, with e^-|g| = h h1, neither of which ends before |g| = 174: h = 2^y with y about half of the exponent, h1 = h with
// what y's roundings have lost.  1 / (1 + h h1) is silu over g, times h h1 where g < 0: h1 before up and h behind
// it, so that no product is infinite or subnormal before the result is.  Seven steps at most (2.8 seen in 200000
// gates), and two roundings of a subnormal result; gates past 174 are -0 or themselves.  (From 1000 on the gate is held there, so that nothing is infinite
// but g itself; it comes in again as a factor, as does NaN.)
template <typename OT>
__device__ inline float mx4_silu_times(float g, float up) {
  if constexpr (sizeof(OT) == 2) {
    constexpr float kLog2e = 1.44269502f;
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-g * kLog2e)) * up;
  } else {
    constexpr float kHalfLog2e = 0.721347511f, kLn4 = 1.38629436f, kLn4Low = -3.80930843e-9f;
    const float size = fabsf(__builtin_amdgcn_fmed3f(g, -1000.f, 1000.f));
    const float y = -kHalfLog2e * size;
    const float h = __builtin_amdgcn_exp2f(y);
    const float lost = fmaf(y, -kLn4Low, fmaf(y, -kLn4, -size));  // -size - 2 y ln 2
    const float h1 = fmaf(h, lost, h), r = __builtin_amdgcn_rcpf(fmaf(h, h1, 1.0f));
    const bool below = g < 0.f;
    return g * (below ? h1 : 1.0f) * r * up * (below ? h : 1.0f);
  }
}
__device__ inline float mx4_load(const float* p) { return *p; }
__device__ inline float mx4_load(const __half* p) { return __half2float(*p); }
__device__ inline void mx4_store(float* p, float v) { *p = v; }
__device__ inline void mx4_store(__half* p, float v) { *p = __float2half_rn(v); }

// Neighbouring sums from column col on (a multiple of as many), with bias, and as silu(gate) * up where the columns are such
// pairs.
template <typename OT, bool PAIRS, int PIECES>
__device__ inline void mx4_values(const Mx4Out& o, uint32_t col, const v4f* sum, float (&v)[4 * PIECES]) {
#pragma unroll
  for (int i = 0; i < 4 * PIECES; ++i) v[i] = sum[i / 4][i % 4];
  if (o.bias) {
#pragma unroll
    for (int i = 0; i < 4 * PIECES; ++i) v[i] += o.bias[least(col + i, o.n - 1)];
  }
  if constexpr (PAIRS) {
#pragma unroll
    for (int i = 0; i < 2 * PIECES; ++i) v[i] = mx4_silu_times<OT>(v[2 * i], v[2 * i + 1]);
  }
}
// COUNT neighbouring values of row `row` from column `first` of the result on: residual, one rounding to the stored type.
// STREAM: past the caches.
template <typename OT, int COUNT, bool STREAM>
__device__ inline void mx4_put(const Mx4Out& o, uint32_t row, uint32_t first, uint32_t width, float* v) {
  const size_t at = (size_t)row * width + first;
  OT* out = static_cast<OT*>(o.out) + at;
  const OT* residual = static_cast<const OT*>(o.residual) + at;
  // packs of a row end where the row does (its bytes are a multiple of a pack's, and so is its address)
  auto store = [&](auto bytes) {
    constexpr int kPack = decltype(bytes)::value / (int)sizeof(OT) < COUNT ? decltype(bytes)::value / (int)sizeof(OT) : COUNT;
    struct alignas(kPack * sizeof(OT)) Pack { OT e[kPack]; };
#pragma unroll
    for (int p = 0; p < COUNT / kPack; ++p) {
      if (first + p * kPack >= width) break;
      Pack pack;
      if (o.residual) {
        pack = reinterpret_cast<const Pack*>(residual)[p];
#pragma unroll
        for (int i = 0; i < kPack; ++i) v[p * kPack + i] += mx4_load(&pack.e[i]);
      }
#pragma unroll
      for (int i = 0; i < kPack; ++i) mx4_store(&pack.e[i], v[p * kPack + i]);
      Pack* const to = reinterpret_cast<Pack*>(out) + p;
      if constexpr (STREAM && sizeof(Pack) == 16) __builtin_nontemporal_store(__builtin_bit_cast(v4i, pack), reinterpret_cast<v4i*>(to));
      else *to = pack;
    }
  };
  if (o.pack == 16u) store(std::integral_constant<int, 16>());
  else if (o.pack == 8u) store(std::integral_constant<int, 8>());
  else store(std::integral_constant<int, (int)sizeof(OT)>());
}
// Four neighbouring sums of row `row` from column col on.
template <typename OT, bool PAIRS>
__device__ inline void mx4_finish(const Mx4Out& o, uint32_t row, uint32_t col, const v4f& sum) {
  if (row >= o.m || col >= o.n) return;
  float v[4];
  mx4_values<OT, PAIRS, 1>(o, col, &sum, v);
  mx4_put<OT, PAIRS ? 2 : 4, false>(o, row, PAIRS ? col / 2 : col, PAIRS ? o.n / 2 : o.n, v);
}
// Bytes that rows of `width` results, `count` neighbours a lane, can be stored in at once.
inline uint32_t mx4_pack(uint32_t width, uint32_t count, krm_buf out, krm_buf residual, size_t eb) {
  for (size_t pack : {(size_t)16, (size_t)8}) {
    const size_t mine = pack < count * eb ? pack : count * eb;
    if ((uint64_t)width * eb % mine == 0 && aligned(out | residual, mine)) return (uint32_t)pack;
  }
  return (uint32_t)eb;
}

}  // namespace
}  // namespace krm
