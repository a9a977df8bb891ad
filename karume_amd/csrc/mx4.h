// Blocks of 32 e2m1 numbers that share a power of two (microscaled 4-bit floating point).
//
// A code is sign, two bits of exponent, one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives; a
// row's element 2j is the low nibble of its byte j.  Scale byte E stands for 2^(E - 127), 255 for NaN.  What
// the matrix cores read is the same: a lane's 16 bytes of codes and one scale byte are one block.
#pragma once

#include "krm_internal.h"

namespace krm {

constexpr uint32_t kMx4Block = 32;

// What rows of floats to be quantised have to be, for every entry point that takes them.
int32_t check_mx4_rows(krm_ctx* ctx, const char* what, krm_buf x, uint32_t dim, uint64_t x_stride, int32_t x_dtype,
                       int32_t scale_rule);

#if defined(__HIPCC__)
namespace {

// Largest magnitude of four neighbouring lanes; as bits, so that an infinity or a NaN is larger than any number.
__device__ inline uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));  // lane ^ 1
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));  // lane ^ 2
}

// Scale byte of a block whose largest magnitude has the f32 bits `top`: its exponent less 2, so that it comes to
// stand in [4, 8) (and above 6 is clipped), or one more where it would be clipped (`ceil`).  Subnormal maxima and
// those below 2^-125 meet the lowest scale.
__device__ inline uint32_t mx4_scale_byte(uint32_t top, bool ceil) {
  if (top >= 0x7f800000u) return 255u;
  const int32_t byte = (int32_t)(top >> 23) - 2 + (ceil && (top & 0x7fffffu) > 0x400000u ? 1 : 0);
  return (uint32_t)max(byte, 0);
}

// f32 bits of 2^(byte - 127); 2^-127 is a subnormal.  255 (whose codes are 0) gives a number like any other.
__device__ inline float mx4_scale(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : (byte == 255u ? 127u : byte) << 23);
}

// Eight codes: x / scale rounded half to even, clipped at 6; a negative that rounds to zero is -0.
__device__ inline uint32_t mx4_codes(const float (&v)[8], float scale) {
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0], v[1], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2], v[3], scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4], v[5], scale, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6], v[7], scale, 3);
  return codes;
}

// Eight neighbouring elements of a row (16-byte aligned) as they are loaded, in each of four lanes that hold a block ->
// this lane's codes; `byte`: the block's scale, in all four.
struct Mx4F32 {
  float4 low, high;
};
struct Mx4F16 {
  uint4 all;
};
__device__ inline Mx4F32 mx4_load8(const float* p) {
  return {*reinterpret_cast<const float4*>(p), *reinterpret_cast<const float4*>(p + 4)};
}
__device__ inline Mx4F16 mx4_load8(const __half* p) { return {*reinterpret_cast<const uint4*>(p)}; }

__device__ inline uint32_t mx4_quantise8(const Mx4F32& e, bool ceil, uint32_t& byte) {
  const float v[8] = {e.low.x, e.low.y, e.low.z, e.low.w, e.high.x, e.high.y, e.high.z, e.high.w};
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  byte = mx4_scale_byte(quad_max(top), ceil);
  const uint32_t codes = mx4_codes(v, mx4_scale(byte));
  return byte == 255u ? 0u : codes;
}
// (halves compare as their bits do; two at a time)
__device__ inline uint32_t mx4_quantise8(const Mx4F16& e, bool ceil, uint32_t& byte) {
  typedef unsigned short v2u __attribute__((ext_vector_type(2)));
  typedef _Float16 v2h __attribute__((ext_vector_type(2)));
  const uint32_t w[4] = {e.all.x, e.all.y, e.all.z, e.all.w};
  v2u top = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(v2u, w[i] & 0x7fff7fffu));
  const uint16_t bits = (uint16_t)quad_max(max((uint32_t)top[0], (uint32_t)top[1]));
  byte = mx4_scale_byte(__float_as_uint((float)__builtin_bit_cast(_Float16, bits)), ceil);
  const float scale = mx4_scale(byte);
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(v2h, w[0]), scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(v2h, w[1]), scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(v2h, w[2]), scale, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(v2h, w[3]), scale, 3);
  return byte == 255u ? 0u : codes;
}

}  // namespace
#endif
}  // namespace krm
