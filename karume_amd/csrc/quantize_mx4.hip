// Rows of floats to blocks of 32 e2m1 codes with a power of two each, and back (no counterpart in the
// reference, whose 4-bit weights are integers with a float scale a group:
// packages/runtime/src/format/i4.ts:63-118).
#include "mx4.h"
#include "rows8.h"

using namespace krm;

namespace {

constexpr int kThreads = 256;

// A thread has eight elements, four threads a block (they exchange its largest magnitude in registers): whole pieces of 16
// bytes in, a word of codes out.  Bound by bytes, 2 or 4 in and 17/32 out an element: 4099 rows of 11008 that come from
// memory, f32 38.8 us, 5.3 TB/s, fp16 23.1, 4.9 (a copy of them 5.6); from the last-level cache 29.6 and 18.1; f32 rows behind a
// kernel whose 180 MB of results are still on their way to memory 47.5.  (Two or four rows a thread: within 3 %, and few
// rows slower.)  16 rows of 4096 a launch.
template <typename XT>
__global__ __launch_bounds__(kThreads) void quantize_mx4_kernel(const XT* __restrict__ x,
                                                                uint32_t* __restrict__ codes,
                                                                uint8_t* __restrict__ scales,
                                                                uint32_t rows, uint32_t eighths,
                                                                uint64_t x_stride, bool ceil) {
  const uint32_t at = blockIdx.x * kThreads + threadIdx.x;
  if (at >= eighths) return;  // (eighths is a multiple of four: a block's threads leave together)
  for (uint32_t row = blockIdx.y; row < rows; row += gridDim.y) {
    uint32_t byte;
    const uint32_t packed = mx4_quantise8(mx4_load8(x + row * x_stride + (size_t)at * 8), ceil, byte);
    codes[(size_t)row * eighths + at] = packed;
    if ((at & 3u) == 0) scales[(size_t)row * (eighths / 4) + at / 4] = (uint8_t)byte;
  }
}

// f32 value of a code: exact, except that 2^126 and more times the largest codes is infinite.
__device__ inline float mx4_value(uint32_t code, uint32_t byte) {
  const uint32_t size = code & 7u;
  float v = size < 2u ? 0.5f * size : __uint_as_float((126u + (size >> 1)) << 23 | (size & 1u) << 22);
  v *= mx4_scale(byte);
  if (byte == 255u) v = NAN;
  return code & 8u ? -v : v;
}

// Bound by what it writes: the same rows back as f32 48.6 us, 4.2 TB/s, as fp16 30.4, 3.8; as f32 behind each
// quantisation 33.6, where the next quantisation is what waits for the results' way to memory.
template <typename OT>
__global__ __launch_bounds__(kThreads) void dequant_mx4_kernel(const uint32_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales,
                                                               OT* __restrict__ out, uint64_t eighths) {
  const uint64_t stride = (uint64_t)gridDim.x * kThreads;
  for (uint64_t at = (uint64_t)blockIdx.x * kThreads + threadIdx.x; at < eighths; at += stride) {
    const uint32_t word = codes[at], byte = scales[at / 4];
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mx4_value(word >> (4 * i) & 15u, byte);
    store8(out + at * 8, v);
  }
}

}  // namespace

int32_t krm::check_mx4_rows(krm_ctx* ctx, const char* what, krm_buf x, uint32_t dim, uint64_t x_stride, int32_t x_dtype,
                            int32_t scale_rule) {
  KRM_REQUIRE(ctx, valid_dtype(x_dtype), "%s: unknown dtype %d", what, x_dtype);
  KRM_REQUIRE(ctx, scale_rule == KRM_MX4_FLOOR || scale_rule == KRM_MX4_CEIL, "%s: unknown scale rule %d", what, scale_rule);
  KRM_REQUIRE(ctx, dim > 0 && dim % kMx4Block == 0, "%s: dim must be a positive multiple of 32 (%u)", what, dim);
  KRM_REQUIRE(ctx, x_stride >= dim && x_stride <= (1ull << 40) && x_stride * dtype_bytes(x_dtype) % 16 == 0,
              "%s: x_stride %llu must be at least dim (%u) and keep rows 16-byte aligned", what,
              (unsigned long long)x_stride, dim);
  KRM_REQUIRE(ctx, aligned(x, 16), "%s: x needs 16-byte alignment", what);
  return KRM_OK;
}

extern "C" int32_t krm_quantize_mx4(krm_ctx* ctx, krm_buf x, krm_buf codes, krm_buf scales,
                                    uint32_t rows, uint32_t dim, uint64_t x_stride, int32_t x_dtype,
                                    int32_t scale_rule) {
  KRM_TRY(enter(ctx));
  KRM_TRY(check_mx4_rows(ctx, "quantize mx4", x, dim, x_stride, x_dtype, scale_rule));
  KRM_REQUIRE(ctx, rows <= 0x7fffffffu, "quantize mx4: %u rows", rows);  // (a row's number and the step to the next fit 32 bits)
  if (rows == 0) return KRM_OK;
  KRM_REQUIRE(ctx, x && codes && scales, "quantize mx4: null buffer");
  KRM_REQUIRE(ctx, aligned(codes, 16), "quantize mx4: codes need 16-byte alignment");
  KRM_REQUIRE(ctx, x != codes && x != scales && codes != scales, "quantize mx4: two of x, codes and scales are one buffer");
  const uint32_t eighths = dim / 8;
  const dim3 grid((eighths + kThreads - 1) / kThreads, rows < 65535u ? rows : 65535u);
  const bool ceil = scale_rule == KRM_MX4_CEIL;
  if (x_dtype == KRM_F16)
    quantize_mx4_kernel<<<grid, kThreads, 0, ctx->stream>>>(krm::ptr<const __half>(x), krm::ptr<uint32_t>(codes),
                                                            krm::ptr<uint8_t>(scales), rows, eighths, x_stride, ceil);
  else
    quantize_mx4_kernel<<<grid, kThreads, 0, ctx->stream>>>(krm::ptr<const float>(x), krm::ptr<uint32_t>(codes),
                                                            krm::ptr<uint8_t>(scales), rows, eighths, x_stride, ceil);
  return launched(ctx, "quantize_mx4_kernel");
}

extern "C" int32_t krm_dequant_mx4(krm_ctx* ctx, krm_buf codes, krm_buf scales, krm_buf out,
                                   uint32_t rows, uint32_t dim, int32_t out_dtype) {
  KRM_TRY(enter(ctx));
  KRM_REQUIRE(ctx, valid_dtype(out_dtype), "dequant mx4: unknown dtype %d", out_dtype);
  KRM_REQUIRE(ctx, dim > 0 && dim % kMx4Block == 0,
              "dequant mx4: dim must be a positive multiple of 32 (%u)", dim);
  KRM_REQUIRE(ctx, rows <= 0x7fffffffu, "dequant mx4: %u rows", rows);
  if (rows == 0) return KRM_OK;
  KRM_REQUIRE(ctx, codes && scales && out, "dequant mx4: null buffer");
  KRM_REQUIRE(ctx, aligned(codes, 16) && aligned(out, 16),
              "dequant mx4: codes and out need 16-byte alignment");
  KRM_REQUIRE(ctx, out != codes && out != scales, "dequant mx4: out is the codes' or the scales' buffer");
  const uint64_t eighths = (uint64_t)rows * (dim / 8);
  const uint64_t blocks = (eighths + kThreads - 1) / kThreads;
  const dim3 grid((uint32_t)(blocks < 65536 ? blocks : 65536));
  if (out_dtype == KRM_F16)
    dequant_mx4_kernel<<<grid, kThreads, 0, ctx->stream>>>(krm::ptr<const uint32_t>(codes),
                                                           krm::ptr<const uint8_t>(scales), krm::ptr<__half>(out), eighths);
  else
    dequant_mx4_kernel<<<grid, kThreads, 0, ctx->stream>>>(krm::ptr<const uint32_t>(codes),
                                                           krm::ptr<const uint8_t>(scales), krm::ptr<float>(out), eighths);
  return launched(ctx, "dequant_mx4_kernel");
}
