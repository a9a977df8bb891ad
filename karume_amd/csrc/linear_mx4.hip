// `linear` over rows of x and w that are blocks of 32 e2m1 codes with a power of two each (the reference's linear
// has integer weights: packages/runtime/src/kernels/gemm.ts:115,315-327; this is the same op over the format that
// gfx950's matrix cores multiply as it is stored):
//
//   out[m, n] = epilogue(sum over blocks b of 2^(xs + ws - 254) * (sum over the block of xe * we) + bias[n]) + residual
#include "mx4_product.h"

using namespace krm;

namespace {

// A workgroup has 16 rows of w and 16 of x; its waves take the steps of 128 codes in turn and join their sums.
template <typename OT, bool PAIRS, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void linear_mx4_rows_kernel(
    const uint8_t* __restrict__ xq, const uint8_t* __restrict__ xs, const uint8_t* __restrict__ w,
    const uint8_t* __restrict__ ws, uint32_t blocks, Mx4Out o) {
  __shared__ v4f s_sum[WAVES][64];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kb = lane >> 4;
  const uint32_t col0 = blockIdx.x * 16, steps = (blocks + 3) / 4;
  const size_t w_row = (size_t)min(col0 + r, o.n - 1) * blocks;
  for (uint32_t row0 = blockIdx.y * 16; row0 < o.m; row0 += gridDim.y * 16) {
    const size_t x_row = (size_t)min(row0 + r, o.m - 1) * blocks;
    v4f sum = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t step = wave; step < steps; step += WAVES) {
      const uint32_t block = step * 4 + kb;
      const bool there = block < blocks;  // past the end of K: codes and scales of nothing
      const size_t wb = w_row + (there ? block : 0u), xb = x_row + (there ? block : 0u);
      const v4i wc = *reinterpret_cast<const v4i*>(w + wb * 16);
      v4i xc = *reinterpret_cast<const v4i*>(xq + xb * 16);
      uint32_t w_scale = ws[wb], x_scale = xs[xb];
      if (!there) {
        xc = v4i{0, 0, 0, 0};
        w_scale = x_scale = 127u;
      }
      sum = mx4_step(wc, w_scale, xc, x_scale, sum);
    }
    s_sum[wave][lane] = sum;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int i = 1; i < WAVES; ++i) sum += s_sum[i][lane];
      mx4_finish<OT, PAIRS>(o, row0 + r, col0 + 4 * kb, sum);
    }
    __syncthreads();
  }
}

int32_t check_product(krm_ctx* ctx, krm_buf w, krm_buf w_scales, krm_buf bias, krm_buf residual, krm_buf out,
                      uint32_t n, uint32_t k, int32_t out_dtype, int32_t epilogue) {
  KRM_REQUIRE(ctx, valid_dtype(out_dtype), "linear mx4: unknown dtype %d", out_dtype);
  KRM_REQUIRE(ctx, epilogue == KRM_EPILOGUE_NONE || epilogue == KRM_EPILOGUE_SILU_PAIRS,
              "linear mx4: unknown epilogue %d", epilogue);
  KRM_REQUIRE(ctx, epilogue == KRM_EPILOGUE_NONE || n % 2 == 0, "linear mx4: pairs need an even n (%u)", n);
  KRM_REQUIRE(ctx, k > 0 && k % kMx4Block == 0, "linear mx4: k must be a positive multiple of 32 (%u)", k);
  const size_t eb = dtype_bytes(out_dtype);
  KRM_REQUIRE(ctx, aligned(w, 16) && aligned(out, eb) && aligned(residual, eb) && aligned(bias, 4),
              "linear mx4: misaligned buffer (codes need 16 bytes)");
  return KRM_OK;
}

int32_t launch_product(krm_ctx* ctx, krm_buf xq, krm_buf xs, krm_buf w, krm_buf w_scales, krm_buf bias,
                       krm_buf residual, krm_buf out, uint32_t m, uint32_t n, uint32_t k, int32_t out_dtype,
                       int32_t epilogue) {
  const bool pairs = epilogue == KRM_EPILOGUE_SILU_PAIRS;
  const uint32_t width = pairs ? n / 2 : n, count = pairs ? 2 : 4;
  Mx4Out o{ptr<const float>(bias), ptr<const void>(residual), ptr<void>(out), m, n, false};
  o.wide = width % count == 0 && aligned(out | residual, count * dtype_bytes(out_dtype));
  const dim3 grid((n + 15) / 16, min((m + 15) / 16, 65535u));
  auto launch = [&](auto kernel) {
    kernel<<<grid, 256, 0, ctx->stream>>>(ptr<const uint8_t>(xq), ptr<const uint8_t>(xs), ptr<const uint8_t>(w),
                                          ptr<const uint8_t>(w_scales), k / kMx4Block, o);
  };
  if (out_dtype == KRM_F16) {
    if (pairs) launch(linear_mx4_rows_kernel<__half, true, 4>); else launch(linear_mx4_rows_kernel<__half, false, 4>);
  } else {
    if (pairs) launch(linear_mx4_rows_kernel<float, true, 4>); else launch(linear_mx4_rows_kernel<float, false, 4>);
  }
  return launched(ctx, "linear_mx4_rows_kernel");
}

}  // namespace

extern "C" int32_t krm_linear_mx4(krm_ctx* ctx, krm_buf xq, krm_buf xs, krm_buf w, krm_buf w_scales, krm_buf bias,
                                  krm_buf residual, krm_buf out, uint32_t m, uint32_t n, uint32_t k,
                                  int32_t out_dtype, int32_t epilogue) {
  KRM_TRY(enter(ctx));
  KRM_TRY(check_product(ctx, w, w_scales, bias, residual, out, n, k, out_dtype, epilogue));
  KRM_REQUIRE(ctx, aligned(xq, 16), "linear mx4: misaligned buffer (codes need 16 bytes)");
  if (m == 0 || n == 0) return KRM_OK;
  KRM_REQUIRE(ctx, xq && xs && w && w_scales && out, "linear mx4: null buffer");
  return launch_product(ctx, xq, xs, w, w_scales, bias, residual, out, m, n, k, out_dtype, epilogue);
}

extern "C" int32_t krm_linear_mx4_fused(krm_ctx* ctx, krm_buf x, krm_buf xq, krm_buf xs, krm_buf w,
                                        krm_buf w_scales, krm_buf bias, krm_buf residual, krm_buf out, uint32_t m,
                                        uint32_t n, uint32_t k, uint64_t x_stride, int32_t x_dtype,
                                        int32_t out_dtype, int32_t scale_rule, int32_t epilogue) {
  KRM_TRY(enter(ctx));
  KRM_TRY(check_product(ctx, w, w_scales, bias, residual, out, n, k, out_dtype, epilogue));
  if (m == 0 || n == 0) return KRM_OK;
  KRM_REQUIRE(ctx, x && w && w_scales && out, "linear mx4: null buffer");
  KRM_REQUIRE(ctx, xq && xs, "linear mx4 (fused): this shape (m=%u, k=%u) takes two launches and needs the xq and xs "
              "work buffers", m, k);
  KRM_REQUIRE(ctx, aligned(xq, 16), "linear mx4: misaligned buffer (codes need 16 bytes)");
  KRM_TRY(krm_quantize_mx4(ctx, x, xq, xs, m, k, x_stride, x_dtype, scale_rule));
  return launch_product(ctx, xq, xs, w, w_scales, bias, residual, out, m, n, k, out_dtype, epilogue);
}
