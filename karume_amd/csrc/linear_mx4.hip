// `linear` over rows of x and w that are blocks of 32 e2m1 codes with a power of two each (the reference's linear
// has integer weights: packages/runtime/src/kernels/gemm.ts:115,315-327; this is the same op over the format that
// gfx950's matrix cores multiply as it is stored):
//
//   out[m, n] = epilogue(sum over blocks b of 2^(xs + ws - 254) * (sum over the block of xe * we) + bias[n]) + residual
#include "mx4_tiles.h"

using namespace krm;

namespace {

int32_t check_product(krm_ctx* ctx, krm_buf w, krm_buf w_scales, krm_buf bias, krm_buf residual, krm_buf out,
                      uint32_t m, uint32_t n, uint32_t k, int32_t out_dtype, int32_t epilogue) {
  KRM_REQUIRE(ctx, valid_dtype(out_dtype), "linear mx4: unknown dtype %d", out_dtype);
  KRM_REQUIRE(ctx, epilogue == KRM_EPILOGUE_NONE || epilogue == KRM_EPILOGUE_SILU_PAIRS,
              "linear mx4: unknown epilogue %d", epilogue);
  KRM_REQUIRE(ctx, epilogue == KRM_EPILOGUE_NONE || n % 2 == 0, "linear mx4: pairs need an even n (%u)", n);
  KRM_REQUIRE(ctx, k <= (1u << 24), "linear mx4: k %u is above 2^24", k);
  // (a launch has fewer than 2^32 threads: 256 a tile, of 64 x 128 at least)
  KRM_REQUIRE(ctx, ((m + 63ull) / 64) * ((n + 127ull) / 128) < (1u << 24) - 8u, "linear mx4: %u x %u is too large", m, n);
  KRM_REQUIRE(ctx, k > 0 && k % kMx4Block == 0, "linear mx4: k must be a positive multiple of 32 (%u)", k);
  const size_t eb = dtype_bytes(out_dtype);
  KRM_REQUIRE(ctx, aligned(w, 16) && aligned(out, eb) && aligned(residual, eb) && aligned(bias, 4),
              "linear mx4: misaligned buffer (codes need 16 bytes)");
  return KRM_OK;
}

Mx4Product product_of(krm_buf xq, krm_buf xs, krm_buf w, krm_buf w_scales, krm_buf bias, krm_buf residual, krm_buf out,
                      uint32_t m, uint32_t n, uint32_t k, int32_t out_dtype, bool pairs, uint32_t at_once) {
  Mx4Product p{ptr<const uint8_t>(xq), ptr<const uint8_t>(xs), ptr<const uint8_t>(w), ptr<const uint8_t>(w_scales),
               k / kMx4Block, {ptr<const float>(bias), ptr<const void>(residual), ptr<void>(out), m, n, 0}};
  // (at_once: sums of a lane)
  p.out.pack = mx4_pack(pairs ? n / 2 : n, pairs ? at_once / 2 : at_once, out, residual, dtype_bytes(out_dtype));
  return p;
}

int32_t launch_product(krm_ctx* ctx, krm_buf xq, krm_buf xs, krm_buf w, krm_buf w_scales, krm_buf bias,
                       krm_buf residual, krm_buf out, uint32_t m, uint32_t n, uint32_t k, int32_t out_dtype,
                       int32_t epilogue) {
  const bool pairs = epilogue == KRM_EPILOGUE_SILU_PAIRS, half = out_dtype == KRM_F16;
  // (parts of a tile are joined through the context's scratch, which ops share in launch order)
  const bool serial = ctx->stream == ctx->main_stream;
  const Mx4Form form = mx4_form(m, n, k, ctx->num_cus, serial ? 2 * kGemmPartialBytes * ctx->num_cus : 0,
                                serial ? kTicketSlots : 0);
  const bool tiles = form.kernel == Mx4Kernel::kTiles;
  const Mx4Product p = product_of(xq, xs, w, w_scales, bias, residual, out, m, n, k, out_dtype, pairs, tiles ? 16 : 4);
  if (form.kernel == Mx4Kernel::kRows) return launch_mx4_rows(ctx, p, half, pairs);
  return tiles ? launch_mx4_tiles(ctx, p, half, pairs, form) : launch_mx4_batch(ctx, p, half, pairs);
}

}  // namespace

extern "C" int32_t krm_linear_mx4(krm_ctx* ctx, krm_buf xq, krm_buf xs, krm_buf w, krm_buf w_scales, krm_buf bias,
                                  krm_buf residual, krm_buf out, uint32_t m, uint32_t n, uint32_t k,
                                  int32_t out_dtype, int32_t epilogue) {
  KRM_TRY(enter(ctx));
  KRM_TRY(check_product(ctx, w, w_scales, bias, residual, out, m, n, k, out_dtype, epilogue));
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
  KRM_TRY(check_product(ctx, w, w_scales, bias, residual, out, m, n, k, out_dtype, epilogue));
  if (m == 0 || n == 0) return KRM_OK;
  KRM_REQUIRE(ctx, x && w && w_scales && out, "linear mx4: null buffer");
  if (mx4_rows_fit(m, k)) {
    KRM_TRY(check_mx4_rows(ctx, "linear mx4 (fused)", x, k, x_stride, x_dtype, scale_rule));
    const bool pairs = epilogue == KRM_EPILOGUE_SILU_PAIRS;
    const Mx4Product p = product_of(0, 0, w, w_scales, bias, residual, out, m, n, k, out_dtype, pairs, 4);
    return launch_mx4_rows_of(ctx, p, x, x_stride, x_dtype, scale_rule == KRM_MX4_CEIL, out_dtype == KRM_F16, pairs);
  }
  KRM_REQUIRE(ctx, xq && xs, "linear mx4 (fused): this shape (m=%u, k=%u) takes two launches and needs the xq and xs "
              "work buffers", m, k);
  KRM_REQUIRE(ctx, aligned(xq, 16), "linear mx4: misaligned buffer (codes need 16 bytes)");
  KRM_TRY(krm_quantize_mx4(ctx, x, xq, xs, m, k, x_stride, x_dtype, scale_rule));
  return launch_product(ctx, xq, xs, w, w_scales, bias, residual, out, m, n, k, out_dtype, epilogue);
}
