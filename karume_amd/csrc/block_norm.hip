// What stands between two blocks of a decoder layer, in one pass over its rows: the norm behind a block, its gate,
// the scaled residual sum and the norm in front of the next block
// (packages/runtime/src/kernels/rms-norm.ts:35-91 twice, packages/runtime/src/codegen/elementwise.ts between).
#include "krm_internal.h"
#include "rows8.h"

#include <cmath>

using namespace krm;

namespace {

struct NormArgs {
  const void* y;
  const float* post;      // 0: y is not normalised
  const void* gate;       // 0: no gate
  const void* residual;   // 0: nothing is added to
  const float* pre;       // 0: the sum alone is wanted
  void* sum_out;          // 0: not wanted
  void* norm_out;
  uint32_t dim, gate_span, first_row;
  float eps, block_scale, residual_scale;
  bool sigmoid;
};

__device__ inline float element(const float* p) { return *p; }
__device__ inline float element(const __half* p) { return __half2float(*p); }
__device__ inline void put(float* p, float v) { *p = v; }
__device__ inline void put(__half* p, float v) { *p = __float2half_rn(v); }

__device__ inline float logistic(float v) {
  const float t = expf(-fabsf(v));
  return v < 0.f ? t / (1.0f + t) : 1.0f / (1.0f + t);
}

// One workgroup a row, eight elements a thread and piece, in registers from the one read to the last store (so that
// sum_out may be residual and norm_out y).  VEC: rows of whole 16-byte pieces.
// Bound by bytes, y and residual in, the sum and the norm out: 8192 rows of 4096 fp16 49.5 us, 5.4 TB/s (as norm, sum
// and norm the sum would be read and written twice more); 1023 gated f32 rows of 5632 20.3 us, 5.1 TB/s; a single row is a
// launch and two joins of a workgroup's sums, 2.4 us.  A row's threads are as few as hold it: a wave for 512 elements.
template <typename XT, typename OT, int THREADS, int PIECES, bool VEC>
__global__ __launch_bounds__(THREADS) void block_norm_kernel(NormArgs a) {
  __shared__ float s_sum[2][THREADS / 64];
  const uint32_t row = a.first_row + blockIdx.x, dim = a.dim;
  const size_t base = (size_t)row * dim;
  auto index = [&](int p, int e) -> uint32_t {
    return VEC ? (p * THREADS + threadIdx.x) * 8 + e : (p * 8 + e) * THREADS + threadIdx.x;
  };
  auto load = [&](const auto* from, float (&v)[PIECES][8]) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      if (VEC) {
        const uint32_t at = index(p, 0);
        load8(from + (at < dim ? at : 0u), v[p]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[p][e] = element(from + min(index(p, e), dim - 1));
      }
    }
  };
  auto rms = [&](const float (&v)[PIECES][8], int slot) {
    float squares = 0.f;
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) squares = index(p, e) < dim ? fmaf(v[p][e], v[p][e], squares) : squares;
    for (int off = 32; off > 0; off >>= 1) squares += __shfl_xor(squares, off, 64);
    if ((threadIdx.x & 63) == 0) s_sum[slot][threadIdx.x >> 6] = squares;
    __syncthreads();
    float total = 0.f;
    for (int w = 0; w < THREADS / 64; ++w) total += s_sum[slot][w];
    return 1.0f / sqrtf(total / (float)dim + a.eps);
  };
  auto store = [&](auto* to, const float (&v)[PIECES][8]) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      if (VEC) {
        const uint32_t at = index(p, 0);
        if (at < dim) store8(to + at, v[p]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (index(p, e) < dim) put(to + index(p, e), v[p][e]);
      }
    }
  };
  float t[PIECES][8], other[PIECES][8];
  load(static_cast<const XT*>(a.y) + base, t);
  if (a.post) {
    load(a.post, other);
    const float inv = rms(t, 0);
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) t[p][e] = t[p][e] * inv * other[p][e];
  }
  if (a.gate) {
    const size_t gate_row = a.gate_span ? row / a.gate_span : 0u;
    load(static_cast<const XT*>(a.gate) + gate_row * dim, other);
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) t[p][e] *= a.sigmoid ? logistic(other[p][e]) : other[p][e];
  }
  if (a.residual) {
    load(static_cast<const XT*>(a.residual) + base, other);
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) t[p][e] = fmaf(a.block_scale, t[p][e], a.residual_scale * other[p][e]);
  } else {
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) t[p][e] *= a.block_scale;
  }
  if (a.sum_out) store(static_cast<XT*>(a.sum_out) + base, t);
  if (!a.pre) return;
  load(a.pre, other);
  const float inv = rms(t, 1);
#pragma unroll
  for (int p = 0; p < PIECES; ++p)
#pragma unroll
    for (int e = 0; e < 8; ++e) t[p][e] = t[p][e] * inv * other[p][e];
  store(static_cast<OT*>(a.norm_out) + base, t);
}

template <typename XT, typename OT, bool VEC>
void launch_norm(krm_ctx* ctx, uint32_t rows, const NormArgs& a) {
#define KRM_BLOCK_NORM(THREADS, PIECES) \
  block_norm_kernel<XT, OT, THREADS, PIECES, VEC><<<dim3(rows), dim3(THREADS), 0, ctx->stream>>>(a)
  if (a.dim <= 512) KRM_BLOCK_NORM(64, 1);
  else if (a.dim <= 1024) KRM_BLOCK_NORM(128, 1);
  else if (a.dim <= 2048) KRM_BLOCK_NORM(256, 1);
  else if (a.dim <= 4096) KRM_BLOCK_NORM(512, 1);
  else if (a.dim <= 8192) KRM_BLOCK_NORM(512, 2);
  else KRM_BLOCK_NORM(1024, 2);
#undef KRM_BLOCK_NORM
}

}  // namespace

extern "C" int32_t krm_block_norm(krm_ctx* ctx, krm_buf y, krm_buf post_weight, krm_buf gate,
                                  krm_buf residual, krm_buf pre_weight, krm_buf sum_out,
                                  krm_buf norm_out, uint32_t rows, uint32_t dim, uint32_t gate_span,
                                  int32_t gate_kind, float eps, float block_scale,
                                  float residual_scale, int32_t io_dtype, int32_t norm_dtype) {
  KRM_TRY(enter(ctx));
  KRM_REQUIRE(ctx, valid_dtype(io_dtype) && valid_dtype(norm_dtype), "block_norm: unknown dtype %d / %d",
              io_dtype, norm_dtype);
  KRM_REQUIRE(ctx, norm_dtype == io_dtype || norm_dtype == KRM_F16,
              "block_norm: norm_dtype is io_dtype, or fp16 beside f32 rows");
  KRM_REQUIRE(ctx, gate_kind == KRM_GATE_PLAIN || gate_kind == KRM_GATE_SIGMOID,
              "block_norm: unknown gate kind %d", gate_kind);
  KRM_REQUIRE(ctx, dim >= 1 && dim <= 16384, "block_norm: dim %u is outside 1 .. 16384", dim);
  KRM_REQUIRE(ctx, rows <= 0x7fffffffu, "block_norm: %u rows", rows);
  KRM_REQUIRE(ctx, (pre_weight != 0) == (norm_out != 0),
              "block_norm: pre_weight and norm_out are given together");
  KRM_REQUIRE(ctx, sum_out || norm_out, "block_norm: neither sum_out nor norm_out");
  if (rows == 0) return KRM_OK;
  KRM_REQUIRE(ctx, y, "block_norm: null buffer");
  const size_t eb = dtype_bytes(io_dtype), nb = dtype_bytes(norm_dtype);
  KRM_REQUIRE(ctx, aligned(y, eb) && aligned(gate, eb) && aligned(residual, eb) && aligned(sum_out, eb) &&
                       aligned(norm_out, nb) && aligned(post_weight, 4) && aligned(pre_weight, 4),
              "block_norm: misaligned buffer");
  KRM_REQUIRE(ctx, sum_out != norm_out, "block_norm: sum_out and norm_out are one buffer");
  KRM_REQUIRE(ctx, !gate || (gate != sum_out && gate != norm_out), "block_norm: a result is the gate's buffer");
  KRM_REQUIRE(ctx, nb == eb || (!norm_out || (norm_out != y && norm_out != residual)),
              "block_norm: norm_out may be y or residual only if their types are the same");
  NormArgs a{ptr<const void>(y),        ptr<const float>(post_weight), ptr<const void>(gate),
                   ptr<const void>(residual), ptr<const float>(pre_weight),  ptr<void>(sum_out),
                   ptr<void>(norm_out),       dim,                           gate_span, 0u,
                   eps,                       block_scale,                   residual_scale,
                   gate_kind == KRM_GATE_SIGMOID};
  const bool vec = dim % 8 == 0 && aligned(y | gate | residual | sum_out | norm_out | post_weight | pre_weight, 16);
#define KRM_BLOCK_NORM_TYPES(XT, OT) \
  do { if (vec) launch_norm<XT, OT, true>(ctx, count, a); else launch_norm<XT, OT, false>(ctx, count, a); } while (0)
  constexpr uint32_t kRowsALaunch = 1u << 21;  // a launch has fewer than 2^32 threads
  while (a.first_row < rows) {
    const uint32_t count = min(rows - a.first_row, kRowsALaunch);
    if (io_dtype == KRM_F16) KRM_BLOCK_NORM_TYPES(__half, __half);
    else if (norm_dtype == KRM_F16) KRM_BLOCK_NORM_TYPES(float, __half);
    else KRM_BLOCK_NORM_TYPES(float, float);
    KRM_TRY(launched(ctx, "block_norm_kernel"));
    a.first_row += count;
  }
#undef KRM_BLOCK_NORM_TYPES
  return KRM_OK;
}
