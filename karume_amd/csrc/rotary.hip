// Rotary positions beyond the half-split whole-head form: tables made on the device for any set of
// frequencies, and the rotation of interleaved or half-split pairs in part of each head.
#include "kv4_plan.h"
#include "krm_internal.h"
#include "rotary.h"

#include <cmath>

using namespace krm;

namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ inline float ld(const T* p, size_t i);
template <>
__device__ inline float ld<float>(const float* p, size_t i) { return p[i]; }
template <>
__device__ inline float ld<__half>(const __half* p, size_t i) { return __half2float(p[i]); }
template <typename T>
__device__ inline void st(T* p, size_t i, float v);
template <>
__device__ inline void st<float>(float* p, size_t i, float v) { p[i] = v; }
template <>
__device__ inline void st<__half>(__half* p, size_t i, float v) { p[i] = __float2half_rn(v); }

// cos and sin of position * frequency.  The angle and its reduction are in 64 bits: at position 1e6 a
// 32-bit angle is off by 0.03.  a = n pi/2 + r with |r| <= pi/4 (pi/2 in two parts, so that r keeps its
// bits for any n a position can give), then both series in 32 bits on r: the first terms left out are
// r^11/11! < 1.8e-9 and r^12/12! < 1.2e-10, below half a step of the result.
__global__ __launch_bounds__(kThreads) void rope_tables_kernel(const double* __restrict__ freq,
                                                              float* __restrict__ cos_table,
                                                              float* __restrict__ sin_table, uint32_t first,
                                                              uint32_t rows, uint32_t pairs, uint32_t width,
                                                              float amplitude) {
  const size_t total = (size_t)rows * pairs;
  const size_t stride = (size_t)gridDim.x * kThreads;
  for (size_t i = blockIdx.x * (size_t)kThreads + threadIdx.x; i < total; i += stride) {
    const uint32_t j = (uint32_t)(i % pairs);
    const size_t row = i / pairs;
    const double angle = ((double)first + (double)row) * freq[j];
    const double n = rint(angle * 0.63661977236758134308);
    const double part = fma(-n, 1.57079632679489661923, angle);
    const float r = (float)fma(-n, 6.12323399573676603587e-17, part);
    const int quarter = (int)(n - 4.0 * floor(n * 0.25));
    const float r2 = r * r;
    float s = fmaf(r2, 2.7557319e-6f, -1.9841270e-4f);
    s = fmaf(r2, s, 8.3333333e-3f);
    s = fmaf(r2, s, -1.6666667e-1f);
    s = fmaf(r2 * r, s, r);
    float c = fmaf(r2, -2.7557319e-7f, 2.4801587e-5f);
    c = fmaf(r2, c, -1.3888889e-3f);
    c = fmaf(r2, c, 4.1666667e-2f);
    c = fmaf(r2, c, -0.5f);
    c = fmaf(r2, c, 1.0f);
    float cosine = quarter & 1 ? s : c, sine = quarter & 1 ? c : s;
    if (quarter == 1 || quarter == 2) cosine = -cosine;
    if (quarter >= 2) sine = -sine;
    cosine *= amplitude;
    sine *= amplitude;
    const size_t at = row * width + j;
    cos_table[at] = cosine;
    sin_table[at] = sine;
    if (width > pairs) {   // both halves of a row, as krm_rope_half reads them
      cos_table[at + pairs] = cosine;
      sin_table[at + pairs] = sine;
    }
  }
}

template <typename XT>
__global__ __launch_bounds__(kThreads) void rope_rows_kernel(
    const XT* __restrict__ x, const int32_t* __restrict__ positions, const float* __restrict__ cos_table,
    const float* __restrict__ sin_table, XT* __restrict__ out, uint32_t rows, uint32_t heads, RotaryArgs t,
    uint64_t x_stride, uint64_t out_stride, uint32_t to_head_major) {
  // a thread has both elements of a pair (or two elements that are only copied), so that rows may be
  // turned in place
  const uint32_t half = t.head_dim / 2 + (t.head_dim & 1);
  const size_t total = (size_t)rows * heads * half;
  const size_t stride = (size_t)gridDim.x * kThreads;
  for (size_t i = blockIdx.x * (size_t)kThreads + threadIdx.x; i < total; i += stride) {
    const uint32_t j = (uint32_t)(i % half);
    const size_t rest = i / half;
    const uint32_t head = (uint32_t)(rest % heads);
    const size_t row = rest / heads;
    const size_t src = row * x_stride + (size_t)head * t.head_dim;
    const size_t dst = to_head_major ? ((size_t)head * rows + row) * t.head_dim
                                     : row * out_stride + (size_t)head * t.head_dim;
    const uint32_t pairs = t.rotary_dim / 2;
    uint32_t d0, d1;
    if (j < pairs) {
      d0 = t.layout == KRM_ROPE_HALF ? j : 2 * j;
      d1 = t.layout == KRM_ROPE_HALF ? j + pairs : 2 * j + 1;
    } else {
      d0 = 2 * j;
      d1 = 2 * j + 1;
    }
    const float a = ld<XT>(x, src + d0);
    const float b = d1 < t.head_dim ? ld<XT>(x, src + d1) : 0.f;
    float ta = a, tb = b;
    if (j < pairs) {
      const int32_t pos = positions[row];
      if (pos < 0 || (uint32_t)pos >= t.table_rows) {
        ta = tb = NAN;   // no angle: must not look like a rotation
      } else {
        const size_t at = (size_t)pos * t.table_width + j;
        turn_pair(a, b, cos_table[at], sin_table[at], ta, tb);
      }
    }
    st<XT>(out, dst + d0, ta);
    if (d1 < t.head_dim) st<XT>(out, dst + d1, tb);
  }
}

inline unsigned grid_for(size_t total) {
  const size_t blocks = (total + kThreads - 1) / kThreads;
  return (unsigned)(blocks > 8192 ? 8192 : blocks ? blocks : 1);
}

}  // namespace

extern "C" {

int32_t krm_rope_tables(krm_ctx* ctx, krm_buf inv_freq_f64, krm_buf cos_table_f32, krm_buf sin_table_f32,
                        uint32_t first_position, uint32_t rows, uint32_t pairs, uint32_t width, float amplitude) {
  KRM_TRY(enter(ctx));
  KRM_REQUIRE(ctx, pairs >= 1 && (width == pairs || (width % 2 == 0 && width / 2 == pairs)),
              "krm_rope_tables: width %u beside %u pairs (once or twice as many)", width, pairs);
  KRM_REQUIRE(ctx, std::isfinite(amplitude), "krm_rope_tables: amplitude");
  KRM_REQUIRE(ctx, (uint64_t)first_position + rows <= 0x80000000ull,
              "krm_rope_tables: positions from %u, %u of them, pass 2^31", first_position, rows);
  if (rows == 0) return KRM_OK;
  KRM_REQUIRE(ctx, inv_freq_f64 && cos_table_f32 && sin_table_f32, "krm_rope_tables: NULL buffer");
  KRM_REQUIRE(ctx, aligned(inv_freq_f64, 8) && aligned(cos_table_f32, 4) && aligned(sin_table_f32, 4),
              "krm_rope_tables: misaligned buffer");
  rope_tables_kernel<<<dim3(grid_for((size_t)rows * pairs)), dim3(kThreads), 0, ctx->stream>>>(
      ptr<const double>(inv_freq_f64), ptr<float>(cos_table_f32), ptr<float>(sin_table_f32), first_position, rows,
      pairs, width, amplitude);
  return launched(ctx, "rope_tables_kernel");
}

int32_t krm_rope_rows(krm_ctx* ctx, krm_buf x, krm_buf positions_i32, krm_buf cos_table_f32, krm_buf sin_table_f32,
                      krm_buf out, uint32_t rows, uint32_t heads, uint32_t head_dim, uint32_t rotary_dim,
                      int32_t layout, uint32_t table_rows, uint32_t table_width, uint64_t x_stride,
                      uint64_t out_stride, int32_t to_head_major, int32_t io_dtype) {
  KRM_TRY(enter(ctx));
  KRM_REQUIRE(ctx, valid_dtype(io_dtype), "krm_rope_rows: io_dtype %d", io_dtype);
  char why[128];
  KRM_REQUIRE(ctx, head_dim >= 1 && kv4_turn_ok(head_dim, rotary_dim, layout, table_rows, table_width, why, sizeof why),
              "krm_rope_rows: %s", head_dim ? why : "head_dim 0");
  if (rows == 0 || heads == 0) return KRM_OK;
  const uint64_t packed = (uint64_t)heads * head_dim;
  KRM_REQUIRE(ctx, x && out && (rotary_dim == 0 || (positions_i32 && cos_table_f32 && sin_table_f32)),
              "krm_rope_rows: NULL buffer");
  KRM_REQUIRE(ctx, x_stride >= packed && (to_head_major || out_stride >= packed),
              "krm_rope_rows: row strides below %llu elements", (unsigned long long)packed);
  KRM_REQUIRE(ctx, aligned(x, dtype_bytes(io_dtype)) && aligned(out, dtype_bytes(io_dtype)) &&
                       aligned(positions_i32, 4) && aligned(cos_table_f32, 4) && aligned(sin_table_f32, 4),
              "krm_rope_rows: misaligned buffer");
  KRM_REQUIRE(ctx, x != out || rows == 1 ||
                       (to_head_major ? heads == 1 && x_stride == packed : x_stride == out_stride),
              "krm_rope_rows: in place, rows keep their places");
  const RotaryArgs t{head_dim, rotary_dim, table_rows, table_width, layout};
  const dim3 grid(grid_for((size_t)rows * heads * (head_dim / 2 + (head_dim & 1)))), block(kThreads);
#define KRM_ROWS(XT)                                                                                          \
  rope_rows_kernel<XT><<<grid, block, 0, ctx->stream>>>(                                                      \
      ptr<const XT>(x), ptr<const int32_t>(positions_i32), ptr<const float>(cos_table_f32),                   \
      ptr<const float>(sin_table_f32), ptr<XT>(out), rows, heads, t, x_stride, out_stride, (uint32_t)(to_head_major != 0))
  if (io_dtype == KRM_F32) KRM_ROWS(float);
  else KRM_ROWS(__half);
#undef KRM_ROWS
  return launched(ctx, "rope_rows_kernel");
}

}  // extern "C"
