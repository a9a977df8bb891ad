// Rotary positions beyond the half-split whole-head form: tables made on the device for any set of
// frequencies, and the rotation of interleaved or half-split pairs in part of each head.
#include "kv4_plan.h"
#include "i4_codes.h"
#include "krm_internal.h"
#include "rotary.h"
#include "rows8.h"

#include <cmath>

using namespace krm;

namespace {

constexpr int kThreads = 256;

// cos and sin of position * frequency.  The angle and its reduction are in 64 bits: at position 1e6 a 32-bit angle is off
// by 0.03.  The product is kept whole, as its rounded value a and what that left: past 2^30 the rounding alone would move
// the angle by up to 2^-23.  a = n pi/2 + r with |r| <= pi/4 (pi/2 in two parts, so that r keeps its bits for any n a
// position can give), then both series in 32 bits on r: the first terms left out are r^11/11! < 1.8e-9 and r^12/12! <
// 1.2e-10, below half a step of the result.  In units of 2^-25: r is off by 1, the sine by its own rounding and 0.3 more,
// the cosine by 2.5 in all at |r| = pi/4 and less nearer to 1; the amplitude's product rounds by 2 of the result.
// Together below 4, 2^-23 of the amplitude.
// A thread keeps VEC frequencies and walks rows, so that it needs no division and stores 16 bytes at a time (with one
// element a thread and its place by division 131072 x 64 pairs, 67 MB, took 17.7 us; see krm_rope_tables).
template <int VEC>
__global__ __launch_bounds__(kThreads) void rope_tables_kernel(const double* __restrict__ freq,
                                                              float* __restrict__ cos_table,
                                                              float* __restrict__ sin_table, uint32_t first,
                                                              uint32_t rows, uint32_t pairs, uint32_t width,
                                                              float amplitude, uint32_t across, uint32_t at_once) {
  const uint32_t down = threadIdx.x / across, j = (blockIdx.y * across + threadIdx.x - down * across) * VEC;
  if (down >= at_once || j >= pairs) return;
  double f[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = freq[j + i];
  const uint32_t step = gridDim.x * at_once;
  for (uint64_t row = blockIdx.x * (uint64_t)at_once + down; row < rows; row += step) {
    const double position = (double)first + (double)row;
    float c[VEC], s[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const double angle = position * f[i];
      const double n = rint(angle * 0.63661977236758134308);
      const double part = fma(-n, 1.57079632679489661923, angle), left = fma(position, f[i], -angle);
      const float r = (float)(fma(-n, 6.12323399573676603587e-17, part) + left);
      const int quarter = (int)(n - 4.0 * floor(n * 0.25));
      const float r2 = r * r;
      float sn = fmaf(r2, 2.7557319e-6f, -1.9841270e-4f);
      sn = fmaf(r2, sn, 8.3333333e-3f);
      sn = fmaf(r2, sn, -1.6666667e-1f);
      sn = fmaf(r2 * r, sn, r);
      float cs = fmaf(r2, -2.7557319e-7f, 2.4801587e-5f);
      cs = fmaf(r2, cs, -1.3888889e-3f);
      cs = fmaf(r2, cs, 4.1666667e-2f);
      cs = fmaf(r2, cs, -0.5f);
      cs = fmaf(r2, cs, 1.0f);
      const float cosine = quarter & 1 ? sn : cs, sine = quarter & 1 ? cs : sn;
      c[i] = (quarter == 1 || quarter == 2 ? -cosine : cosine) * amplitude;
      s[i] = (quarter >= 2 ? -sine : sine) * amplitude;
    }
    const size_t at = row * width + j;
    auto put = [&](size_t to) {
      if constexpr (VEC == 4) {
        *reinterpret_cast<float4*>(cos_table + to) = make_float4(c[0], c[1], c[2], c[3]);
        *reinterpret_cast<float4*>(sin_table + to) = make_float4(s[0], s[1], s[2], s[3]);
      } else {
        cos_table[to] = c[0];
        sin_table[to] = s[0];
      }
    };
    put(at);
    if (width > pairs) put(at + pairs);   // both halves of a row, as krm_rope_half reads them
  }
}

// Rows whose pieces of 8 elements are whole and 16-byte aligned: a workgroup has `block_rows` rows (or a part of one
// row's heads), whose angles it holds in LDS, so that all heads share one trip to the table; a thread has both sides of
// 8 pairs (interleaved: 4), or 8 elements that are only copied.  What bounds it is memory: 5003 rows of 40 heads of 128
// fp16 head-major, 105 MB: 22.3 us, 4.7 TB/s (two elements and their angles a thread: 55.9).  (x and out may be one
// buffer, and nothing here tells the compiler otherwise.)
template <typename XT, bool HALF>
__global__ __launch_bounds__(kThreads) void rope_pieces_kernel(
    const XT* x, const int32_t* __restrict__ positions, const float* __restrict__ cos_table,
    const float* __restrict__ sin_table, XT* out, uint32_t rows, uint32_t heads, RotaryArgs t,
    uint64_t x_stride, uint64_t out_stride, uint32_t to_head_major, uint32_t block_rows, uint32_t block_heads) {
  extern __shared__ __align__(16) float s_angles[];   // [block_rows][2][R/2]
  const uint32_t pairs = t.rotary_dim / 2, row0 = blockIdx.x * block_rows, head0 = blockIdx.y * block_heads;
  const uint32_t my_rows = min(block_rows, rows - row0), my_heads = min(block_heads, heads - head0);
  const uint32_t turns = HALF ? t.rotary_dim / 16 : t.rotary_dim / 8;     // items of a head that are turned
  const uint32_t per_head = turns + (t.head_dim - t.rotary_dim) / 8, per_row = my_heads * per_head;
  const uint32_t items = my_rows * per_row;
  // (the first item's elements are asked for before the angles; an item has both sides of its pairs, so that rows may
  // be turned in place)
  struct Item {
    float a[8], b[8];
    XT* dst;
    const float* angles;
    uint32_t d;
    bool turned;
  };
  auto ask = [&](uint32_t i) __attribute__((always_inline)) {
    Item w;
    const uint32_t r = i / per_row, in_row = i - r * per_row, h = in_row / per_head, item = in_row - h * per_head;
    const size_t row = row0 + r, head = head0 + h;
    const XT* src = x + row * x_stride + head * t.head_dim;
    w.dst = out + (to_head_major ? (head * rows + row) * t.head_dim : row * out_stride + head * t.head_dim);
    w.angles = s_angles + r * 2 * pairs;
    w.turned = item < turns;
    w.d = w.turned ? 8 * item : t.rotary_dim + 8 * (item - turns);
    load8(src + w.d, w.a);
    if (HALF && w.turned) load8(src + pairs + w.d, w.b);
    return w;
  };
  auto finish = [&](const Item& w) __attribute__((always_inline)) {
    if (!w.turned) {
      store8(w.dst + w.d, w.a);
    } else if constexpr (HALF) {
      float cs[8], sn[8], ta[8], tb[8];
      load8(w.angles + w.d, cs);
      load8(w.angles + pairs + w.d, sn);
#pragma unroll
      for (int k = 0; k < 8; ++k) turn_pair(w.a[k], w.b[k], cs[k], sn[k], ta[k], tb[k]);
      store8(w.dst + w.d, ta);
      store8(w.dst + pairs + w.d, tb);
    } else {
      const float4 cs = *reinterpret_cast<const float4*>(w.angles + w.d / 2);
      const float4 sn = *reinterpret_cast<const float4*>(w.angles + pairs + w.d / 2);
      const float co[4] = {cs.x, cs.y, cs.z, cs.w}, si[4] = {sn.x, sn.y, sn.z, sn.w};
      float turned[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) turn_pair(w.a[2 * k], w.a[2 * k + 1], co[k], si[k], turned[2 * k], turned[2 * k + 1]);
      store8(w.dst + w.d, turned);
    }
  };
  uint32_t i = threadIdx.x;
  Item now;
  if (i < items) now = ask(i);
  for (uint32_t i = threadIdx.x; i < my_rows * pairs; i += kThreads) {
    const uint32_t r = i / pairs, j = i - r * pairs;
    const int32_t pos = positions[row0 + r];
    const bool known = pos >= 0 && (uint32_t)pos < t.table_rows;
    const size_t at = (size_t)(known ? pos : 0) * t.table_width + j;
    // no angle: must not look like a rotation
    s_angles[r * 2 * pairs + j] = known ? cos_table[at] : NAN;
    s_angles[(r * 2 + 1) * pairs + j] = known ? sin_table[at] : NAN;
  }
  __syncthreads();
  while (i < items) {
    finish(now);
    i += kThreads;
    if (i < items) now = ask(i);
  }
}

template <typename XT>
__global__ __launch_bounds__(kThreads) void rope_rows_kernel(
    const XT* x, const int32_t* __restrict__ positions, const float* __restrict__ cos_table,
    const float* __restrict__ sin_table, XT* out, uint32_t rows, uint32_t heads, RotaryArgs t,
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
    const float a = to_f32<XT>(x[src + d0]);
    const float b = d1 < t.head_dim ? to_f32<XT>(x[src + d1]) : 0.f;
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
    out[dst + d0] = from_f32<XT>(ta);
    if (d1 < t.head_dim) out[dst + d1] = from_f32<XT>(tb);
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
  const bool wide = pairs % 4 == 0 && aligned(cos_table_f32, 16) && aligned(sin_table_f32, 16);
  const uint32_t columns = wide ? pairs / 4 : pairs, across = columns < kThreads ? columns : kThreads;
  const uint32_t at_once = kThreads / across;
  const uint64_t blocks = ((uint64_t)rows + at_once - 1) / at_once;
  const dim3 grid(blocks > 4096 ? 4096u : (uint32_t)blocks, (columns + across - 1) / across), block(kThreads);
  KRM_REQUIRE(ctx, grid.y <= 65535, "krm_rope_tables: %u pairs", pairs);
#define KRM_TABLES(VEC)                                                                                               \
  rope_tables_kernel<VEC><<<grid, block, 0, ctx->stream>>>(ptr<const double>(inv_freq_f64), ptr<float>(cos_table_f32), \
                                                           ptr<float>(sin_table_f32), first_position, rows, pairs,     \
                                                           width, amplitude, across, at_once)
  if (wide) KRM_TABLES(4);
  else KRM_TABLES(1);
#undef KRM_TABLES
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
  KRM_REQUIRE(ctx, rows <= 0x7fffffffu, "krm_rope_rows: %u rows", rows);
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
  const size_t eb = dtype_bytes(io_dtype);
  const bool half = layout == KRM_ROPE_HALF;
  if (head_dim % 8 == 0 && rotary_dim % (half ? 16 : 8) == 0 && rotary_dim <= 512 && aligned(x, 16) && aligned(out, 16) &&
      x_stride * eb % 16 == 0 && (to_head_major || out_stride * eb % 16 == 0)) {
    // two pieces a thread or so: several short rows a workgroup, or several workgroups a long row
    const uint32_t per_head = rotary_dim / (half ? 16 : 8) + (head_dim - rotary_dim) / 8;
    const uint64_t items = (uint64_t)heads * per_head;
    uint32_t block_rows = items >= 2 * kThreads ? 1 : (uint32_t)((2 * kThreads + items - 1) / items);
    block_rows = block_rows > 16 ? 16 : block_rows > rows ? rows : block_rows;
    if ((rows + block_rows - 1) / block_rows < 256) block_rows = block_rows > 2 ? block_rows / 2 : 1;
    const uint32_t heads_most = 4 * kThreads / per_head ? 4 * kThreads / per_head : 1;
    const uint32_t block_heads = heads < heads_most ? heads : heads_most;
    const dim3 grid((rows + block_rows - 1) / block_rows, (heads + block_heads - 1) / block_heads), block(kThreads);
    if (grid.x <= 0x7fffffu && grid.y <= 65535) {
#define KRM_PIECES(XT, HALF)                                                                                         \
  rope_pieces_kernel<XT, HALF><<<grid, block, (size_t)block_rows * rotary_dim * sizeof(float), ctx->stream>>>(       \
      ptr<const XT>(x), ptr<const int32_t>(positions_i32), ptr<const float>(cos_table_f32),                          \
      ptr<const float>(sin_table_f32), ptr<XT>(out), rows, heads, t, x_stride, out_stride,                           \
      (uint32_t)(to_head_major != 0), block_rows, block_heads)
      if (io_dtype == KRM_F32) { if (half) KRM_PIECES(float, true); else KRM_PIECES(float, false); }
      else { if (half) KRM_PIECES(__half, true); else KRM_PIECES(__half, false); }
#undef KRM_PIECES
      return launched(ctx, "rope_pieces_kernel");
    }
  }
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
