// Writing and reading back the pages of the 4-bit K/V cache (layout: kv4_plan.h).
//
// A group of g elements along a head is held as x ~ step * code + minimum with code in 0 .. 15:
//   minimum = the largest fp16 not above min(x),  step = the least fp16 not below (max(x) - minimum) / 15,
//   code = round-half-even((x - minimum) / step)
// Both parameters are rounded outwards, so no element is clipped and every one is off by step / 2 at most
// (beside the roundings of the f32 operations).  A group that is constant has step 0 and codes 0.
#include "kv4_plan.h"
#include "i4_codes.h"
#include "krm_internal.h"
#include "rotary.h"
#include "rows8.h"

#include <cmath>

using namespace krm;

namespace {

constexpr int kThreads = 256;
constexpr int kPiece = 8;   // elements of a thread: one word of codes

__device__ inline uint16_t bits_of(__half h) { return __half_as_ushort(h); }
__device__ inline float value_of(uint16_t b) { return __half2float(__ushort_as_half(b)); }
// The largest fp16 not above v / the least not below it (|v| within fp16's range).
__device__ inline uint16_t half_down(float v) {
  uint16_t b = bits_of(__float2half_rn(v));
  if (value_of(b) > v) b = (b & 0x7fff) == 0 ? 0x8001 : (b & 0x8000) ? b + 1 : b - 1;
  return b;
}
__device__ inline uint16_t half_up(float v) {
  uint16_t b = bits_of(__float2half_rn(v));
  if (value_of(b) < v) b = (b & 0x7fff) == 0 ? 0x0001 : (b & 0x8000) ? b - 1 : b + 1;
  return b;
}

struct AppendArgs {
  Kv4Layout layout;
  Kv4Limits limits;
  RotaryArgs turn;
  uint32_t heads, pages;
  uint64_t q_stride, k_stride, v_stride;   // elements between rows
};

// A thread has 8 elements of one head's row, D / 8 neighbouring lanes the row.  A workgroup has 256 * 8 / D of the
// (H + 2 Hkv) heads of one row of the step, whose angles it holds in LDS: queries are turned and stored, keys turned,
// quantised and stored, values quantised and stored.
// What bounds it is memory: 8100 f32 rows of 32 + 2 x 8 heads of 128, 342 MB, take 65 us (5.2 TB/s, some of it from the
// last-level cache); with the read-back 79, and 96 with angles fetched by every head and places found by division.  One
// row of 64 sequences: 3.9 us, less than its launch takes the host.
// PIECES: a thread's elements are turned as whole pieces (pairs within 8 elements, or 8 pairs across two pieces).
template <typename XT, int D, bool PIECES>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(
    const XT* __restrict__ k, const XT* __restrict__ v, uint8_t* __restrict__ cache,
    const int32_t* __restrict__ page_table, const int32_t* __restrict__ cu_rows, const int32_t* __restrict__ lens,
    const XT* q, XT* q_out, const int32_t* __restrict__ positions, const float* __restrict__ cos_table,
    const float* __restrict__ sin_table, uint32_t* __restrict__ fault, AppendArgs a) {
  constexpr int kLanes = D / kPiece;
  __shared__ __align__(16) float s_cos[D / 2], s_sin[D / 2];
  const uint32_t seq = blockIdx.z, row = blockIdx.x;
  const Kv4Sequence s = kv4_sequence(cu_rows[seq], cu_rows[seq + 1], lens[seq], a.limits);
  if (!s.ok) {
    if (fault && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *fault = 1u;
    return;
  }
  if (row >= (uint32_t)s.rows) return;
  const uint32_t hkv = a.layout.kv_heads, units = a.heads + 2 * hkv;
  const uint32_t sub = threadIdx.x % kLanes, mine = blockIdx.y * (kThreads / kLanes) + threadIdx.x / kLanes;
  const bool live = mine < units;
  const uint32_t unit = live ? mine : units - 1;
  const bool is_q = unit < a.heads, is_v = unit >= a.heads + hkv;
  const uint32_t head = is_q ? unit : is_v ? unit - a.heads - hkv : unit - a.heads;
  const uint64_t token = (uint64_t)s.first + row;
  const uint32_t column = (uint32_t)(s.len - s.rows) + row;
  const XT* src = (is_q ? q + token * a.q_stride : is_v ? v + token * a.v_stride : k + token * a.k_stride) + (size_t)head * D;
  const uint32_t pairs = a.turn.rotary_dim / 2, d0 = sub * kPiece;
  const bool by_half = a.turn.layout == KRM_ROPE_HALF;
  const bool turns = !is_v && d0 < a.turn.rotary_dim, second = by_half && d0 >= pairs;   // (PIECES: of the whole piece)
  float x[8], other[8];
  load8(src + d0, x);
  if constexpr (PIECES) {
    if (by_half && turns) load8(src + (second ? d0 - pairs : d0 + pairs), other);   // (before any lane of the row stores)
  }
  const int32_t in_table = (int32_t)column / (int32_t)a.layout.page_rows;
  const int32_t page = page_table[(size_t)seq * a.limits.table_stride + in_table];
  if (pairs) {
    const int32_t pos = positions ? positions[token] : (int32_t)column;
    const bool known = pos >= 0 && (uint32_t)pos < a.turn.table_rows;
    const size_t at = (size_t)(known ? pos : 0) * a.turn.table_width;
    if (threadIdx.x < pairs) {
      s_cos[threadIdx.x] = known ? cos_table[at + threadIdx.x] : __builtin_nanf("");
      s_sin[threadIdx.x] = known ? sin_table[at + threadIdx.x] : __builtin_nanf("");
    }
    __syncthreads();
    if constexpr (PIECES) {
      if (turns && by_half) {
        const uint32_t j = second ? d0 - pairs : d0;
        float c[8], sn[8];
        load8(s_cos + j, c);
        load8(s_sin + j, sn);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float ta, tb;
          turn_pair(second ? other[i] : x[i], second ? x[i] : other[i], c[i], sn[i], ta, tb);
          x[i] = second ? tb : ta;
        }
      } else if (turns) {
        const float4 c = *reinterpret_cast<const float4*>(s_cos + d0 / 2), sn = *reinterpret_cast<const float4*>(s_sin + d0 / 2);
        const float co[4] = {c.x, c.y, c.z, c.w}, si[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float ta, tb;
          turn_pair(x[2 * i], x[2 * i + 1], co[i], si[i], ta, tb);
          x[2 * i] = ta;
          x[2 * i + 1] = tb;
        }
      }
    } else {
      // any even rotary_dim: partners from the row itself, all read before any lane of the row stores
      float turned[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t d = d0 + i;
        const bool pair = !is_v && d < a.turn.rotary_dim, late = by_half ? d >= pairs : d & 1;
        const uint32_t j = !pair ? 0 : by_half ? (late ? d - pairs : d) : d / 2;
        const float o = pair ? to_f32<XT>(src[by_half ? (late ? d - pairs : d + pairs) : d ^ 1]) : 0.f;
        float ta, tb;
        turn_pair(late ? o : x[i], late ? x[i] : o, s_cos[j], s_sin[j], ta, tb);
        turned[i] = !pair ? x[i] : late ? tb : ta;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = turned[i];
    }
  }
  if (is_q) {
    if (live) store8(q_out + (token * a.heads + head) * D + d0, x);
    return;   // (rows of a head lie in one wave's neighbouring lanes: no group below spans a query row)
  }

  float low = x[0], high = x[0];
  bool fine = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    fine = fine && fabsf(x[i]) <= kKv4Limit;   // false for NaN
    low = fminf(low, x[i]);
    high = fmaxf(high, x[i]);
  }
  const uint32_t lanes = a.layout.group / kPiece;
  int ok = fine;
  for (uint32_t off = 1; off < lanes; off <<= 1) {
    low = fminf(low, __shfl_xor(low, off, kWave));
    high = fmaxf(high, __shfl_xor(high, off, kWave));
    ok &= __shfl_xor(ok, off, kWave);
  }
  uint16_t minimum = 0, step = 0x7e00;
  uint32_t word = 0;
  if (ok) {
    minimum = half_down(low + 0.0f);   // (a zero is held as +0)
    const float base = value_of(minimum);
    step = half_up((high - base) / 15.0f);
    const float wide = step ? value_of(step) : 1.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float code = fminf(fmaxf(rintf((x[i] - base) / wide), 0.0f), 15.0f);
      const int nibble = is_v ? i : (i & 1) * 4 + i / 2;
      word |= (uint32_t)code << (4 * nibble);
    }
  }
  if (!live) return;
  const uint32_t in_page = column & (a.layout.page_rows - 1);
  if (page < 0 || (uint32_t)page >= a.pages) {
    if (fault && sub == 0) *fault = 1u;
    return;
  }
  uint8_t* block = cache + (size_t)page * a.layout.page() + (size_t)head * a.layout.block();
  const uint32_t g = d0 / a.layout.group;
  if (is_v) {
    *reinterpret_cast<uint32_t*>(block + a.layout.value_word(in_page, sub)) = word;
    if (sub % lanes == 0) {
      uint16_t* p = reinterpret_cast<uint16_t*>(block + a.layout.value_param(in_page, g));
      p[0] = step;
      p[4] = minimum;
    }
  } else {
    *reinterpret_cast<uint32_t*>(block + a.layout.key_word(in_page, sub)) = word;
    if (sub % lanes == 0)
      *reinterpret_cast<uint32_t*>(block + a.layout.key_param(in_page, g)) = step | (uint32_t)minimum << 16;
  }
}

// The last rows of each sequence as the values they stand for: step * code is exact in f32 and the sum is rounded once.
// Rows on a page that is none of the cache's, and all of a refused sequence, are NaN.  (8100 rows of 2 x 8 heads of 128 to
// fp16, 43 MB: 12.4 us.)
template <typename OT, int D>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(
    const uint8_t* __restrict__ cache, const int32_t* __restrict__ page_table, const int32_t* __restrict__ cu_rows,
    const int32_t* __restrict__ lens, OT* __restrict__ k_out, OT* __restrict__ v_out, uint32_t* __restrict__ fault,
    Kv4Layout layout, Kv4Limits limits, uint32_t pages) {
  constexpr int kLanes = D / kPiece;
  const uint32_t seq = blockIdx.y;
  const Kv4Sequence s = kv4_sequence(cu_rows[seq], cu_rows[seq + 1], lens[seq], limits);
  const uint32_t hkv = layout.kv_heads;
  if (!s.ok) {
    if (fault && blockIdx.x == 0 && threadIdx.x == 0) *fault = 1u;
    const float none[8] = {NAN, NAN, NAN, NAN, NAN, NAN, NAN, NAN};
    const uint64_t pieces = (uint64_t)s.rows * hkv * kLanes;   // (rows: 0 where the offsets are none; may pass max_query)
    const size_t first = (size_t)(uint32_t)s.first * hkv * D;
    for (uint64_t i = blockIdx.x * (uint64_t)kThreads + threadIdx.x; i < pieces; i += (uint64_t)gridDim.x * kThreads) {
      store8(k_out + first + i * kPiece, none);
      store8(v_out + first + i * kPiece, none);
    }
    return;
  }
  const uint64_t item = (blockIdx.x * (uint64_t)kThreads + threadIdx.x) / kLanes;
  if (item >= (uint64_t)s.rows * hkv * 2) return;
  const uint32_t row = (uint32_t)(item / (2 * hkv));
  const uint32_t unit = (uint32_t)(item % (2 * hkv));
  const bool is_v = unit >= hkv;
  const uint32_t head = is_v ? unit - hkv : unit, sub = threadIdx.x % kLanes;
  const uint32_t column = (uint32_t)(s.len - s.rows) + row;
  OT* dst = (is_v ? v_out : k_out) + (((size_t)s.first + row) * hkv + head) * D + sub * kPiece;
  const int32_t page = page_table[(size_t)seq * limits.table_stride + column / layout.page_rows];
  float x[8];
  if (page < 0 || (uint32_t)page >= pages) {
    if (fault && sub == 0) *fault = 1u;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_nanf("");
  } else {
    const uint8_t* block = cache + (size_t)page * layout.page() + (size_t)head * layout.block();
    const uint32_t in_page = column & (layout.page_rows - 1), g = sub * kPiece / layout.group;
    const uint8_t* param = block + (is_v ? layout.value_param(in_page, g) : layout.key_param(in_page, g));
    const uint32_t word = *reinterpret_cast<const uint32_t*>(
        block + (is_v ? layout.value_word(in_page, sub) : layout.key_word(in_page, sub)));
    const float step = value_of(*reinterpret_cast<const uint16_t*>(param));
    const float base = value_of(*reinterpret_cast<const uint16_t*>(param + (is_v ? 8 : 2)));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int nibble = is_v ? i : (i & 1) * 4 + i / 2;
      x[i] = fmaf(step, (float)((word >> (4 * nibble)) & 15u), base);
    }
  }
  store8(dst, x);
}

}  // namespace

extern "C" {

int32_t krm_kv4_page_bytes(uint32_t kv_heads, uint32_t depth, uint32_t group, uint32_t page_rows, size_t* bytes) {
  KRM_REQUIRE(nullptr, bytes != nullptr, "krm_kv4_page_bytes: bytes is NULL");
  char why[128];
  const Kv4Shape s{0, 0, 0, kv_heads, kv_heads, depth, group, page_rows, 1, 1};
  KRM_REQUIRE(nullptr, kv4_layout_ok(s, why, sizeof why), "krm_kv4_page_bytes: %s", why);
  *bytes = (size_t)Kv4Layout{depth, group, page_rows, kv_heads}.page();
  return KRM_OK;
}

int32_t krm_kv4_append(krm_ctx* ctx, krm_buf q, krm_buf k, krm_buf v, krm_buf q_out, krm_buf positions_i32,
                       krm_buf cos_table_f32, krm_buf sin_table_f32, krm_buf cache, krm_buf page_table_i32,
                       krm_buf cu_rows_i32, krm_buf lens_i32, krm_buf fault_u32, uint32_t nseq, uint32_t max_query,
                       uint32_t total_rows, uint32_t heads, uint32_t kv_heads, uint32_t depth, uint32_t group,
                       uint32_t page_rows, uint32_t pages, uint32_t table_stride, uint64_t q_stride,
                       uint64_t k_stride, uint64_t v_stride, uint32_t rotary_dim, int32_t layout,
                       uint32_t table_rows, uint32_t table_width, int32_t io_dtype) {
  KRM_TRY(enter(ctx));
  KRM_REQUIRE(ctx, valid_dtype(io_dtype), "krm_kv4_append: io_dtype %d", io_dtype);
  KRM_REQUIRE(ctx, (q != 0) == (q_out != 0), "krm_kv4_append: q and q_out are given together or not at all");
  const Kv4Shape shape{nseq, max_query, total_rows, q ? heads : kv_heads, kv_heads, depth, group, page_rows, pages,
                       table_stride};
  char why[128];
  KRM_REQUIRE(ctx, kv4_shape_ok(shape, why, sizeof why) &&
                       kv4_turn_ok(depth, rotary_dim, layout, table_rows, table_width, why, sizeof why),
              "krm_kv4_append: %s", why);
  if (nseq == 0 || total_rows == 0) return KRM_OK;
  KRM_REQUIRE(ctx, k && v && cache && page_table_i32 && cu_rows_i32 && lens_i32 &&
                       (rotary_dim == 0 || (cos_table_f32 && sin_table_f32)),
              "krm_kv4_append: NULL buffer");
  const uint64_t kv_row = (uint64_t)kv_heads * depth, q_row = (uint64_t)heads * depth;
  const size_t eb = dtype_bytes(io_dtype);
  KRM_REQUIRE(ctx, k_stride >= kv_row && v_stride >= kv_row && (!q || q_stride >= q_row),
              "krm_kv4_append: a row stride is below its heads x depth");
  KRM_REQUIRE(ctx, aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(q_out, 16) && aligned(cache, 16) &&
                       k_stride * eb % 16 == 0 && v_stride * eb % 16 == 0 && (!q || q_stride * eb % 16 == 0) &&
                       aligned(positions_i32, 4) && aligned(cos_table_f32, 4) && aligned(sin_table_f32, 4) &&
                       aligned(page_table_i32, 4) && aligned(cu_rows_i32, 4) && aligned(lens_i32, 4) &&
                       aligned(fault_u32, 4),
              "krm_kv4_append: misaligned buffer or row stride (rows and cache: 16 bytes)");
  KRM_REQUIRE(ctx, q != q_out || !q || q_stride == q_row, "krm_kv4_append: in place, query rows keep their places");
  const AppendArgs a{{depth, group, page_rows, kv_heads},
                     {total_rows, max_query, 0x7fffffffu, table_stride, page_rows},
                     {depth, rotary_dim, table_rows, table_width, layout},
                     q ? heads : 0u, pages, q_stride, k_stride, v_stride};
  const uint32_t rows = kv4_rows(max_query, total_rows);
  KRM_REQUIRE(ctx, rows <= 0x7fffffu, "krm_kv4_append: %u rows of a sequence are more than one call takes", rows);
  const dim3 grid(rows, ((a.heads + 2 * kv_heads) * (depth / kPiece) + kThreads - 1) / kThreads, nseq);
  const bool pieces = rotary_dim % (layout == KRM_ROPE_HALF ? 16 : 8) == 0;
#define KRM_APPEND(XT, D) { if (pieces) KRM_APPEND_P(XT, D, true); else KRM_APPEND_P(XT, D, false); }
#define KRM_APPEND_P(XT, D, PIECES)                                                                             \
  kv4_append_kernel<XT, D, PIECES><<<grid, dim3(kThreads), 0, ctx->stream>>>(                                    \
      ptr<const XT>(k), ptr<const XT>(v), ptr<uint8_t>(cache), ptr<const int32_t>(page_table_i32),               \
      ptr<const int32_t>(cu_rows_i32), ptr<const int32_t>(lens_i32), ptr<const XT>(q), ptr<XT>(q_out),           \
      ptr<const int32_t>(positions_i32), ptr<const float>(cos_table_f32), ptr<const float>(sin_table_f32),       \
      ptr<uint32_t>(fault_u32), a)
#define KRM_APPEND_D(XT)                      \
  if (depth == 64) KRM_APPEND(XT, 64)         \
  else if (depth == 128) KRM_APPEND(XT, 128)  \
  else KRM_APPEND(XT, 256)
  if (io_dtype == KRM_F32) { KRM_APPEND_D(float) } else { KRM_APPEND_D(__half) }
#undef KRM_APPEND_D
#undef KRM_APPEND_P
#undef KRM_APPEND
  return launched(ctx, "kv4_append_kernel");
}

int32_t krm_kv4_read(krm_ctx* ctx, krm_buf cache, krm_buf page_table_i32, krm_buf cu_rows_i32, krm_buf lens_i32,
                     krm_buf k_out, krm_buf v_out, krm_buf fault_u32, uint32_t nseq, uint32_t max_query,
                     uint32_t total_rows, uint32_t kv_heads, uint32_t depth, uint32_t group, uint32_t page_rows,
                     uint32_t pages, uint32_t table_stride, int32_t out_dtype) {
  KRM_TRY(enter(ctx));
  KRM_REQUIRE(ctx, valid_dtype(out_dtype), "krm_kv4_read: out_dtype %d", out_dtype);
  const Kv4Shape shape{nseq, max_query, total_rows, kv_heads, kv_heads, depth, group, page_rows, pages, table_stride};
  char why[128];
  KRM_REQUIRE(ctx, kv4_shape_ok(shape, why, sizeof why), "krm_kv4_read: %s", why);
  if (nseq == 0 || total_rows == 0) return KRM_OK;
  KRM_REQUIRE(ctx, cache && page_table_i32 && cu_rows_i32 && lens_i32 && k_out && v_out, "krm_kv4_read: NULL buffer");
  KRM_REQUIRE(ctx, aligned(cache, 16) && aligned(k_out, 16) && aligned(v_out, 16) && aligned(page_table_i32, 4) &&
                       aligned(cu_rows_i32, 4) && aligned(lens_i32, 4) && aligned(fault_u32, 4),
              "krm_kv4_read: misaligned buffer (rows and cache: 16 bytes)");
  const Kv4Layout layout{depth, group, page_rows, kv_heads};
  const Kv4Limits limits{total_rows, max_query, 0x7fffffffu, table_stride, page_rows};
  const uint64_t threads = (uint64_t)kv4_rows(max_query, total_rows) * 2 * kv_heads * (depth / kPiece);
  const uint64_t blocks = (threads + kThreads - 1) / kThreads;
  KRM_REQUIRE(ctx, blocks <= 0x7fffffu, "krm_kv4_read: %u rows of a sequence are more than one call takes", max_query);
#define KRM_READ(OT, D)                                                                                        \
  kv4_read_kernel<OT, D><<<dim3((uint32_t)blocks, nseq), dim3(kThreads), 0, ctx->stream>>>(                     \
      ptr<const uint8_t>(cache), ptr<const int32_t>(page_table_i32), ptr<const int32_t>(cu_rows_i32),           \
      ptr<const int32_t>(lens_i32), ptr<OT>(k_out), ptr<OT>(v_out), ptr<uint32_t>(fault_u32), layout, limits, pages)
#define KRM_READ_D(OT)                      \
  if (depth == 64) KRM_READ(OT, 64);        \
  else if (depth == 128) KRM_READ(OT, 128); \
  else KRM_READ(OT, 256)
  if (out_dtype == KRM_F32) { KRM_READ_D(float); } else { KRM_READ_D(__half); }
#undef KRM_READ_D
#undef KRM_READ
  return launched(ctx, "kv4_read_kernel");
}

}  // extern "C"
