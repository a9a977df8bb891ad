// Attention over the pages of the 4-bit K/V cache (layout: kv4_plan.h).
//
// Row r of a sequence stands at column p = len - rows + r and sees columns max(0, p - window + 1) .. p:
//   out = sum_c softmax_c(scale^2 q . k_c) v_c,   k_c = step * code + minimum, v_c alike.
#include "kv4_plan.h"
#include "krm_internal.h"

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

struct AttentionArgs {
  Kv4Layout layout;
  Kv4Limits limits;
  uint32_t heads, pages, window;
  float scale;   // half_scale^2 * log2 e: scores are kept in base 2
};

__device__ inline float half_at(const uint8_t* p) {
  return __half2float(__ushort_as_half(*reinterpret_cast<const uint16_t*>(p)));
}

// One workgroup a (row, head): 256 columns at a time, a score a thread, then an output element a thread
// (256 / D threads share its columns).
template <typename XT, int D>
__global__ __launch_bounds__(kThreads) void kv4_attention_kernel(
    const XT* __restrict__ q, const uint8_t* __restrict__ cache, const int32_t* __restrict__ page_table,
    const int32_t* __restrict__ cu_rows, const int32_t* __restrict__ lens, XT* __restrict__ out,
    uint32_t* __restrict__ fault, AttentionArgs a) {
  constexpr int kParts = kThreads / D;
  __shared__ float s_q[D], s_p[kThreads], s_acc[kThreads], s_red[kThreads / kWave];
  const uint32_t seq = blockIdx.y, tid = threadIdx.x;
  const uint32_t row = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
  const int32_t cu0 = cu_rows[seq], cu1 = cu_rows[seq + 1];
  const Kv4Sequence s = kv4_sequence(cu0, cu1, lens[seq], a.limits);
  const bool in_rows = cu0 >= 0 && cu1 >= cu0 && (uint32_t)cu1 <= a.limits.total_rows && row < (uint32_t)(cu1 - cu0);
  if (!s.ok && fault && blockIdx.x == 0 && tid == 0) *fault = 1u;
  if (!in_rows) return;
  const size_t base = (((size_t)s.first + row) * a.heads + head) * D;
  if (!s.ok) {
    if (tid < D) st<XT>(out, base + tid, NAN);
    return;
  }
  if (tid < D) s_q[tid] = ld<XT>(q, base + tid) * a.scale;
  const int32_t position = s.len - s.rows + (int32_t)row;
  const int32_t first = kv4_first_column(position, a.window);
  const uint32_t kv_head = head / (a.heads / a.layout.kv_heads);
  const int32_t* table = page_table + (size_t)seq * a.limits.table_stride;
  const uint32_t groups = a.layout.groups();
  float m = -INFINITY, l = 0.f, acc = 0.f;
  bool bad = false;
  const uint32_t d = tid % D, part = tid / D;
  __syncthreads();
  for (int32_t c0 = first; c0 <= position; c0 += kThreads) {
    const int32_t c = c0 + (int32_t)tid;
    float score = -INFINITY;
    if (c <= position) {
      const int32_t page = table[c / a.layout.page_rows];
      if (page < 0 || (uint32_t)page >= a.pages) {
        bad = true;
      } else {
        const uint8_t* block = cache + (size_t)page * a.layout.page() + (size_t)kv_head * a.layout.block();
        const uint32_t in_page = c & (a.layout.page_rows - 1);
        score = 0.f;
        for (uint32_t g = 0; g < groups; ++g) {
          float codes = 0.f, sum = 0.f;
          for (uint32_t w = g * a.layout.group / 8; w < (g + 1) * a.layout.group / 8; ++w) {
            const uint32_t word = *reinterpret_cast<const uint32_t*>(block + a.layout.key_word(in_page, w));
            for (int i = 0; i < 8; ++i) {
              const float qi = s_q[w * 8 + i];
              codes = fmaf(qi, (float)((word >> (4 * ((i & 1) * 4 + i / 2))) & 15u), codes);
              sum += qi;
            }
          }
          const uint8_t* param = block + a.layout.key_param(in_page, g);
          score = fmaf(half_at(param), codes, score);
          score = fmaf(half_at(param + 2), sum, score);
        }
      }
    }
    if (__syncthreads_or(bad)) {   // a page that is none of the cache's
      if (tid < D) st<XT>(out, base + tid, NAN);
      if (fault && tid == 0) *fault = 1u;
      return;
    }
    float top = score;
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
    if (tid % kWave == 0) s_red[tid / kWave] = top;
    __syncthreads();
    top = m;
    for (int w = 0; w < kThreads / kWave; ++w) top = fmaxf(top, s_red[w]);
    const float keep = __builtin_amdgcn_exp2f(m - top);
    m = top;
    const float p = c <= position ? __builtin_amdgcn_exp2f(score - m) : 0.f;
    s_p[tid] = p;
    __syncthreads();
    acc *= keep;
    l *= keep;
    for (uint32_t j = part; j < (uint32_t)kThreads && c0 + (int32_t)j <= position; j += kParts) {
      const uint32_t cj = (uint32_t)c0 + j, in_page = cj & (a.layout.page_rows - 1);
      const uint8_t* block =
          cache + (size_t)table[cj / a.layout.page_rows] * a.layout.page() + (size_t)kv_head * a.layout.block();
      const uint32_t word = *reinterpret_cast<const uint32_t*>(block + a.layout.value_word(in_page, d / 8));
      const uint8_t* param = block + a.layout.value_param(in_page, d / a.layout.group);
      acc = fmaf(s_p[j], fmaf(half_at(param), (float)((word >> (4 * (d % 8))) & 15u), half_at(param + 8)), acc);
      l += s_p[j];
    }
    __syncthreads();
  }
  s_acc[tid] = acc;
  s_p[tid] = l;
  __syncthreads();
  if (tid < D) {
    float total = 0.f, sum = 0.f;
    for (int w = 0; w < kParts; ++w) {
      total += s_acc[w * D + tid];
      sum += s_p[w * D + tid];
    }
    st<XT>(out, base + tid, total / sum);
  }
}

}  // namespace

extern "C" {

int32_t krm_kv4_attention_workspace(uint32_t nseq, uint32_t max_query, uint32_t max_columns, uint32_t total_rows,
                                    uint32_t heads, uint32_t kv_heads, uint32_t depth, uint32_t window,
                                    int32_t io_dtype, size_t* bytes) {
  KRM_REQUIRE(nullptr, bytes != nullptr, "krm_kv4_attention_workspace: bytes is NULL");
  KRM_REQUIRE(nullptr, valid_dtype(io_dtype), "krm_kv4_attention_workspace: io_dtype %d", io_dtype);
  char why[128];
  const Kv4Shape shape{nseq, max_query, total_rows, heads, kv_heads, depth, 32, 16, 1, 1};
  KRM_REQUIRE(nullptr, kv4_shape_ok(shape, why, sizeof why), "krm_kv4_attention_workspace: %s", why);
  KRM_REQUIRE(nullptr, max_columns <= 0x7fffffffu, "krm_kv4_attention_workspace: max_columns %u", max_columns);
  (void)window;
  *bytes = 0;
  return KRM_OK;
}

int32_t krm_kv4_attention(krm_ctx* ctx, krm_buf q, krm_buf cache, krm_buf page_table_i32, krm_buf cu_rows_i32,
                          krm_buf lens_i32, krm_buf out, krm_buf fault_u32, uint32_t nseq, uint32_t max_query,
                          uint32_t max_columns, uint32_t total_rows, uint32_t heads, uint32_t kv_heads,
                          uint32_t depth, uint32_t group, uint32_t page_rows, uint32_t pages,
                          uint32_t table_stride, uint32_t window, float half_scale, int32_t io_dtype,
                          krm_buf workspace, size_t workspace_bytes) {
  KRM_TRY(enter(ctx));
  KRM_REQUIRE(ctx, valid_dtype(io_dtype), "krm_kv4_attention: io_dtype %d", io_dtype);
  const Kv4Shape shape{nseq, max_query, total_rows, heads, kv_heads, depth, group, page_rows, pages, table_stride};
  char why[128];
  KRM_REQUIRE(ctx, kv4_shape_ok(shape, why, sizeof why), "krm_kv4_attention: %s", why);
  KRM_REQUIRE(ctx, std::isfinite(half_scale * half_scale), "krm_kv4_attention: half_scale");
  KRM_REQUIRE(ctx, max_columns <= 0x7fffffffu && (max_columns >= kv4_rows(max_query, total_rows)),
              "krm_kv4_attention: max_columns %u beside max_query %u", max_columns, max_query);
  if (nseq == 0 || total_rows == 0) return KRM_OK;
  KRM_REQUIRE(ctx, q && cache && page_table_i32 && cu_rows_i32 && lens_i32 && out, "krm_kv4_attention: NULL buffer");
  KRM_REQUIRE(ctx, aligned(q, 16) && aligned(out, 16) && aligned(cache, 16) && aligned(page_table_i32, 4) &&
                       aligned(cu_rows_i32, 4) && aligned(lens_i32, 4) && aligned(fault_u32, 4) &&
                       aligned(workspace, 16),
              "krm_kv4_attention: misaligned buffer (rows, cache and workspace: 16 bytes)");
  KRM_REQUIRE(ctx, q != out, "krm_kv4_attention: out is q");
  (void)workspace_bytes;
  const AttentionArgs a{{depth, group, page_rows, kv_heads},
                        {total_rows, max_query, max_columns, table_stride, page_rows},
                        heads, pages, window, half_scale * half_scale * 1.4426950408889634f};
  const uint32_t rows = kv4_rows(max_query, total_rows);
  KRM_REQUIRE(ctx, (uint64_t)rows * heads <= 0x7fffffu, "krm_kv4_attention: %u rows of %u heads", rows, heads);
#define KRM_ATTENTION(XT, D)                                                                                    \
  kv4_attention_kernel<XT, D><<<dim3(rows * heads, nseq), dim3(kThreads), 0, ctx->stream>>>(                \
      ptr<const XT>(q), ptr<const uint8_t>(cache), ptr<const int32_t>(page_table_i32),                           \
      ptr<const int32_t>(cu_rows_i32), ptr<const int32_t>(lens_i32), ptr<XT>(out), ptr<uint32_t>(fault_u32), a)
#define KRM_ATTENTION_D(XT)                      \
  if (depth == 64) KRM_ATTENTION(XT, 64);        \
  else if (depth == 128) KRM_ATTENTION(XT, 128); \
  else KRM_ATTENTION(XT, 256)
  if (io_dtype == KRM_F32) { KRM_ATTENTION_D(float); } else { KRM_ATTENTION_D(__half); }
#undef KRM_ATTENTION_D
#undef KRM_ATTENTION
  return launched(ctx, "kv4_attention_kernel");
}

}  // extern "C"
