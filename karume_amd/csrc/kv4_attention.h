// What the two kernels of the 4-bit cache's attention share: their arguments, how a workgroup finds its work and how
// parts of a row are joined.
#pragma once

#include "i4_codes.h"
#include "kv4_plan.h"
#include "krm_internal.h"

namespace krm {

struct Kv4Attention {
  Kv4Layout layout;
  Kv4Limits limits;
  uint32_t nseq, heads, pages, window;
  uint32_t share;                     // query heads of a kv head
  float share_inverse;
  uint32_t least_pairs, most_pairs;   // (row, head) pairs of a sequence and kv head that the launch is for
  float scale;                        // half_scale^2 * log2 e: scores are kept in base 2
  float fraction;                     // scale / 2^frexp_exp(scale), from 0.5 up to 1
  float* partials;                    // parts of rows, as each kernel lays them out
  uint32_t* tickets;
};
// Workgroups that share a launch's columns, one a CU: with 512 and 1024 of them a decode step of 131000 columns took
// 49.4 us, with 256 39.8.
constexpr uint32_t kKv4Groups = 256;
struct Kv4Buffers {
  krm_buf q, cache, page_table, cu_rows, lens, out, fault;
};
// The kernel for many rows (kv4_chunk.hip).
size_t kv4_chunk_workspace(uint32_t depth, uint32_t max_columns);
int32_t launch_kv4_chunk(krm_ctx* ctx, const Kv4Attention& a, const Kv4Buffers& b, int32_t io_dtype);

#if defined(__HIPCC__)
namespace {

typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float2_t __attribute__((ext_vector_type(2)));

constexpr int kJoin = 16;           // parts whose sums are asked for together

// Device-scope load / store of two floats: read from (written through to) memory that every XCD sees.
__device__ inline float2_t observe2(const float* p) {
  return __builtin_bit_cast(float2_t, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                                        __HIP_MEMORY_SCOPE_AGENT));
}
__device__ inline void publish2(float* p, float2_t v) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
// Both rounded to nearest, in one step (and not a second time where a single one of them is used).
__device__ inline half2_t rounded2(float2_t x) {
  uint32_t bits = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, half2_t));
  asm("" : "+v"(bits));
  return __builtin_bit_cast(half2_t, bits);
}
// What rounding to `hi` left of x (one mixed instruction).
__device__ inline _Float16 less(float x, _Float16 hi) {
  float minus = -1.0f;
  asm("" : "+s"(minus));   // (else: a conversion and a subtraction)
  return (_Float16)fmaf((float)hi, minus, x);
}

// Over the lanes 16, 32 and 48 apart.
template <typename F>
__device__ inline float across_quarters(float x, F join) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = join(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return join(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float quarters_max(float x) {
  return across_quarters(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ inline float quarters_sum(float x) {
  return across_quarters(x, [](float a, float b) { return a + b; });
}

__device__ inline half2_t half2_of(uint32_t w) { return __builtin_bit_cast(half2_t, w); }
__device__ inline half8_t join8(half2_t a, half2_t b, half2_t c, half2_t d) {
  return half8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// Codes at the bottom (u) or four bits up (16 u) of the halves of a word, as the exact integers u - LESS.
template <int LESS>
__device__ inline half2_t low_codes(uint32_t x) {
  return half2_of(and_or(x, 0x000F000Fu, 0x64006400u)) -
         half2_t{(_Float16)(1024.0f + LESS), (_Float16)(1024.0f + LESS)};
}
template <int LESS>
__device__ inline half2_t high_codes(uint32_t x) {
  return __builtin_elementwise_fma(half2_of(and_or(x, 0x00F000F0u, 0x64006400u)),
                                   half2_t{(_Float16)0.0625f, (_Float16)0.0625f},
                                   half2_t{(_Float16)(-64.0f - LESS), (_Float16)(-64.0f - LESS)});
}
// step * x + sum with a step in fp16 (one mixed instruction).
__device__ inline float scaled(uint32_t params, float x, float sum) { return fmaf((float)half2_of(params).x, x, sum); }

// Weights are 2^(score - shift).  The shift is the largest score less 10, so that the weights' low parts are no subnormal
// numbers; past 2^24, where f32 does not hold that difference, it is the score itself.  What has been summed goes by the
// shift, in the lanes, in LDS and in a row's parts.
__device__ inline float shift_of(float top) { return fabsf(top) > 0x1p24f ? top : top - 10.0f; }
// The power of two by which a row of queries is multiplied, so that the largest is in [2^5, 2^6).  (Those so small or
// large that the scale would leave f32's range with them are not normalised any further.)  f32 rows are multiplied with
// the scale's fraction too: what is left of the scale is a power of two, with which no product is rounded.
__device__ inline int normal_power(float most, float scale) {
  if (!(most > 0.f && most < INFINITY)) return 0;
  const int of_scale = __builtin_amdgcn_frexp_expf(scale);
  return max(min(6 - __builtin_amdgcn_frexp_expf(most), min(100, of_scale + 100)), of_scale - 110);
}

template <int N>
__device__ inline void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    w[0] = a.x; w[1] = a.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 a = *reinterpret_cast<const uint4*>(p + 16 * i);
      w[4 * i] = a.x; w[4 * i + 1] = a.y; w[4 * i + 2] = a.z; w[4 * i + 3] = a.w;
    }
  }
}

// The same address in every lane, in scalar registers whatever the compiler made of it.
__device__ inline const uint8_t* uniform(const uint8_t* p) {
  const uint64_t at = (uint64_t)p;
  return (const uint8_t*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32)) << 32 |
                          (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at));
}
// x / d for x up to 2^24, `inverse` = 1 / d: the quotient in floating point, put right by the remainder.
__device__ inline uint32_t divided(uint32_t x, uint32_t d, float inverse) {
  const uint32_t guess = (uint32_t)((float)x * inverse);
  const int32_t rest = (int32_t)(x - guess * d);
  return rest < 0 ? guess - 1 : rest >= (int32_t)d ? guess + 1 : guess;
}

// A piece of work: some (row, head) pairs of one kv head of a sequence, over some of the columns that they see.
struct Work {
  uint32_t seq, kv_head;
  uint32_t count, row0, head0;        // pairs; the first one's row in the step and its head in the kv head
  int32_t cu0, first_row, last_row;   // the sequence's first row in `q`; columns at which the first and last row stand
  int32_t low, high, begin, end;      // columns that any of them sees; tiles of this piece
};
__device__ inline uint32_t row_of(const Kv4Attention& a, const Work& w, uint32_t pair) {   // from row0 on
  return divided(w.head0 + pair, a.share, a.share_inverse);
}
__device__ inline size_t row_at(const Kv4Attention& a, const Work& w, uint32_t pair, uint32_t depth) {
  const uint32_t row = row_of(a, w, pair), head = w.kv_head * a.share + w.head0 + pair - row * a.share;
  return (((size_t)(uint32_t)w.cu0 + w.row0 + row) * a.heads + head) * depth;
}
// The rows of a refused sequence, in the heads of one kv head, are NaN.
template <typename XT, int D, int kThreads>
__device__ inline void refuse(const Kv4Attention& a, uint32_t kv_head, int32_t cu0, int32_t cu1, XT* __restrict__ out) {
  const uint32_t wide = a.share * D;
  uint32_t tid = threadIdx.x;
  asm volatile("" : "+v"(tid));   // (addresses are found here, not beside all of a kernel's work)
  for (int32_t row = cu0; row < cu1; ++row) {
    XT* to = out + ((size_t)(uint32_t)row * a.heads + kv_head * a.share) * D;
    for (uint32_t e = tid; e < wide; e += kThreads) to[e] = from_f32<XT>(NAN);
  }
}
// Counts this workgroup's part of some rows, which it has published; true in the one that counts last, which joins the
// parts in order, whichever it is, and leaves the counter at zero.
__device__ inline bool arrived_last(uint32_t* ticket, uint32_t parts) {
  __shared__ uint32_t s_ticket;
  // every store of this workgroup is through before it is counted (a release fence would write the whole L2 back)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) s_ticket = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  const bool last = s_ticket + 1 == parts;
  if (last && threadIdx.x == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return last;
}

}  // namespace
#endif

}  // namespace krm
