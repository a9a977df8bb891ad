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
  uint32_t share;          // query heads of a kv head
  uint32_t row_tiles;      // blocks of (row, head) pairs of a kv head, a workgroup each
  float share_inverse, row_tiles_inverse, of_sequence_inverse;
  uint32_t max_splits;     // workgroups that one block's columns are dealt to at most
  uint32_t partial_rows;   // pairs that a part of kv4_decode_kernel has room for
  uint32_t least;          // tiles, at least, of a split
  uint32_t least_pairs, most_pairs;   // of a sequence and kv head that this launch is for
  float share_of_work;     // of all sequences' tiles, in one workgroup
  float scale;             // half_scale^2 * log2 e: scores are kept in base 2
  float* partials;         // [unit][split]: sums of all pairs, then their (max, sum); as each kernel lays them out
  uint32_t* tickets;
};
struct Kv4Buffers {
  krm_buf q, cache, page_table, cu_rows, lens, out, fault;
};
// Blocks of kv4_chunk_pairs() pairs a workgroup (kv4_chunk.hip).
uint32_t kv4_chunk_pairs(uint32_t depth);
uint32_t kv4_chunk_columns(uint32_t depth);   // of a tile
int32_t launch_kv4_chunk(krm_ctx* ctx, const Kv4Attention& a, const Kv4Buffers& b, uint32_t units, int32_t io_dtype);

#if defined(__HIPCC__)
namespace {

typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float2_t __attribute__((ext_vector_type(2)));

constexpr int kJoin = 32;           // parts whose sums are asked for together

// Device-scope store / load of one float: written through to (read from) memory that every XCD sees.
__device__ inline void publish(float* p, float v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ inline float observe(const float* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

__device__ inline float2_t observe2(const float* p) {
  return __builtin_bit_cast(float2_t, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

__device__ inline void publish2(float* p, float2_t v) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
// Over all lanes.
__device__ inline float wave_sum(float x) {
#define KRM_ADD_DPP(CTRL, ROWS) \
  x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false))
  KRM_ADD_DPP(0x111, 0xf);   // row_shr:1
  KRM_ADD_DPP(0x112, 0xf);
  KRM_ADD_DPP(0x114, 0xf);
  KRM_ADD_DPP(0x118, 0xf);
  KRM_ADD_DPP(0x142, 0xa);   // row_bcast:15
  KRM_ADD_DPP(0x143, 0xc);   // row_bcast:31
#undef KRM_ADD_DPP
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}


// The work of a workgroup: kPairs (row, head) pairs of one kv head of a sequence, over some of their columns.
struct Work {
  uint32_t unit, seq, kv_head, split, nsplit;
  uint32_t count, row0, head0;        // pairs; the first one's row in the step and its head in the kv head
  int32_t cu0, first_row, last_row;   // the sequence's first row in `q`; columns at which the first and last row stand
  int32_t low, high, begin, end;      // columns that any of them sees; this split's tiles
};
__device__ inline uint32_t row_of(const Kv4Attention& a, const Work& w, uint32_t pair) {   // from row0 on
  return divided(w.head0 + pair, a.share, a.share_inverse);
}
__device__ inline size_t row_at(const Kv4Attention& a, const Work& w, uint32_t pair, uint32_t depth) {
  const uint32_t row = row_of(a, w, pair), head = w.kv_head * a.share + w.head0 + pair - row * a.share;
  return (((size_t)(uint32_t)w.cu0 + w.row0 + row) * a.heads + head) * depth;
}
// Grid (units, splits): workgroups go to the XCDs in turn, and a unit (sequence, kv head, block of pairs) has its
// next split on the next XCD, so that neither first splits nor a long sequence gather on one of them (32 sequences
// of up to 4096 columns with splits along x, two XCDs at work: 182 us, so 42.6).
__device__ inline void find_unit(const Kv4Attention& a, Work& w, uint32_t& block) {
  const uint32_t units = gridDim.x, of_sequence = a.layout.kv_heads * a.row_tiles;
  w.split = blockIdx.y;
  w.unit = blockIdx.x;
  if (w.split) {
    w.unit += units > w.split ? w.split : w.split % units;
    if (w.unit >= units) w.unit -= units;
  }
  w.seq = divided(w.unit, of_sequence, a.of_sequence_inverse);
  const uint32_t in_sequence = w.unit - w.seq * of_sequence;
  w.kv_head = divided(in_sequence, a.row_tiles, a.row_tiles_inverse);
  block = in_sequence - w.kv_head * a.row_tiles;
}
// False: nothing to do (or done: rows of a refused sequence are NaN).
template <typename XT, int D, int kThreads, int kPairs, int kTile, int kWaves>
__device__ inline bool find_work(const Kv4Attention& a, Work& w, uint32_t block, const int32_t* __restrict__ cu_rows,
                                 const int32_t* __restrict__ lens, XT* __restrict__ out, uint32_t* __restrict__ fault) {
  const uint32_t tid = threadIdx.x, pair0 = block * kPairs;
  float work = 0.f;
  if (a.max_splits > 1) {
    for (uint32_t i = tid % kWave; i < a.nseq; i += kWave) {
      const uint32_t n = min((uint32_t)max(lens[i], 0), a.limits.max_columns);
      work += (float)((a.window ? min(n, a.window) : n) / kTile + 1);
    }
  }
  const int32_t cu1 = cu_rows[w.seq + 1];
  w.cu0 = cu_rows[w.seq];
  const Kv4Sequence s = kv4_sequence(w.cu0, cu1, lens[w.seq], a.limits);
  if (!s.ok && fault && w.split == 0 && tid == 0) *fault = 1u;   // (whichever launch its rows belong to)
  if (w.cu0 < 0 || cu1 < w.cu0 || (uint32_t)cu1 > a.limits.total_rows) return false;
  const uint64_t pairs = (uint64_t)(uint32_t)(cu1 - w.cu0) * a.share;
  if (pair0 >= pairs || pairs < a.least_pairs || pairs > a.most_pairs) return false;
  w.count = min((uint64_t)kPairs, pairs - pair0);
  w.row0 = divided(pair0, a.share, a.share_inverse);
  w.head0 = pair0 - w.row0 * a.share;
  if (!s.ok) {
    if (w.split == 0)
      for (uint32_t e = tid; e < w.count * D; e += kThreads) out[row_at(a, w, e / D, D) + e % D] = from_f32<XT>(NAN);
    return false;
  }
  w.first_row = s.len - s.rows + (int32_t)w.row0;
  w.last_row = w.first_row + (int32_t)row_of(a, w, w.count - 1);
  w.low = kv4_first_column(w.first_row, a.window);
  w.high = w.last_row;
  const int32_t tile0 = w.low / kTile;
  const uint32_t tiles = (uint32_t)(w.high / kTile - tile0 + 1);
  uint32_t per = tiles;
  w.nsplit = 1;
  if (a.max_splits > 1) {
    // the step's tiles, as far as they go by the lengths, are dealt evenly to the workgroups that fit the machine
    per = max((uint32_t)(wave_sum(work) * a.share_of_work), a.least) + kWaves - 1;
    per = max(per / kWaves * kWaves, (tiles + a.max_splits - 1) / a.max_splits);
    w.nsplit = (tiles + per - 1) / per;
    if (w.split >= w.nsplit) return false;
  }
  w.begin = tile0 + (int32_t)min(w.split * per, tiles);
  w.end = tile0 + (int32_t)min((w.split + 1) * per, tiles);
  return true;
}

// A workgroup's part of its rows is published; the workgroup that arrives last joins the parts in order, whichever it
// is.  `s_part`: nsplit * count * 2 floats of LDS that nobody needs any more.
template <typename XT, int D, int kThreads>
__device__ inline void join_parts(const Kv4Attention& a, const Work& w, XT* __restrict__ out, float* s_part) {
  __shared__ uint32_t s_ticket;
  const uint32_t tid = threadIdx.x, nsplit = w.nsplit, count = w.count;
  const size_t part_size = (size_t)a.partial_rows * (D + 2);
  const float* const parts = a.partials + (size_t)w.unit * a.max_splits * part_size;
  // every store of this workgroup is through before it is counted (a release fence would write the whole L2 back)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  uint32_t* ticket = a.tickets + (size_t)w.unit * kTicketStride;
  if (tid == 0) s_ticket = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s_ticket + 1 != nsplit) return;
  if (tid == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (uint32_t i = tid; i < nsplit * count; i += kThreads) {   // [row][nsplit] (max, sum)
    const float* state = parts + (i / count) * part_size + a.partial_rows * D + 2 * (i % count);
    float* to = s_part + ((i % count) * nsplit + i / count) * 2;
    to[0] = observe(state);
    to[1] = observe(state + 1);
  }
  __syncthreads();
  for (uint32_t e = 2 * tid; e < count * D; e += 2 * kThreads) {
    const float* states = s_part + (e / D) * nsplit * 2;
    float most = -INFINITY, weight = 0.f;
    float2_t total = {0.f, 0.f};
    for (uint32_t p = 0; p < nsplit; ++p) most = fmaxf(most, states[2 * p]);
    const float ref = most == -INFINITY ? 0.f : most;
    for (uint32_t p0 = 0; p0 < nsplit; p0 += kJoin) {
      float2_t o[kJoin];
#pragma unroll
      for (int i = 0; i < kJoin; ++i) o[i] = observe2(parts + min(p0 + i, nsplit - 1) * part_size + e);
#pragma unroll
      for (int i = 0; i < kJoin; ++i) {
        if (p0 + i < nsplit) {
          const float k = __builtin_amdgcn_exp2f(states[2 * (p0 + i)] - ref);
          total[0] = fmaf(k, o[i][0], total[0]);
          total[1] = fmaf(k, o[i][1], total[1]);
          weight = fmaf(k, states[2 * (p0 + i) + 1], weight);
        }
      }
    }
    XT* to = out + row_at(a, w, e / D, D) + e % D;
    to[0] = from_f32<XT>(total[0] / weight);
    to[1] = from_f32<XT>(total[1] / weight);
  }
}

}  // namespace
#endif

}  // namespace krm
