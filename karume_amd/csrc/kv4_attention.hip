// Attention over the pages of the 4-bit K/V cache (layout: kv4_plan.h).
//
// Row r of a sequence stands at column p = len - rows + r and sees columns max(0, p - window + 1) .. p:
//   out = sum_c softmax_c(scale^2 q . k_c) v_c,   k_c = step * code + minimum, v_c alike.
// This is the kernel for few rows.  A long sequence is bound by memory (131000 columns, 8 kv heads x 4, D 128, groups of
// 64, 151 MB: 38 us, 4.0 TB/s), ragged batches by the vector instructions that turn codes (about 340 a tile of 32 columns
// beside 28 matrix ones) and by unequal pieces (32 sequences of 128 to 4096 columns 33 us), short ones by the chain
// lengths, pages, columns, waves' join (500 columns 9.1 us).
// What is rounded to fewer than 22 bits: fp16 rows' values, to fp16, once.  Their products with the weights' two parts are
// half of the matrix instructions, and a low part of the values would make them half as many again.  The result, fp16
// itself, is off from 64 bits by 2.8e-4 (2-norm); of exact values it would be by 2.0e-4.
#include "kv4_attention.h"
#include "lds_stream.h"
#include "rows8.h"

#include <cmath>

using namespace krm;

namespace {

constexpr int kStages = 2;         // tiles of a wave on their way
constexpr int kTile = 32;          // columns a wave takes at a time
constexpr int kRows = 16;          // (row, head) pairs of a workgroup
constexpr float kLog2e = 1.4426950408889634f;

// What a wave needs of 32 columns, two halves of 16, and where it lies in the wave's part of LDS.  Lane (i = lane %
// 16, c = lane / 16) of an operand needs of each half
//   keys    words (c, .) of row i, all parameters of rows i and 4 c .. 4 c + 3
//   values  rows 4 c .. 4 c + 3: word columns i (+ 16) and the parameters of their groups
// (a depth of 64 has eight word columns: lanes 8 .. 15 carry the upper half words of columns 0 .. 7).  Codes come in
// 16-byte pieces that a lane asks for and reads itself, so LDS is only where they wait; parameters are shared.
template <int D, int NG>
struct Stage {
  static constexpr int kSteps = D / 32;
  static constexpr int kColumns = D <= 128 ? 1 : D / 128;     // word columns of a lane
  static constexpr int kParts = kColumns;                     // pieces of a half's key row that a lane has
  static constexpr int kWords = NG <= 4 ? 1 : 2;              // dwords a lane of a half's parameters
  static constexpr uint32_t kParams = 256 * kWords;           // bytes of a half's parameters
  static constexpr uint32_t kKeys = 0, kValues = 2 * kParts * 1024, kKeyParams = 4 * kParts * 1024,
                            kValueParams = kKeyParams + 2 * kParams, kBytes = kValueParams + 2 * kParams;
  static constexpr int kLoads = 4 * kParts + 4 * kWords;      // that fill it
};

struct DecodeAttention : Kv4Attention {
  uint32_t row_tiles;      // blocks of kRows pairs of a kv head, a workgroup each
  float row_tiles_inverse, of_sequence_inverse;
  uint32_t max_splits;     // workgroups that one block's columns are dealt to at most
  uint32_t partial_rows;   // pairs that a part has room for; parts are [unit][split]: sums of all pairs, their (max, sum)
  uint32_t least;          // tiles, at least, of a split
  float share_of_work;     // of all sequences' tiles of a kv head, in one workgroup
};
struct DecodeWork : Work {
  uint32_t unit, split, nsplit;
};
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
// Grid (units, splits): workgroups go to the XCDs in turn, and a unit (sequence, kv head, block of pairs) has its
// next split on the next XCD, so that neither first splits nor a long sequence gather on one of them (32 sequences
// of up to 4096 columns with splits along x, two XCDs at work: 182 us, so 42.6).
__device__ inline void find_unit(const DecodeAttention& a, DecodeWork& w, uint32_t& block) {
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
template <typename XT, int D, int kWaves>
__device__ inline bool find_work(const DecodeAttention& a, DecodeWork& w, uint32_t block, const int32_t* __restrict__ cu_rows,
                                 const int32_t* __restrict__ lens, XT* __restrict__ out, uint32_t* __restrict__ fault) {
  constexpr int kThreads = kWaves * kWave;
  const uint32_t tid = threadIdx.x, pair0 = block * kRows;
  float work = 0.f;
  if (a.max_splits > 1) {
    for (uint32_t i = tid % kWave; i < a.nseq; i += kWave) {
      work += kv4_tiles((uint32_t)(cu_rows[i + 1] - cu_rows[i]), lens[i], a.share, a.least_pairs, a.most_pairs, kRows,
                        a.window, a.limits.max_columns, kTile);
    }
  }
  const int32_t cu1 = cu_rows[w.seq + 1];
  w.cu0 = cu_rows[w.seq];
  const Kv4Sequence s = kv4_sequence(w.cu0, cu1, lens[w.seq], a.limits);
  if (!s.ok && fault && w.split == 0 && tid == 0) *fault = 1u;   // (whichever launch its rows belong to)
  if (w.cu0 < 0 || cu1 < w.cu0 || (uint32_t)cu1 > a.limits.total_rows) return false;
  const uint64_t pairs = (uint64_t)(uint32_t)(cu1 - w.cu0) * a.share;
  if (pair0 >= pairs || pairs < a.least_pairs || pairs > a.most_pairs) return false;
  if (!s.ok) {
    if (w.split == 0 && block == 0) refuse<XT, D, kThreads>(a, w.kv_head, w.cu0, cu1, out);
    return false;
  }
  w.count = min((uint64_t)kRows, pairs - pair0);
  w.row0 = divided(pair0, a.share, a.share_inverse);
  w.head0 = pair0 - w.row0 * a.share;
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
    // (sequences that share rows, which no valid offsets give, could add up to any number)
    per = max((uint32_t)fminf(wave_sum(work) * a.share_of_work, 0x1p30f), a.least) + kWaves - 1;
    per = max(per / kWaves * kWaves, (tiles + a.max_splits - 1) / a.max_splits);
    w.nsplit = (tiles + per - 1) / per;
    if (w.split >= w.nsplit) return false;
  }
  w.begin = tile0 + (int32_t)min(w.split * per, tiles);
  w.end = tile0 + (int32_t)min((w.split + 1) * per, tiles);
  return true;
}

__device__ inline void store4(float* to, float4_t x) { *reinterpret_cast<float4_t*>(to) = x; }
__device__ inline void store4(__half* to, float4_t x) {
  const half2_t a = {(_Float16)x[0], (_Float16)x[1]}, b = {(_Float16)x[2], (_Float16)x[3]};
  *reinterpret_cast<uint2*>(to) = make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
}

// A workgroup's part of its rows is published; the workgroup that arrives last joins the parts in order, whichever it
// is.
template <typename XT, int D, int kThreads>
__device__ inline void join_parts(const DecodeAttention& a, const DecodeWork& w, XT* __restrict__ out) {
  const uint32_t tid = threadIdx.x, nsplit = w.nsplit, count = w.count;
  const size_t part_size = (size_t)a.partial_rows * (D + 2);
  const float* const parts = a.partials + (size_t)w.unit * a.max_splits * part_size;
  if (!arrived_last(a.tickets + (size_t)w.unit * kTicketStride, nsplit)) return;
  for (uint32_t e = 4 * tid; e < count * D; e += 4 * kThreads) {
    float top = -INFINITY, weight = 0.f;
    float4_t total = {};
    for (uint32_t p0 = 0; p0 < nsplit; p0 += kJoin) {
      float2_t o[kJoin][2] = {}, state[kJoin];
#pragma unroll
      for (int i = 0; i < kJoin; ++i) {
        state[i] = {-INFINITY, 0.f};
        if (p0 + i < nsplit) {
          const float* from = parts + (p0 + i) * part_size;
          state[i] = observe2(from + a.partial_rows * D + 2 * (e / D));
          o[i][0] = observe2(from + e);
          o[i][1] = observe2(from + e + 2);
        }
      }
      float now = top;
#pragma unroll
      for (int i = 0; i < kJoin; ++i) now = fmaxf(now, state[i][0]);
      const float ref = now == -INFINITY ? 0.f : now, keep = __builtin_amdgcn_exp2f(top - ref);
      top = now;
      weight *= keep;
      total *= keep;
#pragma unroll
      for (int i = 0; i < kJoin; ++i) {
        const float k = __builtin_amdgcn_exp2f(state[i][0] - ref);
#pragma unroll
        for (int j = 0; j < 4; ++j) total[j] = fmaf(k, o[i][j / 2][j % 2], total[j]);
        weight = fmaf(k, state[i][1], weight);
      }
    }
    store4(out + row_at(a, w, e / D, D) + e % D, total / weight);
  }
}

// (Three waves a SIMD: LDS has room for three workgroups of four waves of fp16 rows, up to D = 128, and so have 168
// registers.  With 176 and more, two of them, 32 sequences of 128 to 4096 columns take 37 us, so 33.)
template <typename XT, int D, int NG, int kWaves>
__global__ __launch_bounds__(kWaves* kWave, kWaves == 4 && D <= 128 && sizeof(XT) == 2 ? 3 : 1) void kv4_decode_kernel(
    const XT* __restrict__ q, const uint8_t* __restrict__ cache, const int32_t* __restrict__ page_table,
    const int32_t* __restrict__ cu_rows, const int32_t* __restrict__ lens, XT* __restrict__ out,
    uint32_t* __restrict__ fault, DecodeAttention a) {
  constexpr bool kF32 = sizeof(XT) == 4;
  constexpr int kThreads = kWaves * kWave;
  using S = Stage<D, NG>;
  constexpr int kSteps = S::kSteps, kColumns = S::kColumns;
  constexpr int kPerGroup = kSteps / NG;
  constexpr int kOuts = D == 64 ? 4 : 8;        // elements of a word column that a lane's rows carry
  constexpr int kStride = D + 4;                // of a row in LDS
  extern __shared__ __align__(16) uint8_t s_ring[];   // [wave][stage]; behind the tiles [wave][partial_rows][kStride] f32
  __shared__ float s_max[kWaves][kRows], s_sum[kWaves][kRows];

  const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  DecodeWork w;
  uint32_t block;
  find_unit(a, w, block);
  // the sequence's first 64 pages are asked for beside its lengths
  const int32_t* table = page_table + (size_t)w.seq * a.limits.table_stride;
  const uint32_t entry = (uint32_t)table[min(lane, a.limits.table_stride - 1)];
  if (!find_work<XT, D, kWaves>(a, w, block, cu_rows, lens, out, fault)) return;
  const uint32_t count = w.count;
  const int32_t first_row = w.first_row, last_row = w.last_row, low = w.low, high = w.high;
  // this wave's tiles are mine0, mine0 + kWaves, .. (the waves' next tiles lie together: in one long run for each wave
  // 131000 columns took 44.4 us, so 39.8)
  const int32_t mine0 = w.begin + (int32_t)wave;
  const int32_t mine = mine0 < w.end ? (int32_t)((uint32_t)(w.end - mine0 + kWaves - 1) / kWaves) : 0;

  // ---- the queries: lane (m = lane % 16, c): elements 32 s + 8 c .. + 7 of pair m for each step s
  const uint32_t m = lane & 15, c = lane >> 4;
  const bool live = m < count;
  const int32_t position = first_row + (int32_t)row_of(a, w, live ? m : 0);
  const int32_t from = kv4_first_column(position, a.window);
  float x[kSteps][8];
  {
    const XT* src = q + row_at(a, w, live ? m : 0, D) + 8 * c;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) load8(src + 32 * st, x[st]);
  }
  // Pages of 64 of this wave's tiles, a tile a lane.  kBad: outside the cache (page 0 is read in its place, its scores
  // become NaN and its values 0).  A half that no row sees has no page: page 0 is read, and nothing of it is used.
  const uint32_t page_shift = 31 - __builtin_clz(a.layout.page_rows);
  constexpr uint32_t kBad = 0x80000000u;
  uint32_t ids[2];
  auto find_pages = [&](int32_t index) {
    const bool near = (uint32_t)high >> page_shift < kWave;   // all in the entries that every wave has
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int32_t column = (mine0 + (index + (int32_t)lane) * kWaves) * kTile + 16 * h;
      const bool seen = index + (int32_t)lane < mine && column <= high && column + 15 >= low;
      const uint32_t at = seen ? (uint32_t)column >> page_shift : 0u;
      uint32_t id = near ? (uint32_t)__builtin_amdgcn_ds_bpermute((int)at * 4, (int)entry) : (uint32_t)table[at];
      if (!seen) id = 0;
      ids[h] = id < a.pages ? id : kBad;
    }
  };
  find_pages(0);

  // ---- a wave's ring: kStages tiles on their way
  auto lds_address = [](const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)p;
  };
  uint8_t* const ring = s_ring + wave * (kStages * S::kBytes);
  const uint32_t ring_at = lds_address(ring);
  const uint64_t page_bytes = a.layout.page();
  const uint8_t* head_base = cache + (size_t)w.kv_head * a.layout.block();
  const uint32_t column_of_lane = D == 64 ? (m & 7) : m;
  const uint32_t lane_k = m * (D / 2) + (D == 64 ? (c / 2) * 16 : c * (D / 8));
  const uint32_t lane_v = (c * (D / 8) + column_of_lane) * 16;
  uint32_t bad_halves = 0;   // two bits a stage
  auto ask = [&](int32_t index, uint32_t stage) {   // of this wave's tile `index`
    bad_halves &= ~(3u << (2 * stage));
    const uint32_t at = ring_at + stage * S::kBytes;
    const int32_t tile = mine0 + index * kWaves;
    if (index > 0 && (index & 63) == 0) find_pages(index);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int32_t column = tile * kTile + 16 * h;
      const uint32_t found = __builtin_amdgcn_readlane(ids[h], index & 63), id = found & ~kBad;
      if (found & kBad) bad_halves |= 1u << (2 * stage + h);
      const uint32_t in_page = (uint32_t)column & (a.layout.page_rows - 1);
      const uint8_t* block = uniform(head_base + id * page_bytes);
      const uint8_t* keys = block + in_page * (D / 2);
      const uint8_t* values = keys + a.layout.value_codes();
#pragma unroll
      for (int i = 0; i < S::kParts; ++i) {
        stream_to_lds(at + S::kKeys + (h * S::kParts + i) * 1024, lane_k + 16 * i, keys);
        stream_to_lds(at + S::kValues + (h * S::kParts + i) * 1024, lane_v + 256 * i, values);
      }
      const uint8_t* key_params = block + a.layout.key_params() + in_page * (NG * 4);
      const uint8_t* value_params = block + a.layout.value_params() + in_page * (NG * 4);
#pragma unroll
      for (int i = 0; i < S::kWords; ++i) {   // (16 rows' parameters are 64 NG bytes: lanes past them repeat the last)
        const uint32_t offset = min(lane * 4 + 256 * i, 64u * NG - 4);
        stream_word_to_lds(at + S::kKeyParams + h * S::kParams + 256 * i, offset, key_params, false);
        stream_word_to_lds(at + S::kValueParams + h * S::kParams + 256 * i, offset, value_params, false);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kStages; ++i)
    if (i < mine) ask(i, i);

  // ---- queries as operands.  x * 2^e has its row's largest magnitude in [2^5, 2^6) (f32 rows: times the scale's
  // fraction, so that their scale is a power of two).  Codes enter the matrix cores as they are masked out of a word: the
  // fp16 subnormals u 2^-24 and 16 u 2^-24, exact; their queries are x 2^(e+8) and x 2^(e+4).  A group's sum of products
  // is then 2^(e-16) times its own; steps multiply it in f32, and the minima meet the group's sum of queries (fp16 hi +
  // lo: 22 bits) in an instruction of their own.
  half8_t qh[kSteps], ql[kF32 ? kSteps : 1], qs_h, qs_l;
  float scale;
  {
    float most = 0.f;
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[st][i] = live ? x[st][i] : 0.f;
        most = fmaxf(most, fabsf(x[st][i]));
      }
    most = quarters_max(most);
    const int e = normal_power(most, a.scale);
    scale = kF32 ? ldexpf(1.0f, __builtin_amdgcn_frexp_expf(a.scale) + 2 - e) : ldexpf(a.scale, 16 - e);
    float sums[NG] = {};
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float z = kF32 ? ldexpf(x[st][i], e) * a.fraction : ldexpf(x[st][i], e);
        const float y = z * (!kF32 && (i & 2) ? 16.0f : 256.0f);   // elements 2, 3, 6, 7 lie four bits up
        qh[st][i] = (_Float16)y;
        if constexpr (kF32) ql[st][i] = (_Float16)(y - (float)qh[st][i]);
        sum += z;
      }
      sums[st / kPerGroup] += quarters_sum(sum);
    }
#pragma unroll
    for (int g = 0; g < 8; ++g) {   // the groups along the contracted index, in lanes c = 0
      const float y = c == 0 && g < NG ? sums[g < NG ? g : 0] : 0.f;
      qs_h[g] = (_Float16)y;
      qs_l[g] = (_Float16)(y - (float)qs_h[g]);
    }
  }

  float4_t acc[kColumns][kOuts] = {}, base[kF32 ? kColumns : 1] = {};
  float top = -INFINITY, sum = 0.f;
  bool lost = false;   // a page outside the cache was seen

  auto consume = [&](int32_t index, uint32_t stage, bool more) {
    const int32_t column0 = (mine0 + index * kWaves) * kTile;
    const uint8_t* at = ring + stage * S::kBytes;
    uint32_t k[2][kSteps], own[2][NG], theirs[2][4 * NG];
    uint4 v[2][kColumns], vp[2][kColumns];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < S::kParts; ++i) {
        const uint8_t* piece = at + S::kKeys + (h * S::kParts + i) * 1024 + lane * 16;
        if constexpr (D == 64) {
          const uint2 w = *reinterpret_cast<const uint2*>(piece + (c & 1) * 8);
          k[h][0] = w.x; k[h][1] = w.y;
        } else {
          const uint4 w = *reinterpret_cast<const uint4*>(piece);
          k[h][4 * i] = w.x; k[h][4 * i + 1] = w.y; k[h][4 * i + 2] = w.z; k[h][4 * i + 3] = w.w;
        }
        v[h][i] = *reinterpret_cast<const uint4*>(at + S::kValues + (h * S::kParts + i) * 1024 + lane * 16);
        vp[h][i] = *reinterpret_cast<const uint4*>(at + S::kValueParams + h * S::kParams + c * (NG * 16) +
                                                   (column_of_lane + 16 * i) * 8 * NG / D * 16);
      }
      const uint8_t* params = at + S::kKeyParams + h * S::kParams;
      load_words(params + m * (NG * 4), own[h]);
      load_words(params + c * (NG * 16), theirs[h]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read before the stage is filled again
    const bool bad[2] = {(bad_halves >> (2 * stage) & 1) != 0, (bad_halves >> (2 * stage) & 2) != 0};
    if (more) ask(index + kStages, stage);

    // some row does not see some column, or a page is bad
    const bool edge = column0 < kv4_first_column(last_row, a.window) || column0 + kTile - 1 > first_row || bad[0] || bad[1];
    if (edge) {
      lost = lost || bad[0] || bad[1];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (bad[h]) {
#pragma unroll
          for (int g = 0; g < 4 * NG; ++g) theirs[h][g] = 0x7e007e00u;
        }
#pragma unroll
        for (int i = 0; i < kColumns; ++i) {
          uint32_t w[4] = {vp[h][i].x, vp[h][i].y, vp[h][i].z, vp[h][i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {   // columns that no row sees hold anything: 0 times it has to be 0
            const int32_t column = column0 + 16 * h + 4 * (int32_t)c + j;
            const uint32_t keep = column >= low && column <= high && !bad[h] ? 0xffffffffu : 0xffff0000u >> (16 * (j & 1));
            w[j / 2] &= keep;
            w[2 + j / 2] &= keep;
          }
          vp[h][i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }

    float4_t sc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      half8_t minima = {};
#pragma unroll
      for (int g = 0; g < NG; ++g) minima[g] = half2_of(own[h][g]).y;   // (lanes c > 0: times 0)
      float4_t total = {};
      if constexpr (kF32) {   // step * 8 + minimum = hi + lo
        half8_t rest = {};
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float x = scaled(own[h][g], 8.0f, (float)minima[g]);
          minima[g] = (_Float16)x;
          rest[g] = less(x, minima[g]);
        }
        total = __builtin_amdgcn_mfma_f32_16x16x32_f16(rest, qs_h, total, 0, 0, 0);
      }
      total = __builtin_amdgcn_mfma_f32_16x16x32_f16(minima, qs_l, total, 0, 0, 0);
      total = __builtin_amdgcn_mfma_f32_16x16x32_f16(minima, qs_h, total, 0, 0, 0);
      total *= kF32 ? 0x1p-2f : 0x1p-16f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float4_t part = {};
#pragma unroll
        for (int st = g * kPerGroup; st < (g + 1) * kPerGroup; ++st) {
          const uint32_t word = k[h][st], upper = word >> 8;
          half2_t u[4] = {half2_of(word & 0x000F000Fu), half2_of(word & 0x00F000F0u), half2_of(upper & 0x000F000Fu),
                          half2_of(upper & 0x00F000F0u)};
          if constexpr (kF32) {
            // (u - 8) / 1024: the matrix cores drop low bits of sums with subnormal numbers, and sums around zero
            // lose less to the minima's
            const half2_t low2 = {(_Float16)16384.0f, (_Float16)16384.0f}, high2 = {(_Float16)1024.0f, (_Float16)1024.0f};
            const half2_t middle = {(_Float16)-0.0078125f, (_Float16)-0.0078125f};
            u[0] = __builtin_elementwise_fma(u[0], low2, middle);
            u[1] = __builtin_elementwise_fma(u[1], high2, middle);
            u[2] = __builtin_elementwise_fma(u[2], low2, middle);
            u[3] = __builtin_elementwise_fma(u[3], high2, middle);
          }
          const half8_t codes = join8(u[0], u[1], u[2], u[3]);
          if constexpr (kF32) part = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, ql[st], part, 0, 0, 0);
          part = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, qh[st], part, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) total[r] = scaled(theirs[h][r * NG + g], part[r], total[r]);
      }
      sc[h] = total;
    }
    // ---- softmax: lane (m, c) has columns 4 c .. 4 c + 3 of each half.  (fp16 rows: all products with the scale are
    // rounded as the maximum is.  In one mixed operation with the shift, a large one's rounding would be the weight's: up
    // to 2^1 at 2^24, and more than fp16 has room for from 2^26 on.)
    if constexpr (!kF32) {
      sc[0] *= scale;
      sc[1] *= scale;
    }
    const float factor = kF32 ? scale : 1.0f;
    if (edge) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int32_t column = column0 + 16 * h + 4 * (int32_t)c + r;
          if (column < from || column > position) sc[h][r] = -INFINITY;
        }
    }
    float here = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                       fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
    here = quarters_max(here) * factor;
    // The sums are brought to a new maximum where one has grown by more than 2^4: weights, with the 2^10 of their shift,
    // are at most 2^14.
    if (__any(here - top > 4.0f)) {   // (not top + 4: past 2^26 it rounds to top + 8)
      const float now = fmaxf(here, top);
      const float keep = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(shift_of(top) - shift_of(now));
      top = now;
      sum *= keep;
#pragma unroll
      for (int i = 0; i < kColumns; ++i) {
        if constexpr (kF32) base[i] *= keep;
#pragma unroll
        for (int f = 0; f < kOuts; ++f) acc[i][f] *= keep;
      }
    }
    const float shift = top == -INFINITY ? 0.f : shift_of(top);
    half8_t ph, pl;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float2_t p = {__builtin_amdgcn_exp2f(fmaf(sc[j / 4][j % 4], factor, -shift)),
                          __builtin_amdgcn_exp2f(fmaf(sc[j / 4][j % 4 + 1], factor, -shift))};
      const half2_t hi = rounded2(p);
      sum += p[0] + p[1];
      ph[j] = hi.x;
      ph[j + 1] = hi.y;
      pl[j] = less(p[0], hi.x);
      pl[j + 1] = less(p[1], hi.y);
    }

    // ---- values: lane (i, c) has rows 4 c .. 4 c + 3 of each half, the same order as the weights
#pragma unroll
    for (int i = 0; i < kColumns; ++i) {
      half2_t step[4], least[4];   // of rows (0, 1), (2, 3) of each half
      step[0] = half2_of(vp[0][i].x); step[1] = half2_of(vp[0][i].y);
      step[2] = half2_of(vp[1][i].x); step[3] = half2_of(vp[1][i].y);
      least[0] = half2_of(vp[0][i].z); least[1] = half2_of(vp[0][i].w);
      least[2] = half2_of(vp[1][i].z); least[3] = half2_of(vp[1][i].w);
      half8_t fix = {};
      bool any_fix = false;
      if (edge) {
        // a row that does not see a column of no numbers must not meet it as 0 * NaN: the column enters as 0
        // and the rows that do see it are marked afterwards
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool sound = fabsf((float)step[j][e]) < INFINITY && fabsf((float)least[j][e]) < INFINITY;
            fix[2 * j + e] = sound ? (_Float16)0.0f : (_Float16)1.0f;
            if (!sound) step[j][e] = least[j][e] = (_Float16)0.0f;
            any_fix = any_fix || !sound;
          }
        }
      }
      const uint32_t words[8] = {v[0][i].x, v[0][i].y, v[0][i].z, v[0][i].w,
                                 v[1][i].x, v[1][i].y, v[1][i].z, v[1][i].w};
#pragma unroll
      for (int b = 0; b < kOuts / 2; ++b) {
        const uint32_t byte = D == 64 ? b + (m >> 3) * 2 : b;
        const uint32_t select = byte | 0x0c000c00u | (4 + byte) << 16;
        half2_t lo2[4], hi2[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x = __builtin_amdgcn_perm(words[2 * j + 1], words[2 * j], select);
          // (f32 rows: sums around zero, beside which the minima's are small; a mean of many values is far below 8
          // steps)
          lo2[j] = low_codes<kF32 ? 8 : 0>(x);
          hi2[j] = high_codes<kF32 ? 8 : 0>(x);
        }
        if constexpr (!kF32) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            lo2[j] = __builtin_elementwise_fma(lo2[j], step[j], least[j]);
            hi2[j] = __builtin_elementwise_fma(hi2[j], step[j], least[j]);
          }
          const half8_t lo8 = join8(lo2[0], lo2[1], lo2[2], lo2[3]), hi8 = join8(hi2[0], hi2[1], hi2[2], hi2[3]);
          acc[i][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo8, pl, acc[i][2 * b], 0, 0, 0);
          acc[i][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo8, ph, acc[i][2 * b], 0, 0, 0);
          acc[i][2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi8, pl, acc[i][2 * b + 1], 0, 0, 0);
          acc[i][2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi8, ph, acc[i][2 * b + 1], 0, 0, 0);
        } else {
          half2_t rest[4];
          auto add = [&](half2_t(&u)[4], float4_t& to) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const half2_t whole = u[j] * step[j];
              rest[j] = __builtin_elementwise_fma(u[j], step[j], -whole);
              u[j] = whole;
            }
            const half8_t hi = join8(u[0], u[1], u[2], u[3]);
            to = __builtin_amdgcn_mfma_f32_16x16x32_f16(join8(rest[0], rest[1], rest[2], rest[3]), ph, to, 0, 0, 0);
            to = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, pl, to, 0, 0, 0);
            to = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, ph, to, 0, 0, 0);
          };
          add(lo2, acc[i][2 * b]);
          add(hi2, acc[i][2 * b + 1]);
        }
      }
      if constexpr (kF32) {
        half8_t minima, rest2;   // step * 8 + minimum = hi + lo
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = fmaf((float)step[j / 2][j % 2], 8.0f, (float)least[j / 2][j % 2]);
          minima[j] = (_Float16)x;
          rest2[j] = less(x, minima[j]);
        }
        base[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rest2, ph, base[i], 0, 0, 0);
        base[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(minima, pl, base[i], 0, 0, 0);
        base[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(minima, ph, base[i], 0, 0, 0);
      }
      if (edge && __any(any_fix)) {
        half8_t sees;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int32_t column = column0 + 16 * (j / 4) + 4 * (int32_t)c + j % 4;
          sees[j] = column < from || column > position ? (_Float16)0.0f : (_Float16)1.0f;
        }
        const float4_t hits = __builtin_amdgcn_mfma_f32_16x16x32_f16(fix, sees, float4_t{}, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (hits[r] > 0.f)
#pragma unroll
            for (int f = 0; f < kOuts; ++f) acc[i][f][r] = __builtin_nanf("");
      }
    }
  };

  for (int32_t i = 0; i < mine; ++i) {
    static_assert(kStages == 2, "one tile asked for behind this one, or none");
    if (i + 1 < mine) wait_vm<S::kLoads>();
    else wait_vm<0>();
    consume(i, (uint32_t)i % kStages, i + kStages < mine);
  }
  if (lost && fault && lane == 0) *fault = 1u;
  sum = quarters_sum(sum);

  // ---- the waves' states become one, in order
  __syncthreads();   // (every wave is through its ring)
  float* s_acc = reinterpret_cast<float*>(s_ring);
  if (c == 0) {
    s_max[wave][m] = shift_of(top);
    s_sum[wave][m] = sum;
  }
  if (live) {
    float* row = s_acc + (wave * a.partial_rows + m) * kStride;
#pragma unroll
    for (int i = 0; i < kColumns; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t n = 4 * c + r;
        const uint32_t d = D == 64 ? 8 * (n & 7) + 4 * (n >> 3) : 8 * (n + 16 * i);
#pragma unroll
        for (int f = 0; f < kOuts; f += 4) {
          float4_t o = {acc[i][f][r], acc[i][f + 1][r], acc[i][f + 2][r], acc[i][f + 3][r]};
          if constexpr (kF32) o += base[i][r];
          *reinterpret_cast<float4_t*>(row + d + f) = o;
        }
      }
  }
  __syncthreads();
  // a part: partial_rows x D sums, then (max, sum) of each row
  const size_t part_size = (size_t)a.partial_rows * (D + 2);
  float* const parts = a.partials + (size_t)w.unit * a.max_splits * part_size;
  float* const part = parts + w.split * part_size;
  for (uint32_t e = 4 * tid; e < count * D; e += 4 * kThreads) {
    const uint32_t row = e / D, d = e % D;
    float most = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) most = fmaxf(most, s_max[w][row]);
    const float ref = most == -INFINITY ? 0.f : most;
    float4_t total = {};
    float weight = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float k = __builtin_amdgcn_exp2f(s_max[w][row] - ref);
      const float4_t x = *reinterpret_cast<const float4_t*>(s_acc + (w * a.partial_rows + row) * kStride + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) total[i] = fmaf(k, x[i], total[i]);
      weight = fmaf(k, s_sum[w][row], weight);
    }
    if (w.nsplit == 1) {
      store4(out + row_at(a, w, row, D) + d, total / weight);
    } else {
      publish2(part + e, float2_t{total[0], total[1]});
      publish2(part + e + 2, float2_t{total[2], total[3]});
      if (d == 0) publish2(part + a.partial_rows * D + 2 * row, float2_t{most, weight});
    }
  }
  if (w.nsplit > 1) join_parts<XT, D, kThreads>(a, w, out);
}

// How the columns of a launch of kv4_decode_kernel are dealt.
struct DecodePlan {
  uint32_t waves = 0, row_tiles = 0, units = 0, max_splits = 0, partial_rows = 0, least = 0;
  float share_of_work = 0;
  size_t bytes = 0;
};
// Waves of a workgroup.  With eight a CU has one workgroup, two waves a SIMD, and as few parts to join as can be.  With
// four it has two or three, and one's first loads and last sums run beside another's tiles, which pays where many
// sequences' pieces are unequal or more than the CUs (us, eight / four, 8 kv heads x 4, D 128, fp16: 16 sequences of
// 128 to 4096 columns 26.3 / 23.7, 32 of them 43 / 33, 128 of 300 28 / 18, 128 of 2000 90 / 67, 16 of 4000 31 / 26; but
// 131000 columns 38.0 / 47.7, 128 rows of 8192 68 / 84), or where all pieces together are few (one sequence of 700 or
// 4096 columns 10.6 / 9.2, 11.0 / 9.6).
constexpr uint32_t kFewWaves = 4, kManyWaves = 8;
constexpr uint32_t kManyUnits = 96, kManyGroups = kKv4Groups * 3 / 2;
constexpr uint32_t kMostGroups = 2048;   // in a grid, those without a split among them
constexpr uint32_t kMostSplits = 64;
static_assert(kMostGroups <= kTicketSlots, "a counter a unit");
DecodePlan plan_decode(const Kv4Shape& s, uint32_t max_columns, uint64_t pairs) {
  DecodePlan p;
  const uint64_t row_tiles = (pairs + kRows - 1) / kRows, units = (uint64_t)s.nseq * s.kv_heads * row_tiles;
  p.row_tiles = (uint32_t)row_tiles;
  p.partial_rows = pairs < kRows ? (uint32_t)pairs : kRows;
  p.units = (uint32_t)(units < 0xffffffffu ? units : 0xffffffffu);
  const uint64_t tiles = ((uint64_t)max_columns + kTile - 1) / kTile + 1;
  const bool many = s.depth < 256 && (uint64_t)s.nseq * s.kv_heads >= kManyUnits;
  const bool small = tiles > 2 * kManyWaves + 1 && units * tiles <= 2 * kManyWaves * kKv4Groups;
  p.waves = s.depth == 256 || many || small ? kFewWaves : kManyWaves;
  p.least = 2 * (many ? kManyWaves : p.waves);   // two a wave: joining two parts costs about as much as a tile more
  const uint64_t most = (tiles + p.least - 1) / p.least;
  uint64_t splits = units ? kMostGroups / units : 1;
  splits = splits > kMostSplits ? kMostSplits : splits;
  splits = splits > most ? most : splits;
  p.max_splits = splits < 1 ? 1 : (uint32_t)splits;   // (with more units than kMostGroups, and so than counters: one)
  p.share_of_work = (float)s.kv_heads / (many ? kManyGroups : kKv4Groups);
  p.bytes = splits > 1 ? (size_t)units * splits * p.partial_rows * (s.depth + 2) * sizeof(float) : 0;
  return p;
}
// Which kernel has which sequences.  kv4_decode_kernel takes blocks of 16 (row, head) pairs and reads the columns again
// for each, kv4_chunk_kernel up to 256 of them with one turn of the codes, which pays where blocks of 16 are four times
// the CUs, or twice over long columns (us, decode / chunk, 1024 and 8192 columns; 8 kv heads x 4, D 128, fp16: 128 rows
// 17 / 40 and 71 / 76; 256 rows 29 / 40 and 123 / 83, of 2048 columns 46 / 47; 512 rows 46 / 36 and 229 / 118; eight
// sequences of 64 rows 53 / 38 and 234 / 121; 4 kv heads x 4, D 256: 512 rows 42 / 52 and 233 / 237, eight sequences of
// 128 86 / 73 and 464 / 441; eight of 128 rows of 128 columns, D 128 42 / 21, D 256 33 / 28).  Sequences of up to 64 pairs
// fill a quarter of its workgroup, however many they are (64 sequences of 40 pairs, D 128, 128, 1024 and 4096 columns: 19 /
// 26, 54 / 94, 173 / 328; of 64 pairs 23 / 27, 70 / 95, 227 / 329; of up to 72, 32 of them, 14 / 23, 39 / 71, 116 / 172; of
// up to 128 23 / 22, 65 / 68, 201 / 171; D 256, 64 of 64 pairs 37 / 26, 106 / 115, 313 / 418).
// A step may hold both kinds: sequences of up to kFewPairs pairs then stay with the decode kernel, in a launch of its
// own.
constexpr uint64_t kFewPairs = 32, kManyPairs = 64;
constexpr uint32_t kLongColumns = 2048;
struct AttentionPlan {
  bool few = true, many = false;   // which launches there are
  DecodePlan decode;
  size_t bytes = 0;
};
AttentionPlan plan_attention(const Kv4Shape& s, uint32_t max_columns) {
  AttentionPlan p;
  const uint32_t rows = kv4_rows(s.max_query, s.total_rows);
  const uint64_t pairs = (uint64_t)rows * (s.heads / s.kv_heads);
  const uint64_t blocks = (uint64_t)s.nseq * s.kv_heads * ((pairs + kRows - 1) / kRows);
  p.many = pairs > kManyPairs &&
           blocks >= (s.depth < 256 && max_columns >= kLongColumns ? 2u : 4u) * kKv4Groups;
  p.few = !p.many || (s.nseq > 1 && s.total_rows < (uint64_t)s.nseq * rows);
  if (p.few) p.decode = plan_decode(s, max_columns, p.many ? kFewPairs : pairs);
  p.bytes = p.decode.bytes;
  if (p.many) {
    const size_t chunk = kv4_chunk_workspace(s.depth, max_columns);
    if (chunk > p.bytes) p.bytes = chunk;
  }
  return p;
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
  *bytes = plan_attention(shape, max_columns).bytes;
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
  const float scale = half_scale * half_scale * kLog2e;
  KRM_REQUIRE(ctx, std::isnormal(scale), "krm_kv4_attention: half_scale");
  KRM_REQUIRE(ctx, max_columns <= 0x7fffffffu && (max_columns >= kv4_rows(max_query, total_rows)),
              "krm_kv4_attention: max_columns %u beside max_query %u", max_columns, max_query);
  if (nseq == 0 || total_rows == 0) return KRM_OK;
  KRM_REQUIRE(ctx, q && cache && page_table_i32 && cu_rows_i32 && lens_i32 && out, "krm_kv4_attention: NULL buffer");
  KRM_REQUIRE(ctx, aligned(q, 16) && aligned(out, 16) && aligned(cache, 16) && aligned(page_table_i32, 4) &&
                       aligned(cu_rows_i32, 4) && aligned(lens_i32, 4) && aligned(fault_u32, 4) &&
                       aligned(workspace, 16),
              "krm_kv4_attention: misaligned buffer (rows, cache and workspace: 16 bytes)");
  KRM_REQUIRE(ctx, q != out, "krm_kv4_attention: out is q");
  const AttentionPlan plan = plan_attention(shape, max_columns);
  const uint32_t share = heads / kv_heads;
  const uint64_t blocks = (uint64_t)nseq * kv_heads * ((uint64_t)kv4_rows(max_query, total_rows) * share / kRows + 1);
  KRM_REQUIRE(ctx, blocks <= 0x7fffffu && (uint64_t)kv4_rows(max_query, total_rows) * share <= kKv4MostPairs,
              "krm_kv4_attention: %u sequences of %u rows of %u heads are more than one call takes", nseq, max_query, heads);
  if (plan.bytes) {
    KRM_REQUIRE(ctx, workspace && workspace_bytes >= plan.bytes, "krm_kv4_attention: workspace of %zu bytes, %zu needed",
                workspace ? workspace_bytes : (size_t)0, plan.bytes);
    KRM_TRY(needs_serial_scratch(ctx, "krm_kv4_attention"));
  }
  DecodeAttention a;
  a.layout = {depth, group, page_rows, kv_heads};
  a.limits = {total_rows, max_query, max_columns, table_stride, page_rows};
  a.nseq = nseq;
  a.heads = heads;
  a.pages = pages;
  a.window = window;
  a.share = share;
  a.share_inverse = 1.0f / share;
  int power;
  a.scale = scale;
  a.fraction = std::frexp(scale, &power);
  a.partials = ptr<float>(workspace);
  a.tickets = ctx->tickets;
  if (plan.many) {
    a.least_pairs = plan.few ? (uint32_t)kFewPairs + 1 : 0;
    a.most_pairs = 0xffffffffu;
    KRM_TRY(launch_kv4_chunk(ctx, a, {q, cache, page_table_i32, cu_rows_i32, lens_i32, out, fault_u32}, io_dtype));
    if (!plan.few) return KRM_OK;
  }
  a.least_pairs = 0;
  a.most_pairs = plan.many ? (uint32_t)kFewPairs : 0xffffffffu;
  a.row_tiles = plan.decode.row_tiles;
  a.row_tiles_inverse = 1.0f / a.row_tiles;
  a.of_sequence_inverse = 1.0f / ((float)kv_heads * a.row_tiles);
  a.max_splits = plan.decode.max_splits;
  a.partial_rows = plan.decode.partial_rows;
  a.least = plan.decode.least;
  a.share_of_work = plan.decode.share_of_work;
  const dim3 grid(plan.decode.units, a.max_splits);
  const uint32_t waves = plan.decode.waves;
  const size_t joined = (size_t)waves * a.partial_rows * (depth + 4) * sizeof(float);
#define KRM_ATTENTION(XT, D, NG, WAVES)                                                                    \
  const size_t ring = (size_t)WAVES * kStages * Stage<D, NG>::kBytes, lds = ring > joined ? ring : joined; \
  kv4_decode_kernel<XT, D, NG, WAVES><<<grid, dim3(WAVES * kWave), lds, ctx->stream>>>(                    \
      ptr<const XT>(q), ptr<const uint8_t>(cache), ptr<const int32_t>(page_table_i32),                     \
      ptr<const int32_t>(cu_rows_i32), ptr<const int32_t>(lens_i32), ptr<XT>(out), ptr<uint32_t>(fault_u32), a)
#define KRM_ATTENTION_W(XT, D, NG)                                           \
  {                                                                          \
    if (waves == kManyWaves) { KRM_ATTENTION(XT, D, NG, kManyWaves); }       \
    else { KRM_ATTENTION(XT, D, NG, kFewWaves); }                            \
    break;                                                                   \
  }
#define KRM_ATTENTION_D(XT)                                  \
  switch (depth * 16 + depth / group) {                      \
    case 64 * 16 + 1: KRM_ATTENTION_W(XT, 64, 1)             \
    case 64 * 16 + 2: KRM_ATTENTION_W(XT, 64, 2)             \
    case 128 * 16 + 1: KRM_ATTENTION_W(XT, 128, 1)           \
    case 128 * 16 + 2: KRM_ATTENTION_W(XT, 128, 2)           \
    case 128 * 16 + 4: KRM_ATTENTION_W(XT, 128, 4)           \
    case 256 * 16 + 2: { KRM_ATTENTION(XT, 256, 2, kFewWaves); break; } \
    case 256 * 16 + 4: { KRM_ATTENTION(XT, 256, 4, kFewWaves); break; } \
    default: { KRM_ATTENTION(XT, 256, 8, kFewWaves); }       \
  }
  if (io_dtype == KRM_F32) { KRM_ATTENTION_D(float) } else { KRM_ATTENTION_D(__half) }
#undef KRM_ATTENTION_D
#undef KRM_ATTENTION_W
#undef KRM_ATTENTION
  return launched(ctx, "kv4_decode_kernel");
}

}  // extern "C"
