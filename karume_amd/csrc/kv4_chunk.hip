// Attention of many rows over the pages of the 4-bit K/V cache: kv4_attention.hip's operator where a sequence has
// chunks of rows.
//
// What bounds it is arithmetic, so a tile's codes are turned into fp16 once for all rows of a workgroup: it has kPairs
// (row, head) pairs, 32 a wave, and for each tile of columns half of the waves make keys and half values, in LDS, two
// tiles by turns; every wave then multiplies its rows with all of it.
//   keys    k = hi + lo, two fp16 planes (22 bits): the products with fp16 queries are off by no more than f32 sums;
//           f32 queries are hi + lo too
//   weights p = hi + lo; values rounded to fp16 once (f32 rows: hi + lo), as kv4_attention.hip does and for its reason
// Both hi and lo planes double the products: four prompts of 512 rows behind 200 to 4100 columns (8 kv heads x 4, D 128,
// fp16; 80 GFLOP without them) take 170 to 180 us, 143 of them at the rate of a large product; matrix and vector
// instructions each have about half of a SIMD's time and hardly overlap.
// The scores are formed as K Q^T: a lane has one pair's scores, so its maximum and sum stay in the lane, and the weights
// leave the product in the order in which the next one takes them.
#include "kv4_attention.h"
#include "kv4_marks.h"
#include "rows8.h"

using namespace krm;

namespace {

typedef float float16_t __attribute__((ext_vector_type(16)));

__device__ inline float16_t product(half8_t a, half8_t b, float16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// The same of the lane 32 apart, joined.
template <typename F>
__device__ inline float across_halves(float x, F join) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return join(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// The 16-byte chunks of a row of keys in LDS are exchanged by its number (chunk ^ this), so that 16 rows read at one
// chunk, and four (a depth of 64: eight) rows written at four (two) chunks, lie on different banks.
template <int D>
__device__ inline uint32_t exchanged(uint32_t row) {
  const uint32_t x = row >> 1;
  return D == 64 ? (x & 1) | (x & 2) << 1 | (x & 4) >> 1 : (row & 3) << 2 | (row >> 2 & 3);
}

template <typename XT, int D>
struct Chunk {
  static constexpr bool kF32 = sizeof(XT) == 4;
  static constexpr int kWaves = D == 256 ? 4 : 8;
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kPairs = kWaves * 32;
  static constexpr int kColumns = kWaves * 8;        // of a tile: 16 for each wave that makes keys
  static constexpr int kBlocks = kColumns / 16;
  static constexpr int kKeyPlanes = 2, kValuePlanes = kF32 ? 2 : 1;
  static constexpr uint32_t kPlane = kColumns * D * 2;
  static constexpr uint32_t kTileBytes = (kKeyPlanes + kValuePlanes) * kPlane;
};

// The inclusive sums over the lanes.
__device__ inline uint32_t wave_through(uint32_t x) {
#define KRM_THROUGH(CTRL, ROWS) x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false)
  KRM_THROUGH(0x111, 0xf);   // row_shr:1
  KRM_THROUGH(0x112, 0xf);
  KRM_THROUGH(0x114, 0xf);
  KRM_THROUGH(0x118, 0xf);
  KRM_THROUGH(0x142, 0xa);   // row_bcast:15
  KRM_THROUGH(0x143, 0xc);   // row_bcast:31
#undef KRM_THROUGH
  return x;
}

// The thread's number.  (What hangs on it alone is found anew, and not kept beside all of a kernel's work.)
__device__ inline uint32_t thread_id() {
  uint32_t tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  return tid;
}
// Values that are the same in every lane.
__device__ inline uint32_t scalar(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
template <typename T>
__device__ inline T scalars(const T& from) {
  struct Words {
    uint32_t w[sizeof(T) / 4];
  };
  Words x = __builtin_bit_cast(Words, from);
#pragma unroll
  for (uint32_t i = 0; i < sizeof(T) / 4; ++i) x.w[i] = scalar(x.w[i]);
  return __builtin_bit_cast(T, x);
}

// How blocks of kPairs (row, head) pairs are dealt to kKv4Groups workgroups, one a CU.  Every wave reads the step's
// words itself, 64 sequences at a time.
// A launch's work is one long row of units of 2^grain columns: for each sequence, kv head and block those that its rows
// see. Each workgroup has an equal run of it, which may end one block's columns and begin another's.  (A grid of blocks
// times equal splits: four prompts of 512 rows behind 200 to 4100 columns 190 us, so 178; three of 512 of 2048 104 us,
// so 96.) Beginning a block costs a workgroup as much as kBegin tiles, which its work counts, and joining a block's
// parts several times that, so that a run's end less than kSnap tiles away from a block's is moved there (2048 rows of
// 2048 columns, 4 kv heads x 8, D 64, f32: without both 119.9 us, so 76.5).
// If whole blocks, or equal parts of them, can be dealt one a workgroup, and none has kDearer tiles more than a run,
// they are (512 rows of 1024 columns, 8 kv heads x 4, D 128: runs 44.6 us, parts 38.3; since 36.4).
constexpr uint32_t kBegin = 2, kSnap = 3, kDearer = 8;
struct ChunkAttention : Kv4Attention {
  uint32_t grain;
  uint32_t least;   // units, at least, of a run
};
struct ChunkWork : Work {
  uint32_t refused;                   // the sequence's words break the limits
  int32_t cu1;
  uint32_t first_group, parts, part;  // workgroups that have some of these pairs, and which of them this is
};
// Where the parts lie: the first part of some pairs is its workgroup's last piece, any other one the first.
__device__ inline uint32_t part_slot(const ChunkWork& w, uint32_t part) {
  return 2 * (w.first_group + part) + (part == 0);
}

// (in LDS: a tile's loop has no registers for it)
template <int kWaves, int kPairs, int kTile>
struct Deal {
  struct Sequence {
    uint32_t through;   // work up to the sequence's end
    Kv4Blocks blocks;
    int32_t cu0, cu1, len;
    uint32_t ok;
  };
  struct Run : Kv4Run {
    uint32_t base, before;   // of the sequences at hand: the first one, and the work before them
  };
  Sequence sequences[kWave];   // at hand (every wave writes all of them, the same words)
  Run runs[kWaves];            // each wave's, the same

  // neighbouring runs, which may join parts, lie on one XCD
  __device__ static inline uint32_t group() { return blockIdx.x % 8 * (kKv4Groups / 8) + blockIdx.x / 8; }
  // A lane's sequence of the 64 from `first` on.
  __device__ static inline Sequence read(const ChunkAttention& a, const int32_t* __restrict__ cu_rows,
                                         const int32_t* __restrict__ lens, uint32_t begin, uint32_t first) {
    const uint32_t seq = first + thread_id() % kWave, i = min(seq, a.nseq - 1);
    Sequence s;
    s.cu0 = cu_rows[i];
    s.cu1 = cu_rows[i + 1];
    s.len = lens[i];
    s.ok = kv4_sequence(s.cu0, s.cu1, s.len, a.limits).ok;
    s.blocks = {0, 1, 0};
    if (seq < a.nseq && s.cu0 >= 0 && s.cu1 > s.cu0 && (uint32_t)s.cu1 <= a.limits.total_rows) {
      const uint64_t pairs = (uint64_t)(uint32_t)(s.cu1 - s.cu0) * a.share;
      if (pairs >= a.least_pairs && pairs <= a.most_pairs) {
        s.blocks.blocks = 1;   // (all rows of a refused sequence)
        if (s.ok) s.blocks = kv4_blocks(pairs, a.share, kPairs, s.len, a.window, a.grain);
        s.blocks.first += begin;
      }
    }
    s.through = wave_through(a.layout.kv_heads * s.blocks.all());
    return s;
  }
  __device__ static inline uint32_t last_lane(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_readlane((int)x, kWave - 1);
  }

  __device__ inline void start(const ChunkAttention& a, const int32_t* __restrict__ cu_rows,
                               const int32_t* __restrict__ lens, uint32_t* __restrict__ fault) {
    Run r;
    r.begin = a.nseq > kWave ? kBegin * kTile >> a.grain : 0;
    r.snap = max(kSnap * kTile >> a.grain, 1u);
    r.even = 0;
    uint32_t total = 0;
    Sequence s;
    for (uint32_t first = 0; first < a.nseq; first += kWave) {
      s = read(a, cu_rows, lens, r.begin, first);
      total += last_lane(s.through);
      if (fault && blockIdx.x == 0 && !s.ok) *fault = 1u;
    }
    r.per = max((total + kKv4Groups - 1) / kKv4Groups, a.least);
    if (a.nseq > kWave) {
      s = read(a, cu_rows, lens, r.begin, 0);
    } else {
      const uint32_t widest = s.blocks.blocks ? s.blocks.of(s.blocks.blocks - 1) : 0;
      for (uint32_t more = 0; more <= kDearer && !r.even; ++more) {
        const uint32_t most = r.per + (more * kTile >> a.grain), parts = (widest + most - 1) / most;
        const uint32_t to = wave_through(a.layout.kv_heads * s.blocks.blocks * parts);
        if (last_lane(to) <= kKv4Groups) {
          r.even = 1;
          s.blocks.first = parts;
          s.blocks.step = 0;
          s.through = to;
        }
      }
      if (r.even) {
        r.per = r.snap = 1;
      } else {
        r.begin = kBegin * kTile >> a.grain;
        s.blocks.first += r.begin;
        s.through = wave_through(a.layout.kv_heads * s.blocks.all());
        r.per = max((last_lane(s.through) + kKv4Groups - 1) / kKv4Groups, a.least);
      }
      total = last_lane(s.through);
    }
    sequences[thread_id() % kWave] = s;
    r.at = min(group() * r.per, total);
    r.end = min(r.at + r.per, total);
    r.base = r.before = 0;
    r.fresh = 1;
    runs[scalar(thread_id() / kWave)] = r;
  }
  // The next piece of this workgroup's run; false at its end.
  __device__ inline bool next(const ChunkAttention& a, const int32_t* __restrict__ cu_rows,
                              const int32_t* __restrict__ lens, ChunkWork& w) {
    Run& run = runs[scalar(thread_id() / kWave)];
    Run r = scalars(run);
    for (;;) {
      if (r.at >= r.end) return false;
      uint32_t through = sequences[thread_id() % kWave].through;
      while (r.at - r.before >= last_lane(through)) {
        r.before += last_lane(through);
        r.base += kWave;
        __syncthreads();
        const Sequence s = read(a, cu_rows, lens, r.begin, r.base);
        sequences[thread_id() % kWave] = s;
        through = s.through;
      }
      const uint32_t lane = (uint32_t)__builtin_ctzll(__builtin_amdgcn_ballot_w64(through > r.at - r.before));
      const Sequence& s = sequences[lane];
      const Kv4Blocks blocks = {scalar(s.blocks.blocks), scalar(s.blocks.first), scalar(s.blocks.step)};
      const uint32_t of_head = blocks.all(), start = r.before + scalar(s.through) - a.layout.kv_heads * of_head;
      w.seq = r.base + lane;
      w.kv_head = scalar((r.at - start) / of_head);
      const uint32_t head_at = start + w.kv_head * of_head, block = scalar(blocks.block_at(r.at - head_at));
      const uint32_t block_at = head_at + blocks.before(block), width = blocks.of(block);
      Kv4Cut cut;
      const Kv4Dealt dealt = kv4_cut(r, block_at, width, cut);
      if (dealt == kRunEnds) return false;
      if (dealt == kBlockSkipped) continue;
      run = r;
      w.cu0 = (int32_t)scalar((uint32_t)s.cu0);
      w.cu1 = (int32_t)scalar((uint32_t)s.cu1);
      w.refused = scalar(s.ok) == 0;
      const int32_t rows = w.cu1 - w.cu0;
      const uint32_t pair0 = block * kPairs;
      w.count = (uint32_t)min((uint64_t)kPairs, (uint64_t)(uint32_t)rows * a.share - pair0);
      w.row0 = scalar(divided(pair0, a.share, a.share_inverse));
      w.head0 = pair0 - w.row0 * a.share;
      w.first_row = (int32_t)scalar((uint32_t)s.len) - rows + (int32_t)w.row0;
      w.last_row = w.first_row + (int32_t)scalar(row_of(a, w, w.count - 1));
      w.low = kv4_first_column(w.first_row, a.window);
      w.high = w.last_row;
      const int32_t tile0 = w.low / kTile, tiles = w.high / kTile - tile0 + 1;
      w.begin = tile0 + (int32_t)scalar(kv4_tile(r, cut.from, width, tiles, a.grain, kTile));
      w.end = tile0 + (int32_t)scalar(kv4_tile(r, cut.to, width, tiles, a.grain, kTile));
      w.parts = scalar(cut.parts);
      w.first_group = scalar(cut.first);
      w.part = group() - w.first_group;
      return true;
    }
  }
};

// One piece.  `a` and `w` are in registers, and wait in LDS as s_numbers and s_work for what comes behind the tiles.
template <typename XT, int D, int NG>
__device__ __forceinline__ void chunk_piece(
    const XT* __restrict__ q, const uint8_t* __restrict__ cache, const int32_t* __restrict__ page_table,
    XT* __restrict__ out, uint32_t* __restrict__ fault, float* partials, uint32_t* tickets, const ChunkAttention& a,
    const ChunkWork& w, const ChunkAttention& s_numbers, const ChunkWork& s_work) {
  using C = Chunk<XT, D>;
  constexpr bool kF32 = C::kF32;
  constexpr int kThreads = C::kThreads, kColumns = C::kColumns, kBlocks = C::kBlocks;
  constexpr int kSteps = D / 16, kSubs = kColumns / 32, kOuts = D / 32;
  constexpr int kPieces = D <= 128 ? 1 : D / 128;    // 16-byte pieces of codes that a lane turns
  extern __shared__ __align__(16) uint8_t s_tiles[];  // [2][keys hi, keys lo, values hi (, values lo)]
  __shared__ Kv4Marks<kColumns> s_marks;              // (of tiles that some row does not see in full)

  const uint32_t tid = thread_id(), lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int32_t low = w.low, high = w.high;

  // ---- this wave's rows: lane (m = lane % 32, half)
  const uint32_t m = lane & 31, half = lane >> 5, pair = wave * 32 + m;
  const bool live = pair < w.count;
  const int32_t position = w.first_row + (int32_t)row_of(a, w, live ? pair : 0);
  const int32_t from = kv4_first_column(position, a.window);
  // columns that this wave's rows see (none: it only makes keys or values)
  const bool has_rows = wave * 32 < w.count;
  const int32_t wave_low = kv4_first_column(w.first_row + (int32_t)row_of(a, w, has_rows ? wave * 32 : 0), a.window);
  const int32_t wave_high =
      has_rows ? w.first_row + (int32_t)row_of(a, w, min(wave * 32 + 31, w.count - 1)) : wave_low - 1;
  half8_t qh[kSteps], ql[kF32 ? kSteps : 1];
  float scale = a.scale;
  asm volatile("" : "+v"(scale));
  {
    const XT* src = q + row_at(a, w, live ? pair : 0, D) + 8 * half;
    if constexpr (!kF32) {
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const half8_t x = *reinterpret_cast<const half8_t*>(src + 16 * st);
        qh[st] = live ? x : half8_t{};
      }
    } else {
      // x * 2^e * fraction = hi + lo, x * 2^e with the row's largest magnitude in [2^5, 2^6)
      float x[kSteps][8], most = 0.f;
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        load8(src + 16 * st, x[st]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[st][i] = live ? x[st][i] : 0.f;
          most = fmaxf(most, fabsf(x[st][i]));
        }
      }
      most = across_halves(most, [](float x, float y) { return fmaxf(x, y); });
      const int e = normal_power(most, scale);
      scale = ldexpf(1.0f, __builtin_amdgcn_frexp_expf(scale) - e);
#pragma unroll
      for (int st = 0; st < kSteps; ++st)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float y = ldexpf(x[st][i], e) * a.fraction;
          asm("" : "+v"(y));   // (else the product is rounded to fp16 in one step here and in two there)
          qh[st][i] = (_Float16)y;
          ql[st][i] = (_Float16)(y - (float)qh[st][i]);
        }
    }
  }

  // ---- the other work of a wave: codes of 16 columns of each tile, keys (waves below kBlocks) or values
  const bool makes_values = wave >= kBlocks;
  const uint32_t my_block = makes_values ? wave - kBlocks : wave;
  const int32_t* table = page_table + (size_t)w.seq * a.limits.table_stride;
  const uint32_t page_shift = 31 - __builtin_clz(a.layout.page_rows);
  const uint64_t page_bytes = a.layout.page();
  const uint8_t* head_base = cache + (size_t)w.kv_head * a.layout.block();
  // keys: lane (row r, piece c): words (c, .) of row r; values: lane (rows 4 b .. 4 b + 3, word column).  A depth of 64
  // has half as many pieces: lanes 32 .. 63 repeat those of 0 .. 31 and write nothing.
  const uint32_t at_lane = D == 64 ? lane & 31 : lane;
  const bool idle = D == 64 && lane >= 32;
  const uint32_t key_row = D == 64 ? at_lane / 2 : at_lane / 4, key_piece = D == 64 ? at_lane & 1 : at_lane & 3;
  constexpr uint32_t kWordColumns = D / 8;
  struct Raw {
    uint4 codes[kPieces];
    uint32_t params[NG > 4 ? NG : 4];   // keys: of the row's groups; values: 16 bytes of a piece's group
    uint4 more[kPieces > 1 ? kPieces - 1 : 1];
    uint32_t bad;
  };
  auto fetch = [&](int32_t tile) __attribute__((always_inline)) -> Raw {
    Raw r = {};
    const int32_t column = tile * kColumns + 16 * (int32_t)my_block;
    uint32_t id = 0;
    r.bad = 0;
    if (column <= high && column + 15 >= low) {   // (a block that no row sees has no page: page 0, and nothing is used)
      id = (uint32_t)table[(uint32_t)column >> page_shift];
      if (id >= a.pages) {
        r.bad = 1;
        id = 0;
      }
    }
    const uint32_t in_page = (uint32_t)column & (a.layout.page_rows - 1);
    const uint8_t* base = uniform(head_base + id * page_bytes);
    if (!makes_values) {
      const uint8_t* codes = base + in_page * (D / 2) + key_row * (D / 2);
      if constexpr (D == 64) {
        r.codes[0] = *reinterpret_cast<const uint4*>(codes + key_piece * 16);
      } else {
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
          r.codes[i] = *reinterpret_cast<const uint4*>(codes + key_piece * (D / 8) + 16 * i);
      }
      uint32_t p[NG];
      load_words(base + a.layout.key_params() + (in_page + key_row) * (NG * 4), p);
#pragma unroll
      for (int g = 0; g < NG; ++g) r.params[g] = p[g];
    } else {
      const uint8_t* codes = base + a.layout.value_codes() + in_page * (D / 2);
      const uint8_t* params = base + a.layout.value_params() + in_page * (NG * 4);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const uint32_t piece = at_lane + kWave * i, four = piece / kWordColumns, column_of = piece % kWordColumns;
        r.codes[i] = *reinterpret_cast<const uint4*>(codes + piece * 16);
        const uint4 p = *reinterpret_cast<const uint4*>(params + four * (NG * 16) + column_of * 8 * NG / D * 16);
        if (i == 0) {
          r.params[0] = p.x; r.params[1] = p.y; r.params[2] = p.z; r.params[3] = p.w;
        } else {
          r.more[i - 1] = p;
        }
      }
    }
    return r;
  };
  // Whether a tile has a column that some row does not see, or that lies on no page.
  auto tile_edge = [&](int32_t tile) {
    const int32_t column0 = tile * kColumns;
    return column0 < kv4_first_column(w.last_row, a.window) || column0 + kColumns - 1 > w.first_row;
  };
  bool lost = false;
  auto make = [&](const Raw& r, int32_t tile, uint32_t buffer) __attribute__((always_inline)) {
    uint8_t* const to = s_tiles + buffer * C::kTileBytes;
    const int32_t column0 = tile * kColumns;
    lost = lost || r.bad;
    if (!makes_values) {
      const uint32_t row = 16 * my_block + key_row;
      if (idle) return;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const uint32_t words[4] = {r.codes[i].x, r.codes[i].y, r.codes[i].z, r.codes[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // word (c, s) of the row: elements 32 s + 8 c .. + 7, chunk 4 s + c
          const int at = D == 64 ? j & 1 : 4 * i + j;                               // s
          const uint32_t c = D == 64 ? 2 * key_piece + (j >> 1) : key_piece;
          const half2_t p = half2_of(r.bad ? 0x7e007e00u : r.params[at * NG / (D / 32)]);
          const float step = (float)p.x, least = (float)p.y;
          uint32_t even = words[j] & 0x0f0f0f0fu, odd = (words[j] >> 4) & 0x0f0f0f0fu;
          asm("" : "+v"(even), "+v"(odd));   // (bytes of these, not nibbles of the word, become numbers in one step each)
          // nibble i: element 2 i, nibble 4 + i: element 2 i + 1
          const uint32_t code[8] = {even & 255, even >> 16 & 255, odd & 255, odd >> 16 & 255,
                                    even >> 8 & 255, even >> 24, odd >> 8 & 255, odd >> 24};
          half8_t hi, lo;
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float2_t x = {fmaf(step, (float)code[e], least), fmaf(step, (float)code[e + 1], least)};
            const half2_t h2 = rounded2(x);
            hi[e] = h2.x;
            hi[e + 1] = h2.y;
            lo[e] = less(x[0], h2.x);
            lo[e + 1] = less(x[1], h2.y);
          }
          const uint32_t place = row * (D * 2) + ((4 * (uint32_t)at + c) ^ exchanged<D>(row)) * 16;
          *reinterpret_cast<half8_t*>(to + place) = hi;
          *reinterpret_cast<half8_t*>(to + C::kPlane + place) = lo;
        }
      }
    } else {
      const bool edge = tile_edge(tile) || r.bad;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const uint32_t piece = at_lane + kWave * i, four = piece / kWordColumns, column_of = piece % kWordColumns;
        uint32_t p[4];
        if (i == 0) {
          p[0] = r.params[0]; p[1] = r.params[1]; p[2] = r.params[2]; p[3] = r.params[3];
        } else {
          p[0] = r.more[i - 1].x; p[1] = r.more[i - 1].y; p[2] = r.more[i - 1].z; p[3] = r.more[i - 1].w;
        }
        if (edge) {
          // columns that no row sees hold anything, and 0 times it has to be 0; a column of no numbers that some row
          // does not see enters as 0, and the rows that do see it are marked behind the product
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int32_t column = column0 + 16 * (int32_t)my_block + 4 * (int32_t)four + j;
            const uint32_t mine = 0xffffu << (16 * (j & 1));
            const bool none = column < low || column > high || r.bad;
            const half2_t s2 = half2_of(p[j / 2]), l2 = half2_of(p[2 + j / 2]);
            const bool sound = fabsf((float)s2[j & 1]) < INFINITY && fabsf((float)l2[j & 1]) < INFINITY;
            if (!none && !sound && !idle) {
              atomicOr(&s_marks.groups[buffer][column - column0], 1u << (column_of * 8 * NG / D));
              s_marks.any[buffer] = 1;
            }
            if (none || !sound) {
              p[j / 2] &= ~mine;
              p[2 + j / 2] &= ~mine;
            }
          }
        }
        if (idle) continue;
        const uint32_t words[4] = {r.codes[i].x, r.codes[i].y, r.codes[i].z, r.codes[i].w};
        // rows 4 four .. + 3 of a block of 16: the operand's lanes of `half` four & 1, elements 4 (four / 2) ..
        // (element e of word column x lies at e ^ (x & 7), so that neighbouring columns lie on different banks)
        uint8_t* const at = to + 2 * C::kPlane + ((my_block * 2 + (four & 1)) * D + 8 * column_of) * 16 + (four / 2) * 8;
        const uint32_t turn = (column_of & 7) * 16;
        if constexpr (!kF32) {
          const half2_t s01 = half2_of(p[0]), s23 = half2_of(p[1]), l01 = half2_of(p[2]), l23 = half2_of(p[3]);
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const uint32_t select = (uint32_t)b | 0x0c000c00u | (4u + b) << 16;
            const uint32_t x = __builtin_amdgcn_perm(words[1], words[0], select);
            const uint32_t y = __builtin_amdgcn_perm(words[3], words[2], select);
            const half2_t e0 = __builtin_elementwise_fma(low_codes<0>(x), s01, l01);
            const half2_t e1 = __builtin_elementwise_fma(low_codes<0>(y), s23, l23);
            const half2_t o0 = __builtin_elementwise_fma(high_codes<0>(x), s01, l01);
            const half2_t o1 = __builtin_elementwise_fma(high_codes<0>(y), s23, l23);
            *reinterpret_cast<uint2*>(at + ((2 * b) * 16 ^ turn)) =
                make_uint2(__builtin_bit_cast(uint32_t, e0), __builtin_bit_cast(uint32_t, e1));
            *reinterpret_cast<uint2*>(at + ((2 * b + 1) * 16 ^ turn)) =
                make_uint2(__builtin_bit_cast(uint32_t, o0), __builtin_bit_cast(uint32_t, o1));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            half2_t h[2], l[2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float x = fmaf((float)half2_of(p[j / 2])[j & 1], (float)(words[j] >> (4 * e) & 15u),
                                   (float)half2_of(p[2 + j / 2])[j & 1]);
              h[j / 2][j & 1] = (_Float16)x;
              l[j / 2][j & 1] = less(x, h[j / 2][j & 1]);
            }
            *reinterpret_cast<uint2*>(at + (e * 16 ^ turn)) =
                make_uint2(__builtin_bit_cast(uint32_t, h[0]), __builtin_bit_cast(uint32_t, h[1]));
            *reinterpret_cast<uint2*>(at + C::kPlane + (e * 16 ^ turn)) =
                make_uint2(__builtin_bit_cast(uint32_t, l[0]), __builtin_bit_cast(uint32_t, l[1]));
          }
        }
      }
    }
  };

  // ---- a tile's rows
  float16_t acc[kOuts] = {};
  float top = -INFINITY, sum = 0.f;
  const uint32_t key_lane = m * (D * 2);
  const uint32_t value_lane[2] = {((m & 24) | ((m & 7) ^ (m >> 3))) * 16, ((m & 24) | ((m & 7) ^ (4 + (m >> 3)))) * 16};
  auto consume = [&](int32_t tile, uint32_t buffer) __attribute__((always_inline)) {
    const int32_t column0 = tile * kColumns;
    const uint8_t* keys = s_tiles + buffer * C::kTileBytes;
    const uint8_t* values = keys + 2 * C::kPlane + half * D * 16;
    float16_t sc[kSubs];
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub) sc[sub] = float16_t{};
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const uint32_t chunk = 2 * st + half;
      half8_t hi[kSubs], lo[kSubs];
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
        const uint32_t at = sub * 32 * (D * 2) + key_lane + (chunk ^ exchanged<D>(m)) * 16;
        hi[sub] = *reinterpret_cast<const half8_t*>(keys + at);
        lo[sub] = *reinterpret_cast<const half8_t*>(keys + C::kPlane + at);
      }
      // (neighbouring products are of different sums, so that none waits for the one before it)
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) sc[sub] = product(lo[sub], qh[st], sc[sub]);
      if constexpr (kF32) {
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub) sc[sub] = product(hi[sub], ql[st], sc[sub]);
      }
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) sc[sub] = product(hi[sub], qh[st], sc[sub]);
    }
    // lane (m, half): columns 8 (r / 4) + 4 half + r % 4 of each 32
    if (tile_edge(tile)) {
      int32_t first = column0 + 4 * (int32_t)half;
      asm volatile("" : "+v"(first));   // (stays behind the branch: in every tile these are a fifth of its instructions)
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int32_t column = first + 32 * sub + 8 * (r / 4) + r % 4;
          if (column < from || column > position) sc[sub][r] = -INFINITY;
        }
    }
    float here = sc[0][0];
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
      for (int r = 0; r < 16; ++r) here = fmaxf(here, sc[sub][r]);
    here = across_halves(here, [](float x, float y) { return fmaxf(x, y); }) * scale;
    // weights may grow to 2^(4 + 10) before the sums are brought to a new maximum
    if (__any(here - top > 4.0f)) {   // (not top + 4: past 2^26 it rounds to top + 8)
      const float now = fmaxf(here, top);
      const float keep = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(shift_of(top) - shift_of(now));
      top = now;
      sum *= keep;
#pragma unroll
      for (int o = 0; o < kOuts; ++o) acc[o] *= keep;
    }
    const float shift = top == -INFINITY ? 0.f : shift_of(top);
    // fp16 rows: a product's rounding is missing from the mixed operation below, and is the weight's: up to 2^1 at 2^24,
    // and more than fp16 has room for from 2^26 on.  There all of them are rounded first, as the maximum was.
    float factor = scale;
    if constexpr (!kF32) {
      if (__any(fabsf(top) > 0x1p24f && top > -INFINITY)) {
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub) sc[sub] *= scale;
        factor = 1.0f;
      }
    }
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        half8_t ph, pl;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float2_t p = {__builtin_amdgcn_exp2f(fmaf(sc[sub][8 * ks + j], factor, -shift)),
                              __builtin_amdgcn_exp2f(fmaf(sc[sub][8 * ks + j + 1], factor, -shift))};
          const half2_t hi = rounded2(p);
          sum += p[0] + p[1];
          ph[j] = hi.x;
          ph[j + 1] = hi.y;
          pl[j] = less(p[0], hi.x);
          pl[j + 1] = less(p[1], hi.y);
        }
#pragma unroll
        for (int o = 0; o < kOuts; o += 2) {
          half8_t hi[2], lo[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint8_t* at = values + ((2 * sub + ks) * 2 * D + 32 * (o + i)) * 16 + value_lane[i];
            hi[i] = *reinterpret_cast<const half8_t*>(at);
            if constexpr (kF32) lo[i] = *reinterpret_cast<const half8_t*>(at + C::kPlane);
          }
          if constexpr (kF32) {
            acc[o] = product(lo[0], ph, acc[o]);
            acc[o + 1] = product(lo[1], ph, acc[o + 1]);
          }
          acc[o] = product(hi[0], pl, acc[o]);
          acc[o + 1] = product(hi[1], pl, acc[o + 1]);
          acc[o] = product(hi[0], ph, acc[o]);
          acc[o + 1] = product(hi[1], ph, acc[o + 1]);
        }
      }
    }
    if (s_marks.any[buffer]) {
#pragma unroll 1
      for (int i = 0; i < kColumns; ++i) {
        const uint32_t groups = s_marks.groups[buffer][i];
        const int32_t column = column0 + i;
        if (groups == 0 || column < from || column > position) continue;
#pragma unroll
        for (int o = 0; o < kOuts; ++o)
          if (groups >> (32 * o * NG / D) & 1u) acc[o] = float16_t{} + __builtin_nanf("");
      }
    }
  };

  s_marks.clear(tid, kThreads);
  __syncthreads();
  Raw raw = {};   // (undefined, it would be kept from piece to piece)
  if (w.begin < w.end) raw = fetch(w.begin);
  // (the first turn makes the first tile, and has none to multiply)
  for (int32_t tile = w.begin - 1; tile < w.end; ++tile) {
    const uint32_t buffer = (uint32_t)(tile - w.begin) & 1u;
    // The two waves of a SIMD are a key maker and a value maker: one makes before it multiplies and the other behind,
    // so that one's conversions and exponentials run beside the other's products.
    auto next = [&]() __attribute__((always_inline)) {
      if (tile + 1 < w.end) {
        make(raw, tile + 1, buffer ^ 1u);
        if (tile + 2 < w.end) raw = fetch(tile + 2);
      }
    };
    const bool sees = tile >= w.begin && tile * kColumns <= wave_high && tile * kColumns + kColumns > wave_low;
    if (makes_values) next();
    __builtin_amdgcn_s_setprio(1);   // (products before the other wave's codes: 0.5 % of 39 steps)
    if (sees) consume(tile, buffer);
    __builtin_amdgcn_s_setprio(0);
    if (!makes_values) next();
    s_marks.end_turn(buffer, tid, kThreads, [] { __syncthreads(); });
  }
  if (lost && fault && lane == 0) *fault = 1u;
  sum = across_halves(sum, [](float x, float y) { return x + y; });
  top = shift_of(top);

  // ---- parts: as the lanes hold them, (max, sum) of every lane behind the sums; whoever arrives last joins them in
  // order in the same lanes, its own from registers
  const ChunkAttention numbers = scalars(s_numbers);
  const ChunkWork piece = scalars(s_work);
  bool mine_to_write = true;
  if (piece.parts > 1) {
    constexpr uint32_t kState = kOuts * 16 * kThreads;          // floats before the states
    constexpr size_t kPart = kState + 2 * kThreads;
    float* const mine = partials + part_slot(piece, piece.part) * kPart + 2 * tid;
#pragma unroll
    for (int o = 0; o < kOuts; ++o)
#pragma unroll
      for (int r = 0; r < 16; r += 2)
        publish2(mine + (o * 16 + r) * kThreads, float2_t{acc[o][r], acc[o][r + 1]});
    publish2(mine + kState, float2_t{top, sum});
    mine_to_write = arrived_last(tickets + (size_t)piece.first_group * kTicketStride, piece.parts);
    constexpr bool kKeepsOwn = D < 256 || !kF32;   // (registers: there its own part is read back too)
    if (mine_to_write) {
      const float2_t own_state = {top, sum};
      float16_t own[kOuts];
      top = -INFINITY;
      sum = 0.f;
#pragma unroll
      for (int o = 0; o < kOuts; ++o) {
        own[o] = acc[o];
        acc[o] = float16_t{};
      }
      for (uint32_t p = 0; p < piece.parts; ++p) {
        const float* from_part = partials + part_slot(piece, p) * kPart + 2 * tid;
        float2_t state = own_state, x[kOuts * 8];
        if (kKeepsOwn && p == piece.part) {
#pragma unroll
          for (int i = 0; i < kOuts * 8; ++i) x[i] = {own[i / 8][2 * i % 16], own[i / 8][2 * i % 16 + 1]};
        } else {
          state = observe2(from_part + kState);
#pragma unroll
          for (int i = 0; i < kOuts * 8; ++i) x[i] = observe2(from_part + 2 * i * kThreads);
        }
        const float now = fmaxf(top, state[0]), ref = now == -INFINITY ? 0.f : now;
        const float keep = __builtin_amdgcn_exp2f(top - ref), take = __builtin_amdgcn_exp2f(state[0] - ref);
        top = now;
        sum = fmaf(sum, keep, state[1] * take);
#pragma unroll
        for (int o = 0; o < kOuts; ++o)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[o][r] = fmaf(acc[o][r], keep, x[(o * 16 + r) / 2][r & 1] * take);
      }
    }
  }
  // ---- out: lane (m, half) has elements 32 o + 8 (r / 4) + 4 half + r % 4 of its pair
  if (pair < piece.count && mine_to_write) {
    XT* to = out + row_at(numbers, piece, pair, D) + 4 * half;
    const float inverse = 1.0f / sum;
#pragma unroll
    for (int o = 0; o < kOuts; ++o)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        XT x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = from_f32<XT>(acc[o][r + i] * inverse);
        if constexpr (kF32) *reinterpret_cast<float4*>(to + 32 * o + 2 * r) = *reinterpret_cast<const float4*>(x);
        else *reinterpret_cast<uint2*>(to + 32 * o + 2 * r) = *reinterpret_cast<const uint2*>(x);
      }
  }
  __syncthreads();   // (LDS is the next piece's)
}

template <typename XT, int D, int NG>
__global__ __launch_bounds__((Chunk<XT, D>::kThreads)) void kv4_chunk_kernel(
    const XT* __restrict__ q, const uint8_t* __restrict__ cache, const int32_t* __restrict__ page_table,
    const int32_t* __restrict__ cu_rows, const int32_t* __restrict__ lens, XT* __restrict__ out,
    uint32_t* __restrict__ fault, ChunkAttention given) {
  using C = Chunk<XT, D>;
  __shared__ ChunkAttention s_numbers;
  __shared__ ChunkWork s_work;
  __shared__ Deal<C::kThreads / kWave, C::kPairs, C::kColumns> deal;
  if (threadIdx.x == 0) s_numbers = given;
  deal.start(given, cu_rows, lens, fault);
  __syncthreads();
  for (;;) {
    const ChunkAttention a = scalars(s_numbers);
    ChunkWork w;
    if (!deal.next(a, cu_rows, lens, w)) break;
    if (w.refused) {
      refuse<XT, D, C::kThreads>(a, w.kv_head, w.cu0, w.cu1, out);
    } else {
      s_work = w;   // (every wave writes the same words)
      chunk_piece<XT, D, NG>(q, cache, page_table, out, fault, given.partials, given.tickets, a, w, s_numbers, s_work);
    }
  }
}

template <typename XT, int D, int NG>
void launch(krm_ctx* ctx, const ChunkAttention& a, const Kv4Buffers& b) {
  using C = Chunk<XT, D>;
  kv4_chunk_kernel<XT, D, NG><<<dim3(kKv4Groups), dim3(C::kThreads), 2 * C::kTileBytes, ctx->stream>>>(
      ptr<const XT>(b.q), ptr<const uint8_t>(b.cache), ptr<const int32_t>(b.page_table),
      ptr<const int32_t>(b.cu_rows), ptr<const int32_t>(b.lens), ptr<XT>(b.out), ptr<uint32_t>(b.fault), a);
}
template <typename XT>
void launch_depth(krm_ctx* ctx, const ChunkAttention& a, const Kv4Buffers& b) {
  switch (a.layout.depth * 16 + a.layout.groups()) {
    case 64 * 16 + 1: return launch<XT, 64, 1>(ctx, a, b);
    case 64 * 16 + 2: return launch<XT, 64, 2>(ctx, a, b);
    case 128 * 16 + 1: return launch<XT, 128, 1>(ctx, a, b);
    case 128 * 16 + 2: return launch<XT, 128, 2>(ctx, a, b);
    case 128 * 16 + 4: return launch<XT, 128, 4>(ctx, a, b);
    case 256 * 16 + 2: return launch<XT, 256, 2>(ctx, a, b);
    case 256 * 16 + 4: return launch<XT, 256, 4>(ctx, a, b);
    default: return launch<XT, 256, 8>(ctx, a, b);
  }
}

}  // namespace

namespace krm {

static_assert(kKv4Groups <= kTicketSlots, "a counter a workgroup");

size_t kv4_chunk_workspace(uint32_t depth, uint32_t max_columns) {
  const uint32_t tile = depth == 256 ? Chunk<float, 256>::kColumns : Chunk<float, 64>::kColumns;
  if (max_columns <= tile) return 0;   // (blocks of one tile are in one piece: see launch_kv4_chunk)
  const uint32_t pairs = depth == 256 ? Chunk<float, 256>::kPairs : Chunk<float, 64>::kPairs;
  return 2 * (size_t)kKv4Groups * pairs * (depth + 4) * sizeof(float);
}

int32_t launch_kv4_chunk(krm_ctx* ctx, const Kv4Attention& a, const Kv4Buffers& b, int32_t io_dtype) {
  const uint32_t pairs = a.layout.depth == 256 ? Chunk<float, 256>::kPairs : Chunk<float, 64>::kPairs;
  const uint32_t tile = a.layout.depth == 256 ? Chunk<float, 256>::kColumns : Chunk<float, 64>::kColumns;
  ChunkAttention c;
  static_cast<Kv4Attention&>(c) = a;
  // Units of four columns, of a tile where no block has more; or as many as keep a launch's work in 31 bits.
  const uint64_t rows = kv4_rows(a.limits.max_query, a.limits.total_rows);
  const uint64_t blocks = (uint64_t)a.nseq * a.layout.kv_heads * ((rows * a.share + pairs - 1) / pairs);
  c.grain = a.limits.max_columns <= tile ? 31 - __builtin_clz(tile) : 2;
  while (blocks * (((a.limits.max_columns + (uint64_t)pairs + kBegin * tile) >> c.grain) + 2) >= 1ull << 31) ++c.grain;
  // a run has two tiles at least (45 steps of 16 to 1024 rows: four 1.5 % more time, one 0.2 %)
  c.least = 2 * tile >> c.grain ? 2 * tile >> c.grain : 1;
  if (io_dtype == KRM_F32) launch_depth<float>(ctx, c, b);
  else launch_depth<__half>(ctx, c, b);
  return launched(ctx, "kv4_chunk_kernel");
}

}  // namespace krm
