// Products of many mx4 rows: tiles of rows of x by rows of w, streamed through a ring of stages in LDS.
#include "lds_stream.h"
#include "mx4_product.h"
#include "mx4_tiles.h"

#include <type_traits>

using namespace krm;

namespace {

// mx4_step with the sum in place, in accumulation registers (as the builtin, hundreds of such sums cross a loop's turn in
// other registers than they began in, with a copy each).  What the compiler cannot know is up to the kernel: two
// waits between a vector instruction that writes an operand and the product, sixteen between the last product and a
// sum's reader (settled()).  Inside the loop nothing but LDS writes operands, scales apart, behind which operands_stand().
template <int STEP>
__device__ inline void mx4_step_in_place(v4i w, uint32_t w_scale, v4i x, uint32_t x_scale, v4f& sum) {
#define KRM_MX4_STEP(SELECT)                                                                          \
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " SELECT " cbsz:4 blgp:4"     \
               : "+a"(sum) : "v"(w), "v"(x), "v"(w_scale), "v"(x_scale))
  if constexpr (STEP == 0) KRM_MX4_STEP("op_sel_hi:[0,0,0]");
  else if constexpr (STEP == 1) KRM_MX4_STEP("op_sel:[1,1,0] op_sel_hi:[0,0,0]");
  else if constexpr (STEP == 2) KRM_MX4_STEP("op_sel_hi:[1,1,0]");
  else KRM_MX4_STEP("op_sel:[1,1,0] op_sel_hi:[1,1,0]");
#undef KRM_MX4_STEP
}
// 16 bytes to memory that every XCD sees, straight from a sum's registers (a vector instruction that wrote them next would
// need a wait).
__device__ inline void publish4(v4f* p, v4f& sum) {
  asm volatile("global_store_dwordx4 %1, %0, off sc1\n\ts_nop 0" : "+a"(sum) : "v"(p) : "memory");
}
__device__ inline void operands_stand() { asm volatile("s_nop 1"); }
template <bool WAIT>
__device__ inline void settled(v4f& sum) {
  if constexpr (WAIT) asm volatile("s_nop 15" : "+a"(sum)); else asm volatile("" : "+a"(sum));
}

// Pieces of 16 columns whose sums make 16 bytes of results in a lane: that many pieces of w in LDS hold a lane's neighbours,
// and the four lanes of a row 64 bytes.
template <typename OT, bool PAIRS>
constexpr uint32_t kMx4Beside = (PAIRS ? 2 : 1) * 4 / sizeof(OT);

// The sums of 16 rows from row0 on (a lane's is r) and PIECES x 16 columns from col0 on.  Two neighbouring sets of 64 bytes
// change places between rows eight apart, so that a store writes whole lines of 128 bytes, which go past the caches.  (Halves
// of lines through the caches: 4096 x 22016 x 4096 249 us, past them 230, whole lines past them 220; halves of 32 bytes past
// them no better than through them.)
template <typename OT, bool PAIRS, int PIECES>
__device__ inline void finish_rows(const Mx4Out& o, uint32_t row0, uint32_t col0, uint32_t r, uint32_t kb,
                                   const v4f (&sum)[PIECES]) {
  constexpr uint32_t kBeside = kMx4Beside<OT, PAIRS>, kSets = PIECES / kBeside, kValues = 16 / sizeof(OT);
  constexpr uint32_t kTogether = kSets > 1 ? 2 : 1;
  const uint32_t width = PAIRS ? o.n / 2 : o.n;
#pragma unroll
  for (uint32_t set = 0; set < kSets; set += kTogether) {
    float v[kTogether][4 * kBeside];
#pragma unroll
    for (uint32_t t = 0; t < kTogether; ++t)
      mx4_values<OT, PAIRS, (int)kBeside>(o, col0 + ((set + t) * 4u + kb) * 4u * kBeside, &sum[(set + t) * kBeside], v[t]);
    if constexpr (kTogether == 2) {
#pragma unroll
      for (uint32_t i = 0; i < kValues; ++i) {
        const int a = __float_as_int(v[0][i]), b = __float_as_int(v[1][i]);
        v[0][i] = __int_as_float(__builtin_amdgcn_update_dpp(a, b, 0x128, 0xf, 0xc, false));  // lanes 8 .. 15 from 0 .. 7
        v[1][i] = __int_as_float(__builtin_amdgcn_update_dpp(b, a, 0x128, 0xf, 0x3, false));  // lanes 0 .. 7 from 8 .. 15
      }
    }
#pragma unroll
    for (uint32_t t = 0; t < kTogether; ++t) {
      const uint32_t row = row0 + (kTogether == 2 ? t * 8u + (r & 7u) : r);
      const uint32_t at = set + (kTogether == 2 ? r >> 3 : 0u);
      const uint32_t first = (PAIRS ? col0 / 2u : col0) + (at * 4u + kb) * kValues;
      if (row < o.m && first < width) mx4_put<OT, (int)kValues, true>(o, row, first, width, v[t]);
    }
  }
}

// A workgroup of WM x WN waves has a tile of WM FM 16 rows of x by WN FN 16 rows of w; a wave FM x FN pieces of 16 x 16.
// Three tiles: 256 x 256 (a wave's sums fill its accumulation registers: fewest reads from LDS), 128 x 128 and 64 x 128, of
// which a CU holds two where there are enough.  us of fp16 results, weights from memory:
//   m x n x k                256 x 256   128 x 128   64 x 128
//   8192 x 8192 x 8192             255         358        475   (4.3 PFLOP/s)
//   512 x 22016 x 4096, pairs       36          46         60
//   1001 x 4100 x 11040            100          53         89
//   509 x 2560 x 2048               21         9.5        7.6
// Bound by power and by the matrix cores' waits for operands: at 8192 cubed the cores run at 1.8 GHz and are busy half of the
// time; 232 us without the stores, 245 without the reads from LDS, 196 without reads and loads, 165 at the rate that
// products of random codes reach from registers.
//
// A stage is 256 codes of every row: 128 bytes, a whole line (of half lines a CU gets half as many bytes a second of rows of
// its own: 58 GB/s, so 107; 1001 x 4100 x 11040 in 128 x 128 tiles 84 us, so 65, no tile shared).  PLACES stages in LDS, two steps of 128
// codes in each: two, or as many as fit where no CU has two workgroups (256 x 4096 x 4096 12.4 us with two, 10.5 with five;
// 1024 x 4096 x 4096, two workgroups a CU, 17.8 and 21.2).  The operands of a step are read from LDS during the step before
// it.  In front of a stage's second step the waves meet: the next stage is there, and the place of this one, all of which has
// been read, is asked to be filled again.
// Scales come in runs of 16 blocks (four steps), half of a run to come asked for with every stage; a lane picks the
// four bytes of its block out of a run's words, and the product instruction one of the four.
// Scales that are no whole words in memory (ALIGNED false) come as the words that they lie in: a run's sixteen bytes
// may end in the first word of the next run, so that runs are asked for one earlier.
// Past the end of K both scales are set to 2^-127: their product is below f32's range, so that whatever codes lie there
// add nothing.
// Several workgroups may share a tile, each some of its runs: all but the last to arrive leave their sums in memory, and the
// last one joins them in the order of K.
template <typename OT, bool PAIRS, int FM, int FN, int WM, int WN, int PLACES, bool ALIGNED>
__global__ __launch_bounds__(64 * WM * WN) void linear_mx4_tile_kernel(
    const uint8_t* __restrict__ xq, const uint8_t* __restrict__ xs, const uint8_t* __restrict__ w,
    const uint8_t* __restrict__ ws, uint32_t blocks, uint32_t m_tiles, uint32_t n_tiles, Mx4Split split, Mx4Out o) {
  static_assert(FN % 4 == 0, "pieces come in fours");
  constexpr uint32_t kWaves = WM * WN, kThreads = 64 * kWaves;
  constexpr uint32_t BM = WM * FM * 16, BN = WN * FN * 16;
  constexpr uint32_t kXLoads = BM / 8 / kWaves, kWLoads = BN / 8 / kWaves;     // of a wave and stage
  static_assert(kXLoads * kWaves * 8 == BM && kWLoads * kWaves * 8 == BN, "whole loads");
  // words of scales: four a row and run, four threads a row
  constexpr uint32_t kXWords = BM * 4 / kThreads, kWWords = BN * 4 / kThreads, kWords = kXWords + kWWords;
  static_assert(kXWords * kThreads == BM * 4 && kWWords * kThreads == BN * 4, "whole loads");
  constexpr uint32_t kScaleLoads = (kWords + 1) / 2;                           // of a wave and stage
  constexpr uint32_t kRun = (BM + BN) * 16;                                    // bytes of a run in LDS
  constexpr uint32_t kLead = ALIGNED ? 1 : 2, kRuns = kLead + (PLACES + 1) / 2; // runs asked for ahead, runs in LDS
  constexpr uint32_t kGroup = kXLoads + kWLoads + kScaleLoads;                 // loads of a stage
  __shared__ __align__(1024) uint8_t s_x[PLACES * BM * 128];
  __shared__ __align__(1024) uint8_t s_w[PLACES * BN * 128];
  __shared__ __align__(1024) uint8_t s_scales[kRuns * kRun];

  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t r = lane & 15u, kb = lane >> 4;
  Mx4Tile tile_at;
  if (!mx4_tile_of(blockIdx.x, m_tiles, n_tiles, split.whole, split.parts, tile_at)) return;  // the whole workgroup leaves
  const uint32_t m0 = tile_at.mt * BM, n0 = tile_at.nt * BN;
  const uint32_t wm = wave / WN, wn = wave % WN;
  // this workgroup's runs of the tile
  const uint32_t runs = (blocks + 15u) / 16u;
  const uint32_t part_of = tile_at.part, parts = tile_at.parts;
  const uint32_t run0 = parts > 1u ? split.first_run(part_of) : 0u;
  const uint32_t run_end = parts > 1u ? least(split.first_run(part_of + 1u), runs) : runs;
  const uint32_t stages = least(run_end * 2u, (blocks + 7u) / 8u);
  const uint32_t m_last = o.m - 1u - m0, n_last = o.n - 1u - n0;  // rows past it: itself again, not stored
  const uint8_t* const x_tile = xq + (size_t)m0 * blocks * 16u;
  const uint8_t* const w_tile = w + (size_t)n0 * blocks * 16u;
  auto lds_address = [](const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)p;
  };
  const uint32_t x_lds = lds_address(s_x), w_lds = lds_address(s_w), scales_lds = lds_address(s_scales);
  // the row of w at a row of LDS (piece i of the kBeside has four rows of each 4 kBeside)
  auto w_row_at = [](uint32_t at) {
    constexpr uint32_t kBeside = kMx4Beside<OT, PAIRS>;
    const uint32_t piece = at >> 4 & 3u;
    return (at & ~63u) + ((piece / kBeside * 4u + (at >> 2 & 3u)) * kBeside + piece % kBeside) * 4u + (at & 3u);
  };

  // A load of a wave brings eight rows of a stage; their pieces of 16 bytes are turned by the row's number, so that the
  // rows that are read at once spread over all banks.  A wave's loads are neighbours in LDS, two to an instruction's base.
  constexpr uint32_t kLoads = kXLoads + kWLoads;
  uint32_t code_row[kLoads];
#pragma unroll
  for (uint32_t i = 0; i < kLoads; ++i)
    code_row[i] = (i < kXLoads ? least((wave * kXLoads + i) * 8u + lane / 8u, m_last)
                               : least(w_row_at((wave * kWLoads + i - kXLoads) * 8u + lane / 8u), n_last)) * blocks * 16u;
  const uint32_t piece = (lane & 7u) ^ (lane >> 3);
  auto code_part = [&](uint32_t asked) { return least(least(asked, stages - 1u) * 8u + piece, blocks - 1u) * 16u; };
  // loads `first` and, where there is one of the same rows, the next: how many
  auto pair = [](uint32_t first) { return first + 1 < (first < kXLoads ? kXLoads : kLoads) ? 2u : 1u; };
  auto request = [&](uint32_t part, uint32_t place, uint32_t i) {
    const bool is_x = i < kXLoads;
    const uint32_t lds = is_x ? x_lds + place * BM * 128u + (wave * kXLoads + i) * 1024u
                              : w_lds + place * BN * 128u + (wave * kWLoads + i - kXLoads) * 1024u;
    const uint8_t* const tile = is_x ? x_tile : w_tile;
    if (pair(i) == 2u) stream_two_to_lds(lds, code_row[i] + part, code_row[i + 1] + part, tile);
    else stream_to_lds(lds, code_row[i] + part, tile);
  };
  // Scales are asked for as words from the one that holds the tile's first; a word that is asked for holds a
  // scale of its row.
  const uint8_t* const xs_tile = xs + (size_t)m0 * blocks;
  const uint8_t* const ws_tile = ws + (size_t)n0 * blocks;
  const uint32_t xs_low = ALIGNED ? 0u : (uint32_t)(uintptr_t)xs_tile & 3u;
  const uint32_t ws_low = ALIGNED ? 0u : (uint32_t)(uintptr_t)ws_tile & 3u;
  uint32_t scale_row[kWords];  // where this thread's rows begin
#pragma unroll
  for (uint32_t i = 0; i < kWords; ++i)
    scale_row[i] = i < kXWords ? least(i * kThreads / 4u + threadIdx.x / 4u, m_last) * blocks + xs_low
                               : least(w_row_at((i - kXWords) * kThreads / 4u + threadIdx.x / 4u), n_last) * blocks + ws_low;
  auto word_of = [&](uint32_t first, uint32_t run, uint32_t part) {
    const uint32_t at = run * 16u + part * 4u;
    if constexpr (ALIGNED) return first + least(at, blocks - 4u);
    return least((first & ~3u) + at, (first + blocks - 1u) & ~3u);
  };
  auto request_scales = [&](uint32_t run, uint32_t i) {
    const uint32_t load = least(i, kWords - 1u);  // (the last loads of a run may be spare: its last again)
    stream_word_to_lds(scales_lds + run % kRuns * kRun + wave * 256u + load * kThreads * 4u,
                       word_of(scale_row[load], run, threadIdx.x & 3u),
                       load < kXWords ? xs_tile - xs_low : ws_tile - ws_low, false);
  };

  v4f sum[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) sum[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

  // a step's four pieces of a row's eight: the other step's are 64 bytes off in the turned order
  const uint32_t code_at = r * 128u + ((kb ^ (r & 7u)) * 16u);
  const uint8_t* const w_pieces[2] = {s_w + wn * FN * 2048u + code_at, s_w + wn * FN * 2048u + (code_at ^ 64u)};
  const uint8_t* const x_pieces[2] = {s_x + wm * FM * 2048u + code_at, s_x + wm * FM * 2048u + (code_at ^ 64u)};
  auto read_w = [&](uint32_t place, int step, int i) {
    return *reinterpret_cast<const v4i*>(w_pieces[step] + place * BN * 128u + i * 2048);
  };
  auto read_x = [&](uint32_t place, int step, int j) {
    return *reinterpret_cast<const v4i*>(x_pieces[step] + place * BM * 128u + j * 2048);
  };
  // byte kb of four words, one a step
  const uint32_t pick = 0x0c0c0400u + kb * 0x0101u;
  const uint32_t x_low = (r & 3u) * blocks + xs_low, w_low = (r & 3u) * blocks + ws_low;  // where a row begins in its word
  struct Scales {
    v4i words;
    uint32_t fifth;
  };
  auto read_scales = [&](uint32_t run, int f) {  // of piece f of w, or f - FN of x
    const uint32_t row = f < FN ? BM + wn * FN * 16u + f * 16u + r : wm * FM * 16u + (f - FN) * 16u + r;
    Scales d;
    d.words = *reinterpret_cast<const v4i*>(s_scales + run % kRuns * kRun + row * 16u);
    d.fifth = ALIGNED ? 0u : *reinterpret_cast<const uint32_t*>(s_scales + (run + 1u) % kRuns * kRun + row * 16u);
    return d;
  };
  auto scale_word = [&](const Scales& s, int f, uint32_t keep) {
    uint32_t d[5] = {(uint32_t)s.words[0], (uint32_t)s.words[1], (uint32_t)s.words[2], (uint32_t)s.words[3], s.fifth};
    if constexpr (!ALIGNED) {
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = __builtin_amdgcn_alignbyte(d[i + 1], d[i], f < FN ? w_low : x_low);
    }
    const uint32_t a = __builtin_amdgcn_perm(d[1], d[0], pick), b = __builtin_amdgcn_perm(d[3], d[2], pick);
    return __builtin_amdgcn_perm(b, a, 0x05040100u) & keep;
  };
  auto kept = [&](uint32_t run) {  // bytes of a lane's words that are there
    const int32_t count = (int32_t)(blocks + 3u - kb - run * 16u) >> 2;
    return (uint32_t)((1ull << (8u * (uint32_t)max(min(count, 4), 0))) - 1ull);
  };

#pragma unroll
  for (uint32_t i = 0; i < kLead * 2 * kScaleLoads; ++i) request_scales(run0 + i / (2 * kScaleLoads), i % (2 * kScaleLoads));
#pragma unroll
  for (uint32_t d = 0; d < PLACES; ++d) {
#pragma unroll
    for (uint32_t i = 0; i < kLoads; i += pair(i)) request(code_part(run0 * 2u + d), d, i);
#pragma unroll
    for (uint32_t i = 0; i < kScaleLoads; ++i) request_scales(run0 + d / 2u + kLead, d % 2u * kScaleLoads + i);
  }
  wait_vm<(PLACES - 1) * kGroup>();
  __builtin_amdgcn_s_barrier();
  // operands of a step and of the one behind it
  v4i w_held[2][FN], x_held[2][FM];
  uint32_t w_scale[FN], x_scale[FM];
  {
    const uint32_t keep = kept(run0);
#pragma unroll
    for (int f = 0; f < FN + FM; ++f) {
      if (f < FN) w_scale[f] = scale_word(read_scales(run0, f), f, keep), w_held[0][f] = read_w(0, 0, f);
      else x_scale[f - FN] = scale_word(read_scales(run0, f), f, keep), x_held[0][f - FN] = read_x(0, 0, f - FN);
    }
  }
  // (steps past the end: codes of the last stage, scales of nothing)
  uint32_t place = 0;
  for (uint32_t run = run0; run < run_end; ++run) {
    uint32_t next_scale[FN + FM];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint32_t next_place = place + 1u == PLACES ? 0u : place + 1u;
      if (s % 2 == 1) {
        wait_vm<(PLACES - 2) * kGroup>();                   // the next stage is there
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and all of this one has been read
        __builtin_amdgcn_s_barrier();
      }
      const uint32_t part = code_part(run * 2u + s / 2 + PLACES);
      if (s == 0) operands_stand();
      // Between the products, one every few of them: a stage's loads, and what the next step takes from LDS, in the first
      // three quarters, so that it is there when the waves meet.
      constexpr int kProducts = FN * FM, kReads = FN + FM, kAsks = kLoads + kScaleLoads;
      constexpr int kEvery = kProducts * 3 / 4 / kReads > 0 ? kProducts * 3 / 4 / kReads : 1;
      const uint32_t keep = kept(run + 1u);
      Scales raw[3];
#pragma unroll
      for (int p = 0; p < kProducts; ++p) {
        const int i = p / FM, j = p % FM;
        if (s % 2 == 1) {
          if (const int q = p * kAsks / kProducts; q < (p + 1) * kAsks / kProducts) {
            if (q >= (int)kLoads) request_scales(run + (s / 2 + PLACES) / 2u + kLead, (s / 2 + PLACES) % 2u * kScaleLoads + q - kLoads);
            else if ((q < (int)kXLoads ? q : q - (int)kXLoads) % 2 == 0) request(part, place, q);
          }
        }
        if (p % kEvery == 0 && p / kEvery < kReads) {
          const int f = p / kEvery;
          const uint32_t from = s % 2 == 0 ? place : next_place;
          constexpr int kNext[4] = {1, 0, 1, 0};
          if (f < FM) x_held[kNext[s]][f] = read_x(from, kNext[s], f);
          else w_held[kNext[s]][f - FM] = read_w(from, kNext[s], f - FM);
          if (s == 3) {
            raw[f % 3] = read_scales(run + 1u, f);
            if (f >= 2) next_scale[f - 2] = scale_word(raw[(f - 2) % 3], f - 2, keep);
          }
        }
        if (s == 0) mx4_step_in_place<0>(w_held[0][i], w_scale[i], x_held[0][j], x_scale[j], sum[i][j]);
        if (s == 1) mx4_step_in_place<1>(w_held[1][i], w_scale[i], x_held[1][j], x_scale[j], sum[i][j]);
        if (s == 2) mx4_step_in_place<2>(w_held[0][i], w_scale[i], x_held[0][j], x_scale[j], sum[i][j]);
        if (s == 3) mx4_step_in_place<3>(w_held[1][i], w_scale[i], x_held[1][j], x_scale[j], sum[i][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
      static_assert((kProducts + kEvery - 1) / kEvery >= kReads && kAsks <= kProducts, "one a product at most, and all of them");
      if (s % 2 == 1) place = next_place;
      if (s == 3) {
#pragma unroll
        for (int f = kReads - 2; f < kReads; ++f) next_scale[f] = scale_word(raw[f % 3], f, keep);
      }
    }
#pragma unroll
    for (int f = 0; f < FN + FM; ++f) {
      if (f < FN) w_scale[f] = next_scale[f]; else x_scale[f - FN] = next_scale[f];
    }
  }
  wait_vm<0>();  // (nothing may land in LDS that is another workgroup's)
  if (parts > 1u) {
    // pieces of a workgroup's sums: 16 bytes of thread t at [piece][t]
    constexpr uint32_t kPieces = FN * FM;
    v4f* const tile = reinterpret_cast<v4f*>(split.sums) + (size_t)tile_at.shared * parts * kPieces * kThreads + threadIdx.x;
    uint32_t* const ticket = split.tickets + (size_t)tile_at.shared * kTicketStride;
    __shared__ uint32_t s_arrived;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        if (i == 0 && j == 0) settled<true>(sum[0][0]);
        publish4(tile + ((size_t)part_of * kPieces + i * FM + j) * kThreads, sum[i][j]);
      }
    wait_vm<0>();  // this thread's sums are in memory
    __syncthreads();
    if (threadIdx.x == 0) s_arrived = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (s_arrived + 1u != parts) return;
    if (threadIdx.x == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // sixteen neighbouring columns of some pieces of x from some parts at once: 128 registers of loads on their way, or 64
    // (a CU holds two workgroups of 128 x 128 up to 256 registers a lane)
    constexpr int kX = FM < 4 ? FM : 4, kAtOnce = FM == 4 ? 1 : 8 / kX;
#pragma unroll
    for (int j0 = 0; j0 < FM * (FN / 4); j0 += kX) {
      const int g = j0 / FM;
      v4f whole[kX][4];
      for (uint32_t part = 0; part < parts; part += kAtOnce) {
        uint64_t raw[kAtOnce][kX][4][2];
#pragma unroll
        for (int a = 0; a < kAtOnce; ++a)
#pragma unroll
          for (int j = 0; j < kX; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint64_t* from = reinterpret_cast<const uint64_t*>(
                  tile + ((size_t)least(part + a, parts - 1u) * kPieces + (4 * g + i) * FM + (j0 + j) % FM) * kThreads);
              raw[a][j][i][0] = __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
              raw[a][j][i][1] = __hip_atomic_load(from + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
#pragma unroll
        for (int a = 0; a < kAtOnce; ++a) {
          if (part + a >= parts) break;
#pragma unroll
          for (int j = 0; j < kX; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              struct Raw { uint64_t r[2]; } r = {{raw[a][j][i][0], raw[a][j][i][1]}};
              const v4f add = __builtin_bit_cast(v4f, r);
              whole[j][i] = part + a == 0 ? add : whole[j][i] + add;
            }
        }
      }
#pragma unroll
      for (int j = 0; j < kX; ++j)
        finish_rows<OT, PAIRS, 4>(o, m0 + (wm * FM + (j0 + j) % FM) * 16u, n0 + wn * FN * 16u + g * 64u, r, kb, whole[j]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    v4f row[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      if (j == 0 && i == 0) settled<true>(sum[0][0]); else settled<false>(sum[i][j]);
      row[i] = sum[i][j];
    }
    finish_rows<OT, PAIRS, FN>(o, m0 + (wm * FM + j) * 16u, n0 + wn * FN * 16u, r, kb, row);
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <int FM, int FN, int WM, int WN, int PLACES>
void launch_tiles(krm_ctx* ctx, const Mx4Product& p, bool half, bool pairs, const Mx4Form& form) {
  constexpr uint32_t BM = WM * FM * 16, BN = WN * FN * 16;
  const uint32_t m_tiles = (p.out.m + BM - 1) / BM, n_tiles = (p.out.n + BN - 1) / BN, runs = (p.blocks + 15) / 16;
  const bool aligned = p.blocks % 4 == 0 && krm::aligned((krm_buf)(uintptr_t)p.xs | (krm_buf)(uintptr_t)p.ws, 4);
  const Mx4Split split{form.whole, form.parts, runs / form.parts, runs % form.parts, ctx->gemm_partials, ctx->tickets};
  const dim3 grid(mx4_tile_grid(m_tiles * n_tiles, form.whole, form.parts));
  auto launch = [&](auto kernel) {
    kernel<<<grid, 64 * WM * WN, 0, ctx->stream>>>(p.xq, p.xs, p.w, p.ws, p.blocks, m_tiles, n_tiles, split, p.out);
  };
#define KRM_MX4_TILES(OT, PAIRS)                                                                     \
  do {                                                                                               \
    if (aligned) launch(linear_mx4_tile_kernel<OT, PAIRS, FM, FN, WM, WN, PLACES, true>);            \
    else launch(linear_mx4_tile_kernel<OT, PAIRS, FM, FN, WM, WN, PLACES, false>);                   \
  } while (0)
  if (half) { if (pairs) KRM_MX4_TILES(__half, true); else KRM_MX4_TILES(__half, false); }
  else { if (pairs) KRM_MX4_TILES(float, true); else KRM_MX4_TILES(float, false); }
#undef KRM_MX4_TILES
}

}  // namespace

namespace krm {

int32_t launch_mx4_tiles(krm_ctx* ctx, const Mx4Product& p, bool half, bool pairs, const Mx4Form& form) {
  switch (form.rows) {
    case 256: launch_tiles<8, 8, 2, 2, 2>(ctx, p, half, pairs, form); break;
    case 128:
      if (form.deep) launch_tiles<4, 4, 2, 2, 4>(ctx, p, half, pairs, form);
      else launch_tiles<4, 4, 2, 2, 2>(ctx, p, half, pairs, form);
      break;
    default:
      if (form.deep) launch_tiles<2, 4, 2, 2, 5>(ctx, p, half, pairs, form);
      else launch_tiles<2, 4, 2, 2, 2>(ctx, p, half, pairs, form);
      break;
  }
  return launched(ctx, "linear_mx4_tile_kernel");
}

}  // namespace krm
