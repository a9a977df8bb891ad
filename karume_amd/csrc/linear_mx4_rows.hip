// Products of up to 16 mx4 rows, or rows of floats that are quantised on the way: rows of w are read once and bound
// the time by their bytes.
#include "lds_stream.h"
#include "mx4_tiles.h"

#include <type_traits>

using namespace krm;

namespace {

// Waves that stream and multiply, and waves that bring x.
constexpr uint32_t kStreams = 8, kBringers = 8, kThreads = 64 * (kStreams + kBringers);

// Where the rows of x come from: codes in memory, or floats.
struct Mx4Codes {
  const uint8_t *codes, *scales;
};
template <typename XT>
struct Mx4Floats {
  const XT* x;
  uint64_t stride;
  bool ceil;
};

// (x in LDS: rows of codes 16 bytes apart more than they are long, so that rows at one column spread over all banks, then
// their scales in whole quarters of a run.)

// A turn of a wave is U steps of 128 codes of 16 rows of w: codes, then scales (whole words of a row and step, or a
// byte a lane), DEPTH of them in LDS.
template <int U, bool ALIGNED>
constexpr uint32_t kTurn = U * 1024u + (ALIGNED ? 256u : U * 256u);
constexpr uint32_t kSums = 2 * kStreams * 1024;
template <int U, int DEPTH, bool ALIGNED>
constexpr uint32_t kHeld = 160u * 1024u - kStreams * DEPTH * kTurn<U, ALIGNED> - kSums;  // bytes for x
static_assert(kHeld<4, 2, false> >= kMx4HeldBytes && kHeld<4, 2, true> >= kMx4HeldBytes && kHeld<2, 3, false> >= kMx4HeldBytes &&
                  kHeld<1, 3, false> >= kMx4HeldBytes,
              "what mx4_rows_fit lets in");

// One workgroup a CU walks pieces of 16 rows of w.  Eight waves share a piece's turns in a fixed order, each with a ring
// of its own in LDS that memory fills without registers or barriers, over the ends of pieces too; another eight
// bring x meanwhile and leave.  Those that bring x come first: asked for behind a CU's rows of w, x would arrive behind
// them (1 x 4096 x 4096 4.8 us, so 4.1; 8 x 22016 x 4096 15.0 / 13.1; 1 x 4096 x 11008 8.8 / 7.5).  The streaming waves join
// their sums in LDS, one wave in turn stores a piece.  The order of a row's sums depends on K alone, so that it does not
// matter where x came from.
// Bound by w's bytes: what a CU has on its way (96 KiB) is what keeps memory busy.  1 x 65536 x 4096 26 us, 5.5 TB/s;
// 16 x 32000 x 2048 11.0 us, 3.3 TB/s, eight pieces of two turns a wave each; 1 x 4096 x 4096 3.9 us, of which 2 are a launch.
// (Lines of 128 bytes a load as in the batch's kernel: no difference past 1 %.)
template <typename OT, bool PAIRS, typename X, int U, int DEPTH, bool ALIGNED>
__global__ __launch_bounds__(kThreads) void linear_mx4_rows_kernel(X x, const uint8_t* __restrict__ w,
                                                                   const uint8_t* __restrict__ ws, uint32_t blocks,
                                                                   Mx4Out o) {
  constexpr uint32_t kLoads = U + (ALIGNED ? 1 : U);  // of a turn
  __shared__ __align__(1024) uint8_t s_ring[kStreams][DEPTH][kTurn<U, ALIGNED>];
  __shared__ v4f s_sum[2][kStreams][64];
  __shared__ __align__(16) uint8_t s_x[kHeld<U, DEPTH, ALIGNED>];
  const uint32_t lane = threadIdx.x & 63u, any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t r = lane & 15u, kb = lane >> 4;
  const uint32_t rows = o.m, x_pitch = mx4_code_pitch(blocks), xs_pitch = mx4_scale_pitch(blocks);
  uint8_t* const s_scales = s_x + rows * x_pitch;
  auto met = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };  // (what streams goes on)

  if (any_wave < kBringers) {
    // blocks of codes or pieces of eight floats, one after the other over all rows, a few of a thread's at once
    constexpr bool kCopies = std::is_same<X, Mx4Codes>::value;
    constexpr uint32_t kBringing = kBringers * 64u, kAtOnce = 4;
    const uint32_t length = kCopies ? blocks : blocks * 4u, count = rows * length;
    const uint32_t thread = threadIdx.x;
    uint32_t row = thread / length, at = thread - row * length;
    const uint32_t more_rows = kBringing / length, more = kBringing - more_rows * length;
    for (uint32_t first = thread; first < count; first += kBringing * kAtOnce) {
      uint32_t rows_of[kAtOnce], at_of[kAtOnce];
#pragma unroll
      for (uint32_t i = 0; i < kAtOnce; ++i) {
        rows_of[i] = least(row, rows - 1u);
        at_of[i] = at;
        row += more_rows;
        at += more;
        if (at >= length) at -= length, ++row;
      }
      auto there = [&](uint32_t i) { return first + i * kBringing < count; };
      if constexpr (kCopies) {
        v4i codes[kAtOnce];
        uint8_t scales[kAtOnce];
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i) {
          const size_t from = (size_t)rows_of[i] * blocks + at_of[i];
          codes[i] = *reinterpret_cast<const v4i*>(x.codes + from * 16u);
          scales[i] = x.scales[from];
        }
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i)
          if (there(i)) {
            *reinterpret_cast<v4i*>(s_x + rows_of[i] * x_pitch + at_of[i] * 16u) = codes[i];
            s_scales[rows_of[i] * xs_pitch + at_of[i]] = scales[i];
          }
      } else {
        decltype(mx4_load8(x.x)) e[kAtOnce];
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i) e[i] = mx4_load8(x.x + rows_of[i] * x.stride + (size_t)at_of[i] * 8u);
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i) {
          uint32_t byte;
          const uint32_t codes = mx4_quantise8(e[i], x.ceil, byte);
          if (there(i)) {
            *reinterpret_cast<uint32_t*>(s_x + rows_of[i] * x_pitch + at_of[i] * 4u) = codes;
            if ((at_of[i] & 3u) == 0) s_scales[rows_of[i] * xs_pitch + at_of[i] / 4u] = (uint8_t)byte;
          }
        }
      }
    }
    met();
    return;  // (a barrier waits for the waves that are left)
  }

  const uint32_t wave = any_wave - kBringers;
  const uint32_t steps = (blocks + 3u) / 4u, pieces = (o.n + 15u) / 16u;
  const uint32_t turns = ((steps + U - 1u) / U + kStreams - 1u) / kStreams;  // of a wave and piece
  const uint32_t my_pieces = (pieces - blockIdx.x + gridDim.x - 1u) / gridDim.x, total = my_pieces * turns;
  auto lds_address = [](const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)p;
  };
  const uint32_t ring_lds = lds_address(&s_ring[wave][0][0]);
  struct Place {
    uint32_t piece, turn, slot;
  };
  auto advance = [&](Place& at) {
    if (++at.slot == DEPTH) at.slot = 0;
    if (++at.turn == turns) at.turn = 0, at.piece += gridDim.x;
  };
  auto step_of = [&](const Place& at, uint32_t u) { return (at.turn * kStreams + wave) * U + u; };
  // Four lanes bring 64 neighbouring bytes of a row; the pieces of 16 turned by the row's number, so that rows that
  // are read at once spread over all banks.
  const uint32_t chunk = (lane & 3u) ^ ((lane >> 3) & 3u);
  auto request = [&](const Place& at) {
    const uint32_t n0 = at.piece * 16u, n_last = least(o.n - 1u - n0, 15u);
    const uint8_t* const w_piece = w + (size_t)n0 * blocks * 16u;
    const uint8_t* const ws_piece = ws + (size_t)n0 * blocks;
    const uint32_t lds = ring_lds + at.slot * kTurn<U, ALIGNED>;
    const uint32_t row = least(lane / 4u, n_last) * blocks;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
      stream_to_lds(lds + u * 1024u, (row + least(step_of(at, u) * 4u + chunk, blocks - 1u)) * 16u, w_piece);
    if constexpr (ALIGNED) {
      const uint32_t of_row = least(least(lane / U, 15u), n_last) * blocks;
      stream_word_to_lds(lds + U * 1024u, of_row + least(step_of(at, lane % U) * 4u, blocks - 4u), ws_piece, false);
    } else {
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
        stream_byte_to_lds(lds + U * 1024u + u * 256u, least(r, n_last) * blocks + least(step_of(at, u) * 4u + kb, blocks - 1u), ws_piece);
    }
  };

  Place at{blockIdx.x, 0, 0}, ahead = at;
  uint32_t asked = 0;
  for (; asked < DEPTH && asked < total; ++asked) {
    request(ahead);
    advance(ahead);
  }
  met();  // x is there
  const uint32_t code_at = r * 64u + ((kb ^ ((r >> 1) & 3u)) * 16u);
  const uint32_t x_row = least(r, rows - 1u);
  v4f sum = {0.f, 0.f, 0.f, 0.f};
  uint32_t done = 0;  // pieces
  for (uint32_t t = 0; t < total; ++t) {
    if (asked - t == DEPTH) wait_vm<(DEPTH - 1) * kLoads>(); else wait_vm<0>();
    const uint8_t* const turn = s_ring[wave][at.slot];
    v4i wc[U], xc[U];
    uint32_t w_scale[U], x_scale[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      wc[u] = *reinterpret_cast<const v4i*>(turn + u * 1024u + code_at);
      xc[u] = *reinterpret_cast<const v4i*>(s_x + x_row * x_pitch + least(step_of(at, u) * 4u + kb, blocks - 1u) * 16u);
      if constexpr (ALIGNED) w_scale[u] = *reinterpret_cast<const uint32_t*>(turn + U * 1024u + (r * U + u) * 4u);
      else w_scale[u] = *reinterpret_cast<const uint32_t*>(turn + U * 1024u + u * 256u + lane * 4u);
      x_scale[u] = *reinterpret_cast<const uint32_t*>(s_scales + x_row * xs_pitch + least(step_of(at, u) * 4u, xs_pitch - 4u));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the turn's place is free
    if (asked < total) {
      request(ahead);
      advance(ahead);
      ++asked;
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      // past the end of K both scales are 2^-127: their product is below f32's range
      const bool there = ALIGNED ? step_of(at, u) < steps : step_of(at, u) * 4u + kb < blocks;
      const uint32_t s_w = ALIGNED ? w_scale[u] >> (8u * kb) : w_scale[u], s_x8 = x_scale[u] >> (8u * kb);
      sum = mx4_step(wc[u], there ? s_w : 0u, xc[u], there ? s_x8 : 0u, sum);
    }
    if (at.turn + 1u == turns) {
      s_sum[done & 1u][wave][lane] = sum;
      sum = v4f{0.f, 0.f, 0.f, 0.f};
      met();
      if (wave == done % kStreams) {
        v4f whole = s_sum[done & 1u][0][lane];
#pragma unroll
        for (uint32_t v = 1; v < kStreams; ++v) whole += s_sum[done & 1u][v][lane];
        mx4_finish<OT, PAIRS>(o, r, at.piece * 16u + kb * 4u, whole);
      }
      ++done;
    }
    advance(at);
  }
}

// 17 to 64 rows of x: the same walk by four waves, 256 codes a turn, with the rows of x (MB times 16) streamed beside those
// of w, from the L2 that they stay in.  Tiles that share their rows in LDS hold too few CUs here, and parts of K joined
// through memory cost 4 to 5 us.
// Bound by what a CU takes from its L2: x once for 16 rows of w.  Eight waves with half lines of 64 bytes took 19.0 us for
// 64 x 4096 x 11008 where this takes 15.0, and 13.4 for 32 rows (10.9); 64 x 4096 x 4096 6.9 and 6.5.
constexpr uint32_t kBatchStreams = 4;
template <int MB, bool ALIGNED>
constexpr uint32_t kBatchTurn = (1 + MB) * 2048u + (ALIGNED ? 256u + (MB * 32 + 63) / 64 * 256u : (1 + MB) * 512u);

template <typename OT, bool PAIRS, int MB, int DEPTH, bool ALIGNED>
__global__ __launch_bounds__(64 * kBatchStreams) void linear_mx4_batch_kernel(const uint8_t* __restrict__ xq,
                                                                              const uint8_t* __restrict__ xs,
                                                                              const uint8_t* __restrict__ w,
                                                                              const uint8_t* __restrict__ ws, uint32_t blocks,
                                                                              Mx4Out o) {
  constexpr uint32_t kXWords = (MB * 32 + 63) / 64;                             // loads of x's scales: two words a row
  constexpr uint32_t kLoads = 2 * (1 + MB) + (ALIGNED ? 1 + kXWords : 2 * (1 + MB));  // of a turn
  constexpr uint32_t kBytes = kBatchTurn<MB, ALIGNED>, kScalesAt = (1 + MB) * 2048u;
  __shared__ __align__(1024) uint8_t s_ring[kBatchStreams][DEPTH][kBytes];
  __shared__ v4f s_sum[kBatchStreams / 2][MB][64];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t r = lane & 15u, kb = lane >> 4;
  const uint32_t stages = (blocks + 7u) / 8u, pieces = (o.n + 15u) / 16u, turns = (stages + kBatchStreams - 1u) / kBatchStreams;
  const uint32_t my_pieces = (pieces - blockIdx.x + gridDim.x - 1u) / gridDim.x, total = my_pieces * turns;
  auto met = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  auto lds_address = [](const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)p;
  };
  const uint32_t ring_lds = lds_address(&s_ring[wave][0][0]);
  struct Place {
    uint32_t piece, turn, slot;
  };
  auto advance = [&](Place& at) {
    if (++at.slot == DEPTH) at.slot = 0;
    if (++at.turn == turns) at.turn = 0, at.piece += gridDim.x;
  };
  auto first_block = [&](const Place& at) { return (at.turn * kBatchStreams + wave) * 8u; };
  // eight lanes bring 128 neighbouring bytes of a row, their pieces of 16 turned by the row's number
  const uint32_t chunk = (lane & 7u) ^ (lane >> 3);
  uint32_t x_row[2 * MB];
#pragma unroll
  for (uint32_t b = 0; b < 2 * MB; ++b) x_row[b] = least(b * 8u + lane / 8u, o.m - 1u) * blocks;
  uint32_t x_scale_row[kXWords];
#pragma unroll
  for (uint32_t b = 0; b < kXWords; ++b) x_scale_row[b] = least(b * 32u + lane / 2u, o.m - 1u) * blocks;
  auto request = [&](const Place& at) {
    const uint32_t n0 = at.piece * 16u, n_last = least(o.n - 1u - n0, 15u), from = first_block(at);
    const uint8_t* const w_piece = w + (size_t)n0 * blocks * 16u;
    const uint8_t* const ws_piece = ws + (size_t)n0 * blocks;
    const uint32_t lds = ring_lds + at.slot * kBytes, block = least(from + chunk, blocks - 1u);
#pragma unroll
    for (uint32_t b = 0; b < 2; ++b)
      stream_to_lds(lds + b * 1024u, (least(b * 8u + lane / 8u, n_last) * blocks + block) * 16u, w_piece);
#pragma unroll
    for (uint32_t b = 0; b < 2 * MB; ++b) stream_to_lds(lds + (2u + b) * 1024u, (x_row[b] + block) * 16u, xq);
    if constexpr (ALIGNED) {
      const uint32_t word = least(from + (lane & 1u) * 4u, blocks - 4u);
      stream_word_to_lds(lds + kScalesAt, least(least(lane / 2u, 15u), n_last) * blocks + word, ws_piece, false);
#pragma unroll
      for (uint32_t b = 0; b < kXWords; ++b)
        stream_word_to_lds(lds + kScalesAt + 256u + b * 256u, x_scale_row[b] + word, xs, false);
    } else {
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t byte = least(from + h * 4u + kb, blocks - 1u);
        stream_byte_to_lds(lds + kScalesAt + h * 256u, least(r, n_last) * blocks + byte, ws_piece);
#pragma unroll
        for (uint32_t b = 0; b < MB; ++b)
          stream_byte_to_lds(lds + kScalesAt + ((1u + b) * 2u + h) * 256u, least(b * 16u + r, o.m - 1u) * blocks + byte, xs);
      }
    }
  };

  Place at{blockIdx.x, 0, 0}, ahead = at;
  uint32_t asked = 0;
  for (; asked < DEPTH && asked < total; ++asked) {
    request(ahead);
    advance(ahead);
  }
  const uint32_t code_at = r * 128u + ((kb ^ (r & 7u)) * 16u);
  v4f sum[MB];
#pragma unroll
  for (uint32_t b = 0; b < MB; ++b) sum[b] = v4f{0.f, 0.f, 0.f, 0.f};
  for (uint32_t t = 0; t < total; ++t) {
    if (asked - t == DEPTH) wait_vm<(DEPTH - 1) * kLoads>(); else wait_vm<0>();
    const uint8_t* const turn = s_ring[wave][at.slot];
    v4i wc[2], xc[2][MB];
    uint32_t w_word[2], x_word[2][MB];
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t code = code_at ^ h * 64u;
      wc[h] = *reinterpret_cast<const v4i*>(turn + code);
      w_word[h] = *reinterpret_cast<const uint32_t*>(turn + kScalesAt + (ALIGNED ? r * 2u + h : h * 64u + lane) * 4u);
#pragma unroll
      for (uint32_t b = 0; b < MB; ++b) {
        xc[h][b] = *reinterpret_cast<const v4i*>(turn + (1u + b) * 2048u + code);
        const uint32_t word = ALIGNED ? 256u + ((b * 16u + r) * 2u + h) * 4u : ((1u + b) * 2u + h) * 256u + lane * 4u;
        x_word[h][b] = *reinterpret_cast<const uint32_t*>(turn + kScalesAt + word);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the turn's place is free
    if (asked < total) {
      request(ahead);
      advance(ahead);
      ++asked;
    }
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      // past the end of K both scales are 2^-127: their product is below f32's range
      const bool there = first_block(at) + h * 4u + (ALIGNED ? 0u : kb) < blocks;
      const uint32_t shift = ALIGNED ? 8u * kb : 0u, w_scale = there ? w_word[h] >> shift : 0u;
#pragma unroll
      for (uint32_t b = 0; b < MB; ++b) sum[b] = mx4_step(wc[h], w_scale, xc[h][b], there ? x_word[h][b] >> shift : 0u, sum[b]);
    }
    if (at.turn + 1u == turns) {
      // the upper waves' sums to the lower ones, whose sums then make the rows of 16 of one wave each
      if (wave >= kBatchStreams / 2) {
#pragma unroll
        for (uint32_t b = 0; b < MB; ++b) s_sum[wave - kBatchStreams / 2][b][lane] = sum[b];
      }
      met();
      if (wave < kBatchStreams / 2) {
#pragma unroll
        for (uint32_t b = 0; b < MB; ++b) s_sum[wave][b][lane] = sum[b] + s_sum[wave][b][lane];
      }
      met();
      if (wave < MB) {
        v4f whole = s_sum[0][wave][lane];
#pragma unroll
        for (uint32_t v = 1; v < kBatchStreams / 2; ++v) whole += s_sum[v][wave][lane];
        mx4_finish<OT, PAIRS>(o, wave * 16u + r, at.piece * 16u + kb * 4u, whole);
      }
      met();  // (the sums' place is free)
#pragma unroll
      for (uint32_t b = 0; b < MB; ++b) sum[b] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    advance(at);
  }
}

// Steps a turn: four, or as many as leave every wave a turn.
uint32_t steps_a_turn(uint32_t blocks) {
  const uint32_t steps = (blocks + 3) / 4;
  return steps > 2 * kStreams ? 4 : steps > kStreams ? 2 : 1;
}

template <typename X>
void launch_rows_of(krm_ctx* ctx, const X& x, const Mx4Product& p, bool half, bool pairs) {
  const bool words = p.blocks % 4 == 0 && aligned((krm_buf)(uintptr_t)p.ws, 4);
  const uint32_t pieces = (p.out.n + 15) / 16, grid = pieces < (uint32_t)ctx->num_cus ? pieces : ctx->num_cus;
  const uint32_t u = steps_a_turn(p.blocks);
  const uint64_t held = (uint64_t)p.out.m * (mx4_code_pitch(p.blocks) + mx4_scale_pitch(p.blocks));
  const bool deep = held <= (words ? kHeld<4, 3, true> : kHeld<4, 3, false>);
  auto launch = [&](auto kernel) { kernel<<<grid, kThreads, 0, ctx->stream>>>(x, p.w, p.ws, p.blocks, p.out); };
#define KRM_MX4_ROWS_FORM(OT, PAIRS, U, DEPTH)                                                   \
  do {                                                                                           \
    if (words) launch(linear_mx4_rows_kernel<OT, PAIRS, X, U, DEPTH, true>);                     \
    else launch(linear_mx4_rows_kernel<OT, PAIRS, X, U, DEPTH, false>);                          \
  } while (0)
#define KRM_MX4_ROWS(OT, PAIRS)                          \
  do {                                                   \
    if (u == 1) KRM_MX4_ROWS_FORM(OT, PAIRS, 1, 3);      \
    else if (u == 2) KRM_MX4_ROWS_FORM(OT, PAIRS, 2, 3); \
    else if (deep) KRM_MX4_ROWS_FORM(OT, PAIRS, 4, 3);   \
    else KRM_MX4_ROWS_FORM(OT, PAIRS, 4, 2);             \
  } while (0)
  if (half) { if (pairs) KRM_MX4_ROWS(__half, true); else KRM_MX4_ROWS(__half, false); }
  else { if (pairs) KRM_MX4_ROWS(float, true); else KRM_MX4_ROWS(float, false); }
#undef KRM_MX4_ROWS
#undef KRM_MX4_ROWS_FORM
}

template <int MB, int DEPTH>
void launch_batch(krm_ctx* ctx, const Mx4Product& p, bool half, bool pairs) {
  const bool words = p.blocks % 4 == 0 && aligned((krm_buf)(uintptr_t)p.xs | (krm_buf)(uintptr_t)p.ws, 4);
  const uint32_t pieces = (p.out.n + 15) / 16, grid = pieces < (uint32_t)ctx->num_cus ? pieces : ctx->num_cus;
  auto launch = [&](auto kernel) { kernel<<<grid, 64 * kBatchStreams, 0, ctx->stream>>>(p.xq, p.xs, p.w, p.ws, p.blocks, p.out); };
#define KRM_MX4_BATCH(OT, PAIRS)                                                         \
  do {                                                                                   \
    if (words) launch(linear_mx4_batch_kernel<OT, PAIRS, MB, DEPTH, true>);              \
    else launch(linear_mx4_batch_kernel<OT, PAIRS, MB, DEPTH == 3 ? 2 : DEPTH, false>); \
  } while (0)
  if (half) { if (pairs) KRM_MX4_BATCH(__half, true); else KRM_MX4_BATCH(__half, false); }
  else { if (pairs) KRM_MX4_BATCH(float, true); else KRM_MX4_BATCH(float, false); }
#undef KRM_MX4_BATCH
}

}  // namespace

namespace krm {

int32_t launch_mx4_batch(krm_ctx* ctx, const Mx4Product& p, bool half, bool pairs) {
  if (p.out.m <= 32) launch_batch<2, 5>(ctx, p, half, pairs); else launch_batch<4, 3>(ctx, p, half, pairs);
  return launched(ctx, "linear_mx4_batch_kernel");
}

int32_t launch_mx4_rows(krm_ctx* ctx, const Mx4Product& p, bool half, bool pairs) {
  launch_rows_of(ctx, Mx4Codes{p.xq, p.xs}, p, half, pairs);
  return launched(ctx, "linear_mx4_rows_kernel");
}

int32_t launch_mx4_rows_of(krm_ctx* ctx, const Mx4Product& p, krm_buf x, uint64_t stride, int32_t x_dtype, bool ceil,
                           bool half, bool pairs) {
  if (x_dtype == KRM_F16) launch_rows_of(ctx, Mx4Floats<__half>{ptr<const __half>(x), stride, ceil}, p, half, pairs);
  else launch_rows_of(ctx, Mx4Floats<float>{ptr<const float>(x), stride, ceil}, p, half, pairs);
  return launched(ctx, "linear_mx4_rows_kernel");
}

}  // namespace krm
