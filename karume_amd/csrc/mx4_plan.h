// Which kernel a product of mx4 rows runs in, by its sizes alone.  Nothing here is of the device: the CPU tests compile it.
#pragma once

#include <cstdint>
#include <initializer_list>

namespace krm {

// kRows: up to 16 rows of x that fit LDS, floats too.  kBatch: up to 64 rows of codes.  kTiles: tiles of `rows` rows of x
// (256: by 256 rows of w, else by 128), each shared by `parts` workgroups that have some of K each.
enum class Mx4Kernel : uint32_t { kRows, kBatch, kTiles };
struct Mx4Form {
  Mx4Kernel kernel;
  uint32_t rows, parts;
};

constexpr uint32_t kMx4HeldBytes = 64u * 1024u;  // of x in LDS beside two turns of every wave (linear_mx4_rows.hip)
constexpr uint32_t mx4_code_pitch(uint32_t blocks) { return blocks * 16u + 16u; }
constexpr uint32_t mx4_scale_pitch(uint32_t blocks) { return (blocks + 15u) & ~15u; }
inline bool mx4_rows_fit(uint32_t m, uint32_t k) {
  const uint32_t blocks = k / 32;
  return m <= 16 && (uint64_t)m * (mx4_code_pitch(blocks) + mx4_scale_pitch(blocks)) <= kMx4HeldBytes;
}

// What a form takes, in us: fitted (non-negative least squares of the relative error) to 1025 runs of 102 products of
// 17 to 4096 rows, 64 to 22400 columns and a K of 256 to 12800 whose weights came from memory, within 7 to 10 % (rms).  The forms
// that it picks take 1.005 of the best one's time on average over those products, 1.28 at worst.
inline float mx4_batch_us(uint32_t m, uint32_t n, uint32_t k, uint32_t cus) {
  const uint32_t steps = (k + 127) / 128, pieces = (n + 15) / 16;
  const float rounds = (float)((pieces + cus - 1) / cus), turns = (float)((steps + 7) / 8);
  return 2.19f + rounds * (0.66f + turns * (m <= 32 ? 0.458f : 0.707f));
}
inline float mx4_tiles_us(uint32_t rows, uint32_t parts, uint64_t tiles, uint32_t k, uint32_t cus) {
  struct Fit {
    float fixed, step, next_step, next, joined, part, next_part;  // `next`: of a round of the CUs behind the first
  };
  const Fit f = rows == 256   ? Fit{7.97f, 0.612f, 0.820f, 15.5f, 5.43f, 4.76f, 0.f}
                : rows == 128 ? Fit{4.52f, 0.245f, 0.364f, 2.66f, 0.96f, 1.44f, 1.03f}
                              : Fit{3.60f, 0.204f, 0.309f, 1.57f, 2.12f, 0.60f, 0.68f};
  const uint32_t runs = (k + 511) / 512;
  const float steps = 4.f * (float)((runs + parts - 1) / parts), more = (float)((tiles * parts + cus - 1) / cus - 1);
  const float us = f.fixed + steps * (f.step + more * f.next_step) + more * f.next;
  return parts > 1 ? us + f.joined + (float)parts * (f.part + more * f.next_part) : us;
}
inline uint64_t mx4_tile_count(uint32_t rows, uint32_t m, uint32_t n) {
  const uint32_t columns = rows == 256 ? 256 : 128;
  return (uint64_t)((m + rows - 1) / rows) * ((n + columns - 1) / columns);
}

// `scratch`: bytes for the sums of parts, `counters` of tiles that are shared; 0 where a tile must not be shared.
inline Mx4Form mx4_form(uint32_t m, uint32_t n, uint32_t k, uint32_t cus, uint64_t scratch, uint32_t counters) {
  if (mx4_rows_fit(m, k)) return {Mx4Kernel::kRows, 16, 1};
  Mx4Form best{Mx4Kernel::kBatch, 64, 1};
  float us = m <= 64 ? mx4_batch_us(m, n, k, cus) : 3.4e38f;
  for (uint32_t rows : {64u, 128u, 256u}) {
    const uint64_t tiles = mx4_tile_count(rows, m, n);
    for (uint32_t parts : {1u, 2u, 3u, 4u, 6u, 8u, 12u, 16u}) {
      const uint64_t bytes = tiles * parts * rows * (rows == 256 ? 256u : 128u) * 4u;
      if (parts > 1 && (parts > (k + 511) / 512 || bytes > scratch || tiles > counters)) break;
      const float estimate = mx4_tiles_us(rows, parts, tiles, k, cus);
      if (estimate < us) us = estimate, best = {Mx4Kernel::kTiles, rows, parts};
    }
  }
  return best;
}

}  // namespace krm
