// Which kernel a product of mx4 rows runs in, by its sizes alone.  Nothing here is of the device: the CPU tests compile it.
#pragma once

#include <cstdint>
#include <initializer_list>

namespace krm {

// kRows: up to 16 rows of x that fit LDS, floats too.  kBatch: up to 64 rows of codes.  kTiles: tiles of `rows` rows of x
// (256: by 256 rows of w, else by 128), those behind the first `whole` ones shared by `parts` workgroups that have some of K each.
// `deep`: with a CU's whole LDS to a workgroup, where no CU has two.
enum class Mx4Kernel : uint32_t { kRows, kBatch, kTiles };
struct Mx4Form {
  Mx4Kernel kernel;
  uint32_t rows, parts;
  bool deep;
  uint32_t whole;
};

constexpr uint32_t kMx4HeldBytes = 64u * 1024u;  // of x in LDS beside two turns of every wave (linear_mx4_rows.hip)
constexpr uint32_t mx4_code_pitch(uint32_t blocks) { return blocks * 16u + 16u; }
constexpr uint32_t mx4_scale_pitch(uint32_t blocks) { return (blocks + 15u) & ~15u; }
inline bool mx4_rows_fit(uint32_t m, uint32_t k) {
  const uint32_t blocks = k / 32;
  return m <= 16 && (uint64_t)m * (mx4_code_pitch(blocks) + mx4_scale_pitch(blocks)) <= kMx4HeldBytes;
}

// What a form takes, in us: fitted (non-negative least squares of the relative error) to 2791 runs of 324 products of
// 17 to 9000 rows, 64 to 22400 columns and a K of 256 to 12800 whose weights came from memory, within 5 to 9 % (rms).  The forms
// that it picks take 1.007 of the best one's time on average over those products, 1.18 at worst.
inline float mx4_batch_us(uint32_t m, uint32_t n, uint32_t k, uint32_t cus) {
  const uint32_t pieces = (n + 15) / 16;
  const float rounds = (float)((pieces + cus - 1) / cus), turns = (float)((k + 1023) / 1024);
  return 2.38f + rounds * (0.74f + turns * (m <= 32 ? 0.408f : 0.674f));
}
inline float mx4_tiles_us(uint32_t rows, uint32_t parts, uint64_t tiles, uint32_t k, uint32_t cus) {
  struct Fit {
    // `next`: of a round of the CUs behind the first; `filled`: of as much work as such a round has
    float fixed, step, next_step, filled_step, next, filled, joined, part, next_part;
  };
  const Fit f = rows == 256   ? Fit{10.65f, 0.624f, 0.952f, 0.f, 10.69f, 1.92f, 5.00f, 4.76f, 0.f}
                : rows == 128 ? Fit{5.72f, 0.249f, 0.241f, 0.067f, 0.46f, 1.59f, 1.14f, 1.45f, 1.31f}
                              : Fit{4.60f, 0.189f, 0.206f, 0.016f, 0.11f, 0.94f, 2.32f, 0.59f, 0.70f};
  const uint32_t runs = (k + 511) / 512;
  const uint64_t groups = tiles * parts;
  const float steps = 4.f * (float)((runs + parts - 1) / parts), more = (float)((groups + cus - 1) / cus - 1);
  const float filled = groups > cus ? (float)groups / (float)cus - 1.f : 0.f;
  const float us = f.fixed + steps * (f.step + more * f.next_step + filled * f.filled_step) + more * f.next + filled * f.filled;
  return parts > 1 ? us + f.joined + (float)parts * (f.part + more * f.next_part) : us;
}
inline uint64_t mx4_tile_count(uint32_t rows, uint32_t m, uint32_t n) {
  const uint32_t columns = rows == 256 ? 256 : 128;
  return (uint64_t)((m + rows - 1) / rows) * ((n + columns - 1) / columns);
}

inline bool mx4_deep(uint32_t rows, uint64_t workgroups, uint32_t cus) { return rows < 256 && workgroups <= cus; }

// `scratch`: bytes for the sums of parts, `counters` of tiles that are shared; 0 where a tile must not be shared.
inline Mx4Form mx4_form(uint32_t m, uint32_t n, uint32_t k, uint32_t cus, uint64_t scratch, uint32_t counters) {
  if (mx4_rows_fit(m, k)) return {Mx4Kernel::kRows, 16, 1, false, 0};
  Mx4Form best{Mx4Kernel::kBatch, 64, 1, false, 0};
  float us = m <= 64 ? mx4_batch_us(m, n, k, cus) : 3.4e38f;
  for (uint32_t rows : {64u, 128u, 256u}) {
    const uint64_t tiles = mx4_tile_count(rows, m, n);
    for (uint32_t parts : {1u, 2u, 3u, 4u, 6u, 8u, 12u, 16u}) {
      const uint64_t bytes = tiles * parts * rows * (rows == 256 ? 256u : 128u) * 4u;
      if (parts > 1 && (parts > (k + 511) / 512 || bytes > scratch || tiles > counters)) break;
      const float estimate = mx4_tiles_us(rows, parts, tiles, k, cus);
      if (estimate < us) us = estimate, best = {Mx4Kernel::kTiles, rows, parts, mx4_deep(rows, tiles * parts, cus), parts > 1 ? 0u : (uint32_t)tiles};
    }
  }
  // A last round of few tiles of 128 rows is shared: its CUs would hold one workgroup more than the others.  1.05 to 1.29
  // times as fast where K is above 6144 (1001 x 4100 x 11040, 264 tiles, 65.2 us, so 52.5; 1200 x 4096 x 8192, 320 tiles, 40.6 /
  // 36.4); the join takes it away again below (1100 x 4096 x 4096 21.2 / 22.6).  A last round of up to 7/16 of the CUs: 101
  // tiles for 256 CUs still gain (357 tiles, K of 11744, 76.8 / 68.0), 140 lose (396 tiles, K of 11296, 70.3 / 89.0).  (Tiles
  // of 64 rows are not picked where there are two rounds of them and such a K.)
  const uint32_t runs = (k + 511) / 512;
  if (best.kernel == Mx4Kernel::kTiles && best.rows == 128 && best.parts == 1 && best.whole > cus && runs > 12) {
    const uint32_t last = best.whole % cus, parts = last * 3 <= cus ? 3 : 2;
    if (last > 0 && last * 16 <= cus * 7 && (uint64_t)last * parts * 128u * 128u * 4u <= scratch && last <= counters)
      best.parts = parts, best.whole -= last;
  }
  return best;
}

}  // namespace krm
