// Which workgroup of a product of mx4 rows has which tile, and what the launchers hand over.
#pragma once

#include "mx4_product.h"

namespace krm {

struct Mx4Product {
  const uint8_t *xq, *xs, *w, *ws;
  uint32_t blocks;  // of 32 codes in a row
  Mx4Out out;
};

enum class Mx4Form { kRows, kTiles64, kTiles128, kTiles256 };

// Up to 16 rows of x, in codes or quantised by every workgroup for itself, where they fit LDS.
int32_t launch_mx4_rows(krm_ctx* ctx, const Mx4Product& p, bool half, bool pairs);
bool mx4_rows_fit(uint32_t m, uint32_t k);
int32_t launch_mx4_rows_of(krm_ctx* ctx, const Mx4Product& p, krm_buf x, uint64_t stride, int32_t x_dtype, bool ceil,
                           bool half, bool pairs);
int32_t launch_mx4_tiles(krm_ctx* ctx, const Mx4Product& p, bool half, bool pairs, Mx4Form form);

// Workgroups go to the eight XCDs in turn.  Each XCD has a run of the tiles' order, in which four tiles of x follow
// one another for a tile of w: neighbours in time share both through its L2.
constexpr uint32_t kMx4Xcds = 8, kMx4Band = 4;
__host__ __device__ inline uint32_t mx4_tile_grid(uint32_t m_tiles, uint32_t n_tiles) {
  return (m_tiles * n_tiles + kMx4Xcds - 1) / kMx4Xcds * kMx4Xcds;
}
__host__ __device__ inline bool mx4_tile_of(uint32_t block, uint32_t m_tiles, uint32_t n_tiles, uint32_t& mt,
                                            uint32_t& nt) {
  const uint32_t tiles = m_tiles * n_tiles, run = (tiles + kMx4Xcds - 1) / kMx4Xcds;
  const uint32_t at = block % kMx4Xcds * run + block / kMx4Xcds;
  if (at >= tiles) return false;
  const uint32_t band = at / (kMx4Band * n_tiles), in_band = at - band * kMx4Band * n_tiles;
  const uint32_t high = m_tiles - band * kMx4Band < kMx4Band ? m_tiles - band * kMx4Band : kMx4Band;
  nt = in_band / high;
  mt = band * kMx4Band + in_band % high;
  return true;
}

}  // namespace krm
