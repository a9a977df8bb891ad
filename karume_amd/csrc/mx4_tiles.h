// Which workgroup of a product of mx4 rows has which tile and which part of K, and what the launchers hand over.
#pragma once

#include "mx4_plan.h"
#include "mx4_product.h"

namespace krm {

struct Mx4Product {
  const uint8_t *xq, *xs, *w, *ws;
  uint32_t blocks;  // of 32 codes in a row
  Mx4Out out;
};

int32_t launch_mx4_rows(krm_ctx* ctx, const Mx4Product& p, bool half, bool pairs);
int32_t launch_mx4_rows_of(krm_ctx* ctx, const Mx4Product& p, krm_buf x, uint64_t stride, int32_t x_dtype, bool ceil,
                           bool half, bool pairs);
int32_t launch_mx4_batch(krm_ctx* ctx, const Mx4Product& p, bool half, bool pairs);
int32_t launch_mx4_tiles(krm_ctx* ctx, const Mx4Product& p, bool half, bool pairs, const Mx4Form& form);

// Tiles from `whole` on (in the order below) are shared by `parts` workgroups: runs of 512 codes dealt to them, and where
// they leave their sums.
struct Mx4Split {
  uint32_t whole, parts, each, extra;  // the first `extra` parts have one run more
  float* sums;
  uint32_t* tickets;            // one a tile, kTicketStride words apart, zero at rest
  __host__ __device__ uint32_t first_run(uint32_t part) const { return part * each + (part < extra ? part : extra); }
};

// Workgroups go to the eight XCDs in turn.  Each XCD has a run of the tiles' order, in which four tiles of x follow
// one another for a tile of w (neighbours in time share both through its L2) and the parts of a tile one another.
constexpr uint32_t kMx4Xcds = 8, kMx4Band = 4;
__host__ __device__ inline uint32_t mx4_tile_grid(uint32_t tiles, uint32_t whole, uint32_t parts) {
  return ((whole + kMx4Xcds - 1) / kMx4Xcds + ((tiles - whole) * parts + kMx4Xcds - 1) / kMx4Xcds) * kMx4Xcds;
}
struct Mx4Tile {
  uint32_t mt, nt;
  uint32_t shared, part, parts;  // which of the shared tiles; one part: of none
};
__host__ __device__ inline bool mx4_tile_of(uint32_t block, uint32_t m_tiles, uint32_t n_tiles, uint32_t whole, uint32_t parts,
                                            Mx4Tile& t) {
  const uint32_t alone = (whole + kMx4Xcds - 1) / kMx4Xcds * kMx4Xcds;
  const bool shares = block >= alone;
  const uint32_t count = shares ? (m_tiles * n_tiles - whole) * parts : whole;
  const uint32_t in_order = shares ? block - alone : block, run = (count + kMx4Xcds - 1) / kMx4Xcds;
  const uint32_t unit = in_order % kMx4Xcds * run + in_order / kMx4Xcds;
  if (unit >= count) return false;
  t.parts = shares ? parts : 1u;
  t.shared = unit / t.parts;
  t.part = unit - t.shared * t.parts;
  const uint32_t at = shares ? whole + t.shared : unit;
  const uint32_t band = at / (kMx4Band * n_tiles), in_band = at - band * kMx4Band * n_tiles;
  const uint32_t high = m_tiles - band * kMx4Band < kMx4Band ? m_tiles - band * kMx4Band : kMx4Band;
  t.nt = in_band / high;
  t.mt = band * kMx4Band + in_band % high;
  return true;
}

}  // namespace krm
