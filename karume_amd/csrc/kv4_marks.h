// Marks of columns whose values are no numbers, in the two tiles that a workgroup of kv4_chunk_kernel has at hand: the
// waves that make a tile's values mark it, those that multiply with it read the marks, and the end of that turn clears
// them for the tile that is made there next.  Nothing here needs a device, so a plain C++ compiler can run it with waves
// that are late.
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#define KRM_HD __host__ __device__
#else
#define KRM_HD
#endif

namespace krm {

template <int kColumns>
struct Kv4Marks {
  uint32_t groups[2][kColumns];   // of a column's values: those that are no numbers
  uint32_t any[2];

  // Before a piece's first turn, with a barrier behind it.
  KRM_HD void clear(uint32_t tid, uint32_t threads) {
    for (uint32_t i = tid; i < 2 * kColumns; i += threads) groups[i / kColumns][i % kColumns] = 0;
    if (tid < 2) any[tid] = 0;
  }
  // The end of the turn that multiplied with the tile at `buffer`, for all threads of the workgroup.  Whether they clear
  // has to be one answer: it is read before the barrier, while the other tile is the one that may be marked.  Behind it
  // a wave may have begun the next turn, which marks this one.
  template <typename Barrier>
  KRM_HD void end_turn(uint32_t buffer, uint32_t tid, uint32_t threads, Barrier barrier) {
    const bool marked = any[buffer] != 0;
    barrier();
    if (marked) {
      for (uint32_t i = tid; i < (uint32_t)kColumns; i += threads) groups[buffer][i] = 0;
      if (tid == 0) any[buffer] = 0;
      barrier();
    }
  }
};

}  // namespace krm
