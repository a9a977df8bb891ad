// The rotation that krm_rope_rows and krm_kv4_append share.
#pragma once

#include "krm_internal.h"

namespace krm {

struct RotaryArgs {
  uint32_t head_dim, rotary_dim;   // the first rotary_dim elements of a head are turned
  uint32_t table_rows, table_width;
  int32_t layout;                  // KRM_ROPE_HALF: pairs (j, j + R/2); KRM_ROPE_INTERLEAVED: (2 j, 2 j + 1)
};

#if defined(__HIPCC__)
// (a, b) turned by an angle; both products are rounded before they are joined, as krm_rope_half does.
__device__ inline void turn_pair(float a, float b, float c, float s, float& ta, float& tb) {
  ta = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  tb = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
}
#endif

}  // namespace krm
