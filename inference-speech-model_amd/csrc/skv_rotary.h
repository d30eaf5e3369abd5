// Rotary positions: the (cos, sin) table and the rotation of one 16-byte vector's worth of pairs, shared by the appends
// into 16/32-bit pools and into the 4-bit cache.
#pragma once

#include "skv_device.h"

namespace skv {

// Rows of a projection or a result: element (n, h, d) at base[n * sn + h * sh + d].
struct Rows {
  const char* p;
  int64_t sn, sh;  // bytes
};

struct Rotary {
  const float* table;        // [num_positions][rot]: cos of rot / 2 angles, then sin; NULL: no rotation
  const int64_t* positions;  // [n_tokens]
  int64_t num_positions;
  int32_t rot;
  int32_t interleaved;  // pairs (2i, 2i + 1); else (i, i + rot / 2)
};

// One rotated pair: every product and the sum rounded to fp32 by itself, so the results are those of separate elementary
// operations to the last bit (what the 4-bit codes of values next to a rounding border need to be reproducible).
__device__ __forceinline__ void rotate_pair(float& a, float& b, float c, float s) {
#pragma clang fp contract(off)
  const float ac = a * c, bs = b * s, bc = b * c, as = a * s;
  a = ac - bs;
  b = bc + as;
}

}  // namespace skv
