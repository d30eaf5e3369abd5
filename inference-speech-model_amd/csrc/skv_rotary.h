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

template <int N>
__device__ __forceinline__ void load_floats(const float* p, float* f) {
  static_assert(N % 4 == 0, "load_floats: whole 16-byte vectors");
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p + i);
    f[i] = __uint_as_float(v.x), f[i + 1] = __uint_as_float(v.y);
    f[i + 2] = __uint_as_float(v.z), f[i + 3] = __uint_as_float(v.w);
  }
}

}  // namespace skv
