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

struct RotaryAppend {
  Rows q, k, v, qo, ko;  // qo.p, ko.p NULL: not stored; q.p NULL: no q rows
  char *k_pool, *v_pool;
  const int64_t* slots;
  int64_t num_slots;
  Rotary r;
  DivU32 per_tok, pairs;  // pairs per token, pairs per head
  uint32_t total;
  int32_t q_heads, kv_heads;  // q_heads 0 without q
  uint32_t head_bytes;
};

// Indexes from, from + step, ... of the rows' work: one thread per pair of 16-byte vectors of one head, the two that a rotation
// mixes (neighbours where interleaved, rot / 2 apart otherwise), so a row may be rotated in place. Heads come as q, k, v.
template <int DT, bool INTERLEAVED>
__device__ __forceinline__ void rotate_rows(const RotaryAppend& a, uint32_t from, uint32_t step) {
  constexpr int EPL = Elt<DT>::EPL;
  const uint32_t rot_pairs = (uint32_t)a.r.rot / (2 * EPL);
  for (uint32_t i = from; i < a.total; i += step) {
    const uint32_t n = udiv(i, a.per_tok);
    const uint32_t u = i - n * a.per_tok.d;
    const uint32_t head = udiv(u, a.pairs);
    const uint32_t j = u - head * a.pairs.d;
    // The pair's vectors: rotated ones rot / 2 dims apart, the rest neighbours.
    const bool turn = j < rot_pairs && (int)head < a.q_heads + a.kv_heads;
    const bool apart = !INTERLEAVED && j < rot_pairs;
    const uint32_t c0 = (apart ? j : 2 * j) * 16, c1 = apart ? c0 + rot_pairs * 16 : c0 + 16;
    const int section = (int)head < a.q_heads ? 0 : ((int)head < a.q_heads + a.kv_heads ? 1 : 2);
    const Rows src = section == 0 ? a.q : (section == 1 ? a.k : a.v);
    const int64_t h = (int)head - (section == 0 ? 0 : (section == 1 ? a.q_heads : a.q_heads + a.kv_heads));
    const char* row = src.p + (int64_t)n * src.sn + h * src.sh;
    uint4 x = *reinterpret_cast<const uint4*>(row + c0), y = *reinterpret_cast<const uint4*>(row + c1);
    const int64_t pos = a.r.positions[n];
    const bool known = pos >= 0 && pos < a.r.num_positions;
    const int64_t slot = a.slots[n];
    const bool stored = known && slot >= 0 && slot < a.num_slots;
    if (section < 2 && !known) x = y = make_uint4(0u, 0u, 0u, 0u);
    if (turn && known) {
      const float* t = a.r.table + pos * a.r.rot + j * EPL;
      float c[EPL], s[EPL], f[2 * EPL];
      load_floats<EPL>(t, c);
      load_floats<EPL>(t + a.r.rot / 2, s);
      unpack16<DT>(x, f);
      unpack16<DT>(y, f + EPL);
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        if constexpr (INTERLEAVED)
          rotate_pair(f[2 * e], f[2 * e + 1], c[e], s[e]);
        else
          rotate_pair(f[e], f[EPL + e], c[e], s[e]);
      }
      x = pack16<DT>(f);
      y = pack16<DT>(f + EPL);
    }
    if (section < 2) {
      const Rows dst = section == 0 ? a.qo : a.ko;
      if (dst.p) {
        char* o = const_cast<char*>(dst.p) + (int64_t)n * dst.sn + h * dst.sh;
        *reinterpret_cast<uint4*>(o + c0) = x;
        *reinterpret_cast<uint4*>(o + c1) = y;
      }
    }
    if (section > 0 && stored) {
      char* o = (section == 1 ? a.k_pool : a.v_pool) + (slot * a.kv_heads + h) * (int64_t)a.head_bytes;
      *reinterpret_cast<uint4*>(o + c0) = x;
      *reinterpret_cast<uint4*>(o + c1) = y;
    }
  }
}

}  // namespace skv
