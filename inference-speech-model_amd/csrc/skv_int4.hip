// The paged 4-bit K/V cache: append (with the position rotation on the way), gather, attention.
//
// Format. Each 32 consecutive dims of a (token, head) row share fp16 (scale, low); an element is low + scale * code with
// code = round((x - low) / scale) in 0..15, low = fp16(min x), scale = fp16((max x - low) / 15): 5 bits an element. Values
// beyond +-16384 saturate and a NaN is held as 0, so that everything the cache can hold is finite.
// Pools are uint8 [num_blocks, kv heads, block_size / 16, 10 * D]: a head's 16-token tiles lie one after the other, so a
// workgroup that reads one head reads whole cache lines (rows of 16 to 64 bytes per (token, head), as the 16-bit pools lay
// their rows out, would share each line among heads, whose workgroups sit on different dies).
//   K tile: [16 tokens][D / 2] bytes, a dword per 8 dims with dims 0..7 in nibbles 0, 4, 1, 5, 2, 6, 3, 7; then
//           [16][D / 32] pairs (scale, low).
//   V tile: [4 quads][D / 2][4 tokens] bytes, dims 2m and 2m + 1 in the low and high nibble of byte m; then
//           [4 quads][D / 32][scale, low][4 tokens, in the order 0, 2, 1, 3].
// Both orders are those in which the matrix cores' operands come out of shifts and masks alone: 16-bit halves of a K dword
// hold neighbouring dims, those of a V dword tokens 0, 2 and 1, 3 of one dim.
#include <hip/hip_runtime.h>

#include "skv_common.h"
#include "skv_rotary.h"

using namespace skv;

namespace {

constexpr int kTile = 16;          // tokens of a tile
constexpr int kGroup = 32;         // elements that share a scale
constexpr float kLimit = 16384.f;  // stored values saturate here: low, scale, and low - 16 scale stay within fp16

bool supported_d4(int32_t d) { return d == 32 || d == 64 || d == 128; }

__device__ __forceinline__ float half_bits(uint32_t h) { return (float)__builtin_bit_cast(_Float16, (uint16_t)h); }
__device__ __forceinline__ uint32_t to_half_bits(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }

// ---------------------------------------------------------------------------
// Append.
// ---------------------------------------------------------------------------
struct Int4Append {
  Rows q, k, v, qo, ko;
  char *k_pool, *v_pool;
  const int64_t* slots;
  int64_t num_slots;
  Rotary r;
  DivU32 per_tok;  // lanes per token
  uint32_t total;
  int32_t q_heads, kv_heads;
  DivU32 tiles;     // tiles per (block, head)
};

// 8 dims of a row in fp32.
template <int DT>
__device__ __forceinline__ void load8(const char* row, int c, float* f) {
  if constexpr (DT == SKV_F32) {
    unpack16<DT>(*reinterpret_cast<const uint4*>(row + 32 * c), f);
    unpack16<DT>(*reinterpret_cast<const uint4*>(row + 32 * c + 16), f + 4);
  } else {
    unpack16<DT>(*reinterpret_cast<const uint4*>(row + 16 * c), f);
  }
}
template <int DT>
__device__ __forceinline__ void store8(char* row, int c, const float* f) {
  if constexpr (DT == SKV_F32) {
    *reinterpret_cast<uint4*>(row + 32 * c) = pack16<DT>(f);
    *reinterpret_cast<uint4*>(row + 32 * c + 16) = pack16<DT>(f + 4);
  } else {
    *reinterpret_cast<uint4*>(row + 16 * c) = pack16<DT>(f);
  }
}
// 8 values rounded to the rows' type.
template <int DT>
__device__ __forceinline__ void round8(float* f) {
  if constexpr (DT != SKV_F32) {
    const uint4 v = pack16<DT>(f);
    unpack16<DT>(v, f);
  }
}

// One lane per 8 dims of a row, D / 8 lanes (4 to 16, never across a wave) per row: K rows, V rows, then q rows, which are
// only rotated. A rotated row's lanes all load before any stores, so q and k may be rotated in place. The codes are taken
// from the rotated values rounded to the rows' type, what a 16-bit cache would hold.
template <int DT, int D, bool INTERLEAVED>
__global__ __launch_bounds__(256) void append_int4_kernel(Int4Append a) {
  constexpr int LPR = D / 8;
  for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < a.total; i += gridDim.x * 256u) {
    const uint32_t n = udiv(i, a.per_tok);
    const uint32_t u = i - n * a.per_tok.d;
    const int c = (int)(u % LPR);
    const int head = (int)(u / LPR);
    const int section = head < a.kv_heads ? 0 : (head < 2 * a.kv_heads ? 1 : 2);
    const int h = head - section * a.kv_heads;
    const Rows src = section == 0 ? a.k : (section == 1 ? a.v : a.q);
    const char* row = src.p + (int64_t)n * src.sn + (int64_t)h * src.sh;
    float f[8];
    load8<DT>(row, c, f);
    bool known = true;
    if (section != 1 && a.r.table) {
      const int64_t pos = a.r.positions[n];
      known = pos >= 0 && pos < a.r.num_positions;
      const int half = a.r.rot / 2;
      if (known && 8 * c < a.r.rot) {
        const float* t = a.r.table + pos * a.r.rot;
        if constexpr (INTERLEAVED) {
          float cs[4], sn[4];
          load_floats<4>(t + 4 * c, cs);
          load_floats<4>(t + half + 4 * c, sn);
#pragma unroll
          for (int e = 0; e < 4; ++e) rotate_pair(f[2 * e], f[2 * e + 1], cs[e], sn[e]);
        } else {
          const bool low = 8 * c < half;
          const int j = low ? c : c - half / 8;
          float cs[8], sn[8], g[8];
          load8<DT>(row, low ? c + half / 8 : j, g);
          load_floats<8>(t + 8 * j, cs);
          load_floats<8>(t + half + 8 * j, sn);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float x = low ? f[e] : g[e], y = low ? g[e] : f[e];
            rotate_pair(x, y, cs[e], sn[e]);
            f[e] = low ? x : y;
          }
        }
        round8<DT>(f);
      }
      if (!known) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 0.f;
      }
      const Rows dst = section == 0 ? a.ko : a.qo;
      if (dst.p) store8<DT>(const_cast<char*>(dst.p) + (int64_t)n * dst.sn + (int64_t)h * dst.sh, c, f);
    } else if (section == 1 && a.r.table) {
      const int64_t pos = a.r.positions[n];
      known = pos >= 0 && pos < a.r.num_positions;
    }
    if (section == 2) continue;
    // The group's range, over its 4 lanes.
    float lo = __builtin_huge_valf(), hi = kNegInf;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[e] = f[e] != f[e] ? 0.f : fminf(fmaxf(f[e], -kLimit), kLimit);
      lo = fminf(lo, f[e]);
      hi = fmaxf(hi, f[e]);
    }
    lo = fminf(lo, xor_lane<1>(lo));
    hi = fmaxf(hi, xor_lane<1>(hi));
    lo = fminf(lo, xor_lane<2>(lo));
    hi = fmaxf(hi, xor_lane<2>(hi));
    const int64_t slot = a.slots[n];
    if (!known || slot < 0 || slot >= a.num_slots) continue;
    const uint32_t low_h = to_half_bits(lo);
    const float low = half_bits(low_h);
    const uint32_t scale_h = to_half_bits(fmaxf((hi - low) / 15.f, 0.f));
    const float scale = half_bits(scale_h);
    const float inv = scale > 0.f ? 1.f / scale : 0.f;
    uint32_t code[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) code[e] = (uint32_t)fminf(fmaxf(rintf((f[e] - low) * inv), 0.f), 15.f);
    // slot = (block * tiles + tile of the block) * 16 + token; a (block, head) has tiles.d tiles.
    const int64_t tile = slot >> 4;
    const int t = (int)(slot & 15);
    const int64_t blk = tile / a.tiles.d;
    const int64_t at = ((blk * a.kv_heads + h) * a.tiles.d + (tile - blk * a.tiles.d)) * (10 * D);
    if (section == 0) {
      char* o = a.k_pool + at;
      const uint32_t w = code[0] | code[2] << 4 | code[4] << 8 | code[6] << 12 | code[1] << 16 | code[3] << 20 |
                         code[5] << 24 | code[7] << 28;
      *reinterpret_cast<uint32_t*>(o + t * (D / 2) + 4 * c) = w;
      if ((c & 3) == 0) *reinterpret_cast<uint32_t*>(o + 8 * D + (t * (D / kGroup) + c / 4) * 4) = scale_h | low_h << 16;
    } else {
      char* o = a.v_pool + at;
      const int quad = t >> 2, k = t & 3;
#pragma unroll
      for (int y = 0; y < 4; ++y)
        o[quad * 2 * D + (4 * c + y) * 4 + k] = (char)(code[2 * y] | code[2 * y + 1] << 4);
      if ((c & 3) == 0) {
        char* m = o + 8 * D + (quad * (D / kGroup) + c / 4) * 16 + 2 * ((k & 1) * 2 + (k >> 1));
        *reinterpret_cast<uint16_t*>(m) = (uint16_t)scale_h;
        *reinterpret_cast<uint16_t*>(m + 8) = (uint16_t)low_h;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Gather: out[b, h, t, :] = the values of position t of row b for t < lens[b], zero otherwise.
// ---------------------------------------------------------------------------
// One thread per 8 dims of 4 tokens (a quad) of one head, of K (grid.y 0) or V (1).
template <int DT, int D>
__global__ __launch_bounds__(256) void gather_int4_kernel(const char* k_pool, const char* v_pool, const int32_t* tables,
                                                          int64_t tstride, const int32_t* lens, char* k_out, char* v_out,
                                                          uint32_t total, DivU32 quads, DivU32 heads, int32_t tiles,
                                                          int32_t nb, int32_t max_len) {
  constexpr int LPR = D / 8;
  constexpr int kRow = D * (DT == SKV_F32 ? 4 : 2);
  const bool is_v = blockIdx.y != 0;
  for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < total; i += gridDim.x * 256u) {
    const int c = (int)(i % LPR);
    const uint32_t bhq = i / LPR;
    const uint32_t bh = udiv(bhq, quads);
    const int t0 = (int)(bhq - bh * quads.d) * 4;
    const uint32_t b = udiv(bh, heads);
    const uint32_t h = bh - b * heads.d;
    const int len = min(max(lens[b], 0), max_len);
    char* out = (is_v ? v_out : k_out) + ((int64_t)bh * max_len + t0) * kRow;
    float f[4][8];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) f[k][e] = 0.f;
    if (t0 < len) {
      const int tile = t0 >> 4, in = tile % tiles, blk_i = tile / tiles;
      const uint32_t blk = (uint32_t)tables[(int64_t)b * tstride + blk_i];
      if (blk < (uint32_t)nb) {
        const char* p = (is_v ? v_pool : k_pool) + (((int64_t)blk * heads.d + h) * tiles + in) * (10 * D);
        const int t = t0 & 15, quad = t >> 2;
        if (!is_v) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(p + (t + k) * (D / 2) + 4 * c);
            const uint32_t m = *reinterpret_cast<const uint32_t*>(p + 8 * D + ((t + k) * (D / kGroup) + c / 4) * 4);
            const float scale = half_bits(m & 0xffffu), low = half_bits(m >> 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              f[k][2 * e] = fmaf(scale, (float)((w >> (4 * e)) & 15u), low);
              f[k][2 * e + 1] = fmaf(scale, (float)((w >> (4 * e + 16)) & 15u), low);
            }
          }
        } else {
          const uint4 w4 = *reinterpret_cast<const uint4*>(p + quad * 2 * D + 16 * c);
          const uint4 m4 = *reinterpret_cast<const uint4*>(p + 8 * D + (quad * (D / kGroup) + c / 4) * 16);
          const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
          const uint32_t sc[2] = {m4.x, m4.y}, lw[2] = {m4.z, m4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int sh = 16 * (k >> 1);  // tokens 0, 2 in the first word, 1, 3 in the second
            const float scale = half_bits((sc[k & 1] >> sh) & 0xffffu), low = half_bits((lw[k & 1] >> sh) & 0xffffu);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t byte = (w[y] >> (8 * k)) & 255u;
              f[k][2 * y] = fmaf(scale, (float)(byte & 15u), low);
              f[k][2 * y + 1] = fmaf(scale, (float)(byte >> 4), low);
            }
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (t0 + k >= max_len) break;
      if (t0 + k >= len) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[k][e] = 0.f;
      }
      store8<DT>(out + (int64_t)k * kRow, c, f[k]);
    }
  }
}

// ---------------------------------------------------------------------------
// Attention.
// ---------------------------------------------------------------------------
struct Int4Attn {
  const char *q, *k_pool, *v_pool;
  char* o;
  int64_t qsb, qsq, qsh, osb, osq, osh;  // bytes
  const int32_t *tables, *trows, *lens;
  int64_t tstride;
  float* part;
  float scale_log2;
  int32_t batch, qlen, heads, kv_heads, group, tiles, nb, max_ctx, causal, chunk, nchunk;
};

constexpr int kPad = 4;  // floats (max, sum, unused) ahead of a partial's accumulators
constexpr int kAttnWaves = 4;

// Keys query qi of row b sees.
__device__ __forceinline__ int visible(const Int4Attn& p, int b, int qi) {
  const int len = p.lens[b] - (p.causal ? p.qlen - 1 - qi : 0);
  return min(max(len, 0), p.max_ctx);
}

// One workgroup per (row, query, head, key chunk), everything in fp32: 16-key tiles go to its waves in turn.
// Scores: lane (g, r) takes a quarter of key r's dims. Values: lane m takes dims 2m and 2m + 1 of D / 2 lanes' worth of
// quads. The simple form, for fp32 rows.
template <int DT, int D>
__global__ __launch_bounds__(64 * kAttnWaves) void attention_int4_kernel(Int4Attn p) {
  constexpr int ND = D / 32;        // dwords of a lane's quarter row
  constexpr int LPM = D / 2;        // lanes that cover a row of V
  constexpr int PARTS = 64 / LPM;   // lane sets, each with its share of the quads
  constexpr int QUADS = 4 / PARTS;
  __shared__ __attribute__((aligned(16))) float s_q[D];
  __shared__ float s_state[kAttnWaves][2 + D];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int g = lane >> 4, r = lane & 15;
  const int h = blockIdx.x % p.heads;
  const int rest = blockIdx.x / p.heads;
  const int qi = rest % p.qlen, b = rest / p.qlen;
  const int chunk = blockIdx.y;
  const int kvh = h / p.group;
  const int len = visible(p, b, qi);
  const int t_begin = chunk * p.chunk, t_end = min(len, t_begin + p.chunk);
  if (t_begin >= len && chunk > 0) return;  // the merge knows
  const char* q = p.q + (int64_t)b * p.qsb + (int64_t)qi * p.qsq + (int64_t)h * p.qsh;
  if (threadIdx.x < D / 8) {
    float f[8];
    load8<DT>(q, threadIdx.x, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) s_q[8 * threadIdx.x + e] = f[e];
  }
  __syncthreads();
  float qf[8 * ND], qsum = 0.f;
#pragma unroll
  for (int e = 0; e < 8 * ND; ++e) {
    qf[e] = s_q[g * 8 * ND + e];
    qsum += qf[e];
  }
  const int32_t* trow = p.tables + (int64_t)(p.trows ? p.trows[b] : b) * p.tstride;
  const int m = lane % LPM, part = lane / LPM;
  float top = kNegInf, sum = 0.f, a0 = 0.f, a1 = 0.f;
  for (int t0 = t_begin + wave * kTile; t0 < t_end; t0 += kAttnWaves * kTile) {
    const int tile = t0 >> 4;
    const uint32_t blk = (uint32_t)trow[tile / p.tiles];
    if (blk >= (uint32_t)p.nb) continue;  // wave-uniform
    const int64_t at = (((int64_t)blk * p.kv_heads + kvh) * p.tiles + tile % p.tiles) * (10 * D);
    const char *kt = p.k_pool + at, *vt = p.v_pool + at;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(kt + r * (D / 2) + (g * ND + i) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s = fmaf(qf[8 * i + 2 * e], (float)((w >> (4 * e)) & 15u), s);
        s = fmaf(qf[8 * i + 2 * e + 1], (float)((w >> (4 * e + 16)) & 15u), s);
      }
    }
    const uint32_t km = *reinterpret_cast<const uint32_t*>(kt + 8 * D + (r * (D / kGroup) + g * 8 * ND / kGroup) * 4);
    s = fmaf(s, half_bits(km & 0xffffu), qsum * half_bits(km >> 16));
    s += xor_lane<16>(s);
    s += xor_lane<32>(s);
    s = t0 + r < t_end ? s * p.scale_log2 : kNegInf;
    float mx = s;
    mx = max_score(mx, xor_lane<1>(mx));
    mx = max_score(mx, xor_lane<2>(mx));
    mx = max_score(mx, xor_lane<4>(mx));
    mx = max_score(mx, xor_lane<8>(mx));
    mx = max_score(mx, top);
    const float ref = mx == kNegInf ? 0.f : mx;
    const float w = __builtin_amdgcn_exp2f(s - ref), alpha = __builtin_amdgcn_exp2f(top - ref);
    top = mx;
    sum = fmaf(sum, alpha, group_sum<16>(w));
    a0 *= alpha;
    a1 *= alpha;
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
      const int quad = part * QUADS + i;
      const uint32_t w4 = *reinterpret_cast<const uint32_t*>(vt + quad * 2 * D + 4 * m);
      const uint4 m4 = *reinterpret_cast<const uint4*>(vt + 8 * D + (quad * (D / kGroup) + m / 16) * 16);
      const uint32_t sc[2] = {m4.x, m4.y}, lw[2] = {m4.z, m4.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int sh = 16 * (k >> 1);
        const float scale = half_bits((sc[k & 1] >> sh) & 0xffffu), low = half_bits((lw[k & 1] >> sh) & 0xffffu);
        const uint32_t byte = (w4 >> (8 * k)) & 255u;
        const float pk = __shfl(w, quad * 4 + k);  // lanes 0..15 hold the tile's weights
        if (t0 + quad * 4 + k < t_end) {           // what lies past the row's end may be anything
          a0 = fmaf(pk, fmaf(scale, (float)(byte & 15u), low), a0);
          a1 = fmaf(pk, fmaf(scale, (float)(byte >> 4), low), a1);
        }
      }
    }
  }
  if constexpr (PARTS >= 2) {
    a0 += xor_lane<32>(a0);
    a1 += xor_lane<32>(a1);
  }
  if constexpr (PARTS >= 4) {
    a0 += xor_lane<16>(a0);
    a1 += xor_lane<16>(a1);
  }
  if (lane < LPM) {
    s_state[wave][2 + 2 * lane] = a0;
    s_state[wave][2 + 2 * lane + 1] = a1;
  }
  if (lane == 0) {
    s_state[wave][0] = top;
    s_state[wave][1] = sum;
  }
  __syncthreads();
  if (threadIdx.x >= D) return;
  const int d = threadIdx.x;
  float mm = s_state[0][0];
  for (int w = 1; w < kAttnWaves; ++w) mm = max_score(mm, s_state[w][0]);
  const float ref = mm == kNegInf ? 0.f : mm;
  float l = 0.f, acc = 0.f;
  for (int w = 0; w < kAttnWaves; ++w) {
    const float f = __builtin_amdgcn_exp2f(s_state[w][0] - ref);
    l = fmaf(s_state[w][1], f, l);
    acc = fmaf(s_state[w][2 + d], f, acc);
  }
  if (p.nchunk > 1 && len > p.chunk) {
    float* rec = p.part + ((((int64_t)b * p.qlen + qi) * p.heads + h) * p.nchunk + chunk) * (D + kPad);
    rec[kPad + d] = acc;
    if (d == 0) rec[0] = mm, rec[1] = l;
    return;
  }
  const float out = l > 0.f || l != l ? acc / l : 0.f;
  char* o = p.o + (int64_t)b * p.osb + (int64_t)qi * p.osq + (int64_t)h * p.osh;
  if constexpr (DT == SKV_F32)
    reinterpret_cast<float*>(o)[d] = out;
  else
    reinterpret_cast<uint16_t*>(o)[d] = (uint16_t)pack2<DT>(out, 0.f);
}

// Rows of several chunks: one workgroup of D threads per (row, query, head) joins the chunks' partials.
template <int DT, int D>
__global__ __launch_bounds__(D < 64 ? 64 : D) void merge_int4_kernel(Int4Attn p) {
  const int h = blockIdx.x % p.heads;
  const int rest = blockIdx.x / p.heads;
  const int qi = rest % p.qlen, b = rest / p.qlen;
  const int len = visible(p, b, qi);
  const int n = (len + p.chunk - 1) / p.chunk;
  if (n <= 1 || threadIdx.x >= D) return;
  const int d = threadIdx.x;
  const float* rec = p.part + (((int64_t)b * p.qlen + qi) * p.heads + h) * p.nchunk * (D + kPad);
  float mm = kNegInf;
  for (int c = 0; c < n; ++c) mm = max_score(mm, rec[c * (D + kPad)]);
  const float ref = mm == kNegInf ? 0.f : mm;
  float l = 0.f, acc = 0.f;
  for (int c = 0; c < n; ++c) {
    const float f = __builtin_amdgcn_exp2f(rec[c * (D + kPad)] - ref);
    l = fmaf(rec[c * (D + kPad) + 1], f, l);
    acc = fmaf(rec[c * (D + kPad) + kPad + d], f, acc);
  }
  const float out = l > 0.f || l != l ? acc / l : 0.f;
  char* o = p.o + (int64_t)b * p.osb + (int64_t)qi * p.osq + (int64_t)h * p.osh;
  if constexpr (DT == SKV_F32)
    reinterpret_cast<float*>(o)[d] = out;
  else
    reinterpret_cast<uint16_t*>(o)[d] = (uint16_t)pack2<DT>(out, 0.f);
}

// ---------------------------------------------------------------------------
// Host.
// ---------------------------------------------------------------------------
constexpr int kChunkUnit = 64;  // chunks are multiples of this many keys

int32_t pick_chunk4(int64_t rows, int32_t heads, int32_t max_ctx) {
  const int64_t units = cdiv(max_ctx > 0 ? max_ctx : 1, kChunkUnit);
  const int64_t items = rows * heads;
  int64_t chunks = items >= 1024 ? 1 : cdiv(1024, items > 0 ? items : 1);
  const int64_t most = cdiv(units, 4);
  chunks = chunks > most ? most : chunks;
  return (int32_t)(cdiv(units, chunks) * kChunkUnit);
}

template <int DT, int D>
void launch_attn4(const Int4Attn& p, hipStream_t stream) {
  const uint32_t items = (uint32_t)((int64_t)p.batch * p.qlen * p.heads);
  hipLaunchKernelGGL((attention_int4_kernel<DT, D>), dim3(items, p.nchunk), dim3(64 * kAttnWaves), 0, stream, p);
  if (p.nchunk > 1) hipLaunchKernelGGL((merge_int4_kernel<DT, D>), dim3(items), dim3(D < 64 ? 64 : D), 0, stream, p);
}
template <int DT>
void launch_attn4_d(int d, const Int4Attn& p, hipStream_t stream) {
  if (d == 32)
    launch_attn4<DT, 32>(p, stream);
  else if (d == 64)
    launch_attn4<DT, 64>(p, stream);
  else
    launch_attn4<DT, 128>(p, stream);
}

template <int DT, int D>
void launch_append4(const Int4Append& a, hipStream_t stream) {
  const uint32_t blocks = (uint32_t)(cdiv(a.total, 256) < 65535 ? cdiv(a.total, 256) : 65535);
  if (a.r.interleaved)
    hipLaunchKernelGGL((append_int4_kernel<DT, D, true>), dim3(blocks), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((append_int4_kernel<DT, D, false>), dim3(blocks), dim3(256), 0, stream, a);
}
template <int DT>
void launch_append4_d(int d, const Int4Append& a, hipStream_t stream) {
  if (d == 32)
    launch_append4<DT, 32>(a, stream);
  else if (d == 64)
    launch_append4<DT, 64>(a, stream);
  else
    launch_append4<DT, 128>(a, stream);
}

struct Int4Gather {
  const char *k_pool, *v_pool;
  const int32_t* tables;
  int64_t tstride;
  const int32_t* lens;
  char *k_out, *v_out;
  uint32_t total;
  DivU32 quads, heads;
  int32_t tiles, nb, max_len;
};
template <int DT, int D>
void launch_gather4(const Int4Gather& a, hipStream_t stream) {
  const uint32_t blocks = (uint32_t)(cdiv(a.total, 256) < 65535 ? cdiv(a.total, 256) : 65535);
  hipLaunchKernelGGL((gather_int4_kernel<DT, D>), dim3(blocks, 2), dim3(256), 0, stream, a.k_pool, a.v_pool, a.tables,
                     a.tstride, a.lens, a.k_out, a.v_out, a.total, a.quads, a.heads, a.tiles, a.nb, a.max_len);
}
template <int DT>
void launch_gather4_d(int d, const Int4Gather& a, hipStream_t stream) {
  if (d == 32)
    launch_gather4<DT, 32>(a, stream);
  else if (d == 64)
    launch_gather4<DT, 64>(a, stream);
  else
    launch_gather4<DT, 128>(a, stream);
}

// What every call asks of a 4-bit pool.
int check_pool(const char* who, const void* k_pool, const void* v_pool, int32_t kv_heads, int32_t d, int32_t bs, int64_t nb) {
  if (!supported_d4(d)) return fail(SKV_EINVAL, "%s: head_dim %d not in {32,64,128}", who, d);
  if (kv_heads <= 0 || kv_heads > 65535 || nb < 0 || bs <= 0 || bs % kTile)
    return fail(SKV_EINVAL, "%s: bad pool kv_heads=%d num_blocks=%lld block_size=%d (a multiple of %d)", who, kv_heads,
                (long long)nb, bs, kTile);
  if (!k_pool || !v_pool) return fail(SKV_EINVAL, "%s: null pool", who);
  if (!aligned16(k_pool) || !aligned16(v_pool)) return fail(SKV_EALIGN, "%s: pools must be 16-byte aligned", who);
  return SKV_OK;
}

}  // namespace

extern "C" {

int skv_append_int4(const void* q, int64_t q_stride_n, int64_t q_stride_h, const void* k_new, int64_t k_stride_n,
                    int64_t k_stride_h, const void* v_new, int64_t v_stride_n, int64_t v_stride_h, void* q_out,
                    int64_t qo_stride_n, int64_t qo_stride_h, void* k_out, int64_t ko_stride_n, int64_t ko_stride_h,
                    void* k_pool, void* v_pool, const int64_t* slot_mapping, const int64_t* positions,
                    const float* cos_sin, int64_t num_positions, int32_t rot_dim, int32_t interleaved, int32_t n_tokens,
                    int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int32_t num_blocks,
                    int32_t dtype, void* stream) {
  const char* who = "skv_append_int4";
  const int eb = elt_bytes(dtype);
  if (eb == 0) return fail(SKV_EDTYPE, "%s: unknown dtype %d", who, dtype);
  if (n_tokens < 0 || num_positions < 0 || (q && num_heads <= 0))
    return fail(SKV_EINVAL, "%s: bad sizes n=%d heads=%d positions=%lld", who, n_tokens, num_heads, (long long)num_positions);
  int rc = check_pool(who, k_pool, v_pool, num_kv_heads, head_dim, block_size, num_blocks);
  if (rc != SKV_OK) return rc;
  if (cos_sin && (rot_dim <= 0 || rot_dim > head_dim || rot_dim % 16))
    return fail(SKV_EINVAL, "%s: rot_dim %d must be a multiple of 16, at most head_dim %d", who, rot_dim, head_dim);
  if (n_tokens == 0) return SKV_OK;
  if (!k_new || !v_new || !slot_mapping || (cos_sin && !positions) || (q == nullptr) != (q_out == nullptr) ||
      (!cos_sin && (q || k_out)))
    return fail(SKV_EINVAL, "%s: null pointer argument (q, q_out and k_out come with cos_sin; q and q_out together)", who);
  if (!aligned16(q) || !aligned16(k_new) || !aligned16(v_new) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(cos_sin))
    return fail(SKV_EALIGN, "%s: pointers must be 16-byte aligned", who);
  int64_t odd = k_stride_n | k_stride_h | v_stride_n | v_stride_h;
  if (q) odd |= q_stride_n | q_stride_h | qo_stride_n | qo_stride_h;
  if (k_out) odd |= ko_stride_n | ko_stride_h;
  if (odd % (16 / eb)) return fail(SKV_EALIGN, "%s: strides must be multiples of %d elements", who, 16 / eb);
  Int4Append a{};
  const int64_t lanes = ((q ? num_heads : 0) + 2 * (int64_t)num_kv_heads) * (head_dim / 8);
  if (lanes >= (int64_t)1 << 30) return fail(SKV_EINVAL, "%s: too many heads", who);
  a.per_tok = make_div((uint32_t)lanes);
  a.tiles = make_div((uint32_t)(block_size / kTile));
  a.q_heads = q ? num_heads : 0;
  a.kv_heads = num_kv_heads;
  a.k_pool = (char*)k_pool;
  a.v_pool = (char*)v_pool;
  a.num_slots = (int64_t)num_blocks * block_size;
  a.r = {cos_sin, positions, num_positions, rot_dim, interleaved ? 1 : 0};
  // Indices of a launch stay below 2^31: longer batches go in slices of tokens.
  const int64_t slice = (((int64_t)1 << 31) - 1) / lanes;
  for (int64_t n0 = 0; n0 < n_tokens; n0 += slice) {
    const int64_t n = n_tokens - n0 < slice ? n_tokens - n0 : slice;
    auto rows = [&](const void* p, int64_t sn, int64_t sh) {
      return Rows{p ? (const char*)p + n0 * sn * eb : nullptr, sn * eb, sh * eb};
    };
    a.q = rows(q, q_stride_n, q_stride_h);
    a.k = rows(k_new, k_stride_n, k_stride_h);
    a.v = rows(v_new, v_stride_n, v_stride_h);
    a.qo = rows(q_out, qo_stride_n, qo_stride_h);
    a.ko = rows(k_out, ko_stride_n, ko_stride_h);
    a.slots = slot_mapping + n0;
    a.r.positions = positions ? positions + n0 : nullptr;
    a.total = (uint32_t)(n * lanes);
    switch (dtype) {
      case SKV_F32: launch_append4_d<SKV_F32>(head_dim, a, (hipStream_t)stream); break;
      case SKV_F16: launch_append4_d<SKV_F16>(head_dim, a, (hipStream_t)stream); break;
      default: launch_append4_d<SKV_BF16>(head_dim, a, (hipStream_t)stream); break;
    }
    rc = check_launch(who);
    if (rc != SKV_OK) return rc;
  }
  return SKV_OK;
}

int skv_gather_int4(const void* k_pool, const void* v_pool, const int32_t* block_tables, int32_t table_stride,
                    const int32_t* lens, void* k_out, void* v_out, int32_t batch, int32_t num_kv_heads, int32_t head_dim,
                    int32_t block_size, int32_t num_blocks, int32_t max_len, int32_t dtype, void* stream) {
  const char* who = "skv_gather_int4";
  if (elt_bytes(dtype) == 0) return fail(SKV_EDTYPE, "%s: unknown dtype %d", who, dtype);
  if (batch < 0 || max_len < 0) return fail(SKV_EINVAL, "%s: bad sizes batch=%d max_len=%d", who, batch, max_len);
  const int rc = check_pool(who, k_pool, v_pool, num_kv_heads, head_dim, block_size, num_blocks);
  if (rc != SKV_OK) return rc;
  if (batch == 0 || max_len == 0) return SKV_OK;
  if (!block_tables || !lens || !k_out || !v_out || table_stride <= 0)
    return fail(SKV_EINVAL, "%s: null pointer argument or empty table", who);
  if (max_len > (int64_t)table_stride * block_size)
    return fail(SKV_EINVAL, "%s: max_len %d past the table's %lld positions", who, max_len, (long long)table_stride * block_size);
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(SKV_EALIGN, "%s: outputs must be 16-byte aligned", who);
  const int64_t quads = cdiv(max_len, 4), per_row = (int64_t)num_kv_heads * quads * (head_dim / 8);
  if (per_row >= (int64_t)1 << 31) return fail(SKV_EINVAL, "%s: a row of %lld vectors is too large", who, (long long)per_row);
  const int64_t slice = (((int64_t)1 << 31) - 1) / per_row;
  const int64_t out_bytes = (int64_t)num_kv_heads * max_len * head_dim * elt_bytes(dtype);
  for (int64_t b0 = 0; b0 < batch; b0 += slice) {
    const int64_t n = batch - b0 < slice ? batch - b0 : slice;
    const Int4Gather a{(const char*)k_pool, (const char*)v_pool, block_tables + b0 * table_stride, table_stride, lens + b0,
                       (char*)k_out + b0 * out_bytes, (char*)v_out + b0 * out_bytes, (uint32_t)(n * per_row),
                       make_div((uint32_t)quads), make_div((uint32_t)num_kv_heads), block_size / kTile, num_blocks, max_len};
    switch (dtype) {
      case SKV_F32: launch_gather4_d<SKV_F32>(head_dim, a, (hipStream_t)stream); break;
      case SKV_F16: launch_gather4_d<SKV_F16>(head_dim, a, (hipStream_t)stream); break;
      default: launch_gather4_d<SKV_BF16>(head_dim, a, (hipStream_t)stream); break;
    }
    const int e = check_launch(who);
    if (e != SKV_OK) return e;
  }
  return SKV_OK;
}

int32_t skv_int4_chunk_tokens(int32_t batch, int32_t q_len, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                              int32_t max_ctx, int32_t dtype) {
  if (batch <= 0 || q_len <= 0 || num_heads <= 0) return kChunkUnit;
  return pick_chunk4((int64_t)batch * q_len, num_heads, max_ctx);
}

int64_t skv_int4_workspace_bytes(int32_t batch, int32_t q_len, int32_t num_heads, int32_t head_dim, int32_t max_ctx,
                                 int32_t chunk_tokens) {
  if (batch <= 0 || q_len <= 0 || num_heads <= 0 || head_dim <= 0 || max_ctx <= 0 || chunk_tokens <= 0) return 0;
  const int64_t n = cdiv(max_ctx, chunk_tokens);
  return n <= 1 ? 0 : (int64_t)batch * q_len * num_heads * n * (head_dim + kPad) * (int64_t)sizeof(float);
}

int skv_paged_attention_int4(const void* q, int64_t q_stride_b, int64_t q_stride_q, int64_t q_stride_h,
                             const void* k_pool, const void* v_pool, const int32_t* block_tables, int32_t table_stride,
                             const int32_t* table_rows, const int32_t* ctx_lens, void* out, int64_t o_stride_b,
                             int64_t o_stride_q, int64_t o_stride_h, int32_t batch, int32_t q_len, int32_t num_heads,
                             int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int32_t num_blocks,
                             int32_t max_ctx, float scale, int32_t causal, int32_t dtype, int32_t chunk_tokens,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "skv_paged_attention_int4";
  const int eb = elt_bytes(dtype);
  if (eb == 0) return fail(SKV_EDTYPE, "%s: unknown dtype %d", who, dtype);
  int rc = check_pool(who, k_pool, v_pool, num_kv_heads, head_dim, block_size, num_blocks);
  if (rc != SKV_OK) return rc;
  if (batch < 0 || q_len <= 0 || q_len > 65535 || num_heads <= 0 || num_heads > 65535 || num_heads % num_kv_heads ||
      max_ctx < 0 || table_stride <= 0)
    return fail(SKV_EINVAL, "%s: bad sizes batch=%d q_len=%d heads=%d kv_heads=%d max_ctx=%d table_stride=%d", who, batch,
                q_len, num_heads, num_kv_heads, max_ctx, table_stride);
  if (batch == 0) return SKV_OK;
  if (!q || !out || !block_tables || !ctx_lens) return fail(SKV_EINVAL, "%s: null pointer argument", who);
  const int epl = 16 / eb;
  if (!aligned16(q) || !aligned16(out)) return fail(SKV_EALIGN, "%s: q and out must be 16-byte aligned", who);
  if ((q_stride_b | q_stride_q | q_stride_h | o_stride_b | o_stride_q | o_stride_h) % epl)
    return fail(SKV_EALIGN, "%s: strides must be multiples of %d elements", who, epl);
  const int64_t cap = (int64_t)table_stride * block_size;
  if (max_ctx > cap) max_ctx = (int32_t)cap;
  if (chunk_tokens <= 0)
    chunk_tokens = skv_int4_chunk_tokens(batch, q_len, num_heads, num_kv_heads, head_dim, max_ctx, dtype);
  if (chunk_tokens % kChunkUnit)
    return fail(SKV_EINVAL, "%s: chunk_tokens %d must be a multiple of %d", who, chunk_tokens, kChunkUnit);
  Int4Attn p{};
  p.nchunk = max_ctx > 0 ? (int32_t)cdiv(max_ctx, chunk_tokens) : 1;
  if ((int64_t)batch * q_len * num_heads >= (int64_t)1 << 24 || p.nchunk > 65535)
    return fail(SKV_EINVAL, "%s: launch too large (rows * heads = %lld, chunks = %d)", who,
                (long long)batch * q_len * num_heads, p.nchunk);
  const int64_t need = skv_int4_workspace_bytes(batch, q_len, num_heads, head_dim, max_ctx, chunk_tokens);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(SKV_EWORKSPACE, "%s: workspace needs %lld bytes (16-byte aligned), got %lld", who, (long long)need,
                (long long)workspace_bytes);
  p.q = (const char*)q;
  p.o = (char*)out;
  p.qsb = q_stride_b * eb, p.qsq = q_stride_q * eb, p.qsh = q_stride_h * eb;
  p.osb = o_stride_b * eb, p.osq = o_stride_q * eb, p.osh = o_stride_h * eb;
  p.k_pool = (const char*)k_pool;
  p.v_pool = (const char*)v_pool;
  p.tables = block_tables;
  p.trows = table_rows;
  p.lens = ctx_lens;
  p.tstride = table_stride;
  p.part = (float*)workspace;
  p.scale_log2 = scale * kLog2e;
  p.batch = batch, p.qlen = q_len, p.heads = num_heads, p.kv_heads = num_kv_heads, p.group = num_heads / num_kv_heads;
  p.tiles = block_size / kTile, p.nb = num_blocks, p.max_ctx = max_ctx, p.causal = causal ? 1 : 0, p.chunk = chunk_tokens;
  switch (dtype) {
    case SKV_F32: launch_attn4_d<SKV_F32>(head_dim, p, (hipStream_t)stream); break;
    case SKV_F16: launch_attn4_d<SKV_F16>(head_dim, p, (hipStream_t)stream); break;
    default: launch_attn4_d<SKV_BF16>(head_dim, p, (hipStream_t)stream); break;
  }
  return check_launch(who);
}

}  // extern "C"
