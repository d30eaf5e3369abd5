// The paged 4-bit K/V cache: append (with the position rotation on the way), gather, attention.
//
// Format. Each 32 consecutive dims of a (token, head) row share fp16 (scale, low); an element is low + scale * code with
// code = round((x - low) / scale) in 0..15, low = fp16(min x), scale = fp16((max x - low) * (1 / 15)): 5 bits an element. Values
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

#include <type_traits>

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
  Rows k, v, ko;
  char *k_pool, *v_pool;
  const int64_t* slots;
  int64_t num_slots;
  Rotary r;
  DivU32 per_quad;  // lanes of 4 tokens
  uint32_t total, n;
  int32_t kv_heads;
  uint32_t blocks;  // workgroups of K and V; the others rotate q
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

template <int OFF> __device__ __forceinline__ uint32_t xor_bits(uint32_t x) {
  return __float_as_uint(xor_lane<OFF>(__uint_as_float(x)));
}
__device__ __forceinline__ float min_score(float a, float b) { return __builtin_elementwise_minimum(a, b); }
// Sum without a product ahead of it fused in.
__device__ __forceinline__ float rounded_sum(float a, float b) {
#pragma clang fp contract(off)
  return a + b;
}
// 1 / s of an fp16 value, correctly rounded: the residual of a reciprocal that is off by an ulp at most, times it (held against
// the division for every fp16 number).
__device__ __forceinline__ float reciprocal(float s) {
  const float r = __builtin_amdgcn_rcpf(s);
  return fmaf(fmaf(-s, r, 1.f), r, r);
}

// K and V: one lane per 8 dims of a row, D / 8 lanes (4 to 16) per row, the rows of 4 consecutive tokens side by side (16 to 64
// lanes, never across a wave). A rotated row's lanes all load before any stores, so k may be rotated in place. The codes are
// taken from the rotated values rounded to the rows' type, what a 16-bit cache would hold. Where the 4 tokens fill a quad of a V
// tile (a prompt's do), their lanes exchange bytes and store whole words. q rows go to workgroups of their own.
// What bounds it: about 210 vector operations for a lane's 8 values (range, codes, words), as much as the bytes: bf16 16000 rows
// of 20 x 64 28-30 us (3.6-3.9 TB/s; 36 with bytes stored one by one and divisions), 8192 tokens rotated with 32 / 8 heads x 128 43 us.
template <int DT, int D, bool INTERLEAVED>
__global__ __launch_bounds__(256) void append_int4_kernel(Int4Append a, RotaryAppend q) {
  if (blockIdx.x >= a.blocks) {
    rotate_rows<DT, INTERLEAVED>(q, (blockIdx.x - a.blocks) * 256u + threadIdx.x, (gridDim.x - a.blocks) * 256u);
    return;
  }
  constexpr int LPR = D / 8;
  for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < a.total; i += a.blocks * 256u) {
    const uint32_t n4 = udiv(i, a.per_quad);
    const uint32_t u = i - n4 * a.per_quad.d;
    const int c = (int)(u % LPR), k = (int)(u / LPR % 4);
    const int head = (int)(u / (4 * LPR));
    const bool there = 4 * n4 + k < a.n;  // the last quad may be short: its missing rows are computed and not stored
    const uint32_t n = min(4 * n4 + k, a.n - 1);
    const bool is_v = head >= a.kv_heads;
    const int h = is_v ? head - a.kv_heads : head;
    const Rows src = is_v ? a.v : a.k;
    const char* row = src.p + (int64_t)n * src.sn + (int64_t)h * src.sh;
    const int64_t slot = a.slots[n];
    float f[8];
    load8<DT>(row, c, f);
    bool known = true;
    if (a.r.table) {
      const int64_t pos = a.r.positions[n];
      known = pos >= 0 && pos < a.r.num_positions;
      if (!is_v) {
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
        if (a.ko.p && there) store8<DT>(const_cast<char*>(a.ko.p) + (int64_t)n * a.ko.sn + (int64_t)h * a.ko.sh, c, f);
      }
    }
    // The group's range, over its 4 lanes. NaN carries through these, so one test finds what has to be taken in first.
    float lo = f[0], hi = f[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      lo = min_score(lo, f[e]);
      hi = max_score(hi, f[e]);
    }
    if (__builtin_amdgcn_ballot_w64(!(lo >= -kLimit && hi <= kLimit)) != 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = f[e] != f[e] ? 0.f : fminf(fmaxf(f[e], -kLimit), kLimit);
        lo = e == 0 ? f[0] : fminf(lo, f[e]);
        hi = e == 0 ? f[0] : fmaxf(hi, f[e]);
      }
    }
    lo = min_score(lo, xor_lane<1>(lo));
    hi = max_score(hi, xor_lane<1>(hi));
    lo = min_score(lo, xor_lane<2>(lo));
    hi = max_score(hi, xor_lane<2>(hi));
    const uint32_t low_h = to_half_bits(lo);
    const float low = half_bits(low_h);
    const uint32_t scale_h = to_half_bits(fmaxf((hi - low) * (1.f / 15.f), 0.f));
    const float scale = half_bits(scale_h);
    const float inv = scale > 0.f ? reciprocal(scale) : 0.f;
    // round((x - low) / scale) in the low bits of 1.5 * 2^23 + it, clamped there as integers; words of 8 are sums, the constant
    // part taken off at the end.
    constexpr uint32_t kBase = 0x4b400000u, kBases = kBase * 0x11111111u;
    uint32_t code[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int bits = __float_as_int(rounded_sum((f[e] - low) * inv, 12582912.f));
      code[e] = (uint32_t)min(max(bits, (int)kBase), (int)kBase + 15);
    }
    uint32_t word;
    if (is_v)  // byte y: dims 2y, 2y + 1
      word = code[0] + (code[1] << 4) + (code[2] << 8) + (code[3] << 12) + (code[4] << 16) + (code[5] << 20) +
             (code[6] << 24) + (code[7] << 28) - kBases;
    else
      word = code[0] + (code[2] << 4) + (code[4] << 8) + (code[6] << 12) + (code[1] << 16) + (code[3] << 20) +
             (code[5] << 24) + (code[7] << 28) - kBases;
    const uint32_t meta = scale_h | low_h << 16;
    const bool stored = there && known && slot >= 0 && slot < a.num_slots;
    // Token k's byte y of a V word to lane y's byte k, over the lanes of the 4 tokens; and the (scale, low) of tokens k, k + 2.
    const uint32_t far = xor_bits<2 * LPR>(word);
    const uint32_t half = __builtin_amdgcn_perm(far, word, k < 2 ? 0x05040100u : 0x03020706u);
    const uint32_t near = xor_bits<LPR>(half);
    const uint32_t quad_word = __builtin_amdgcn_perm(near, half, (k & 1) == 0 ? 0x06020400u : 0x03070105u);
    const uint32_t meta2 = xor_bits<2 * LPR>(meta);
    // Whether the 4 tokens go to the 4 places of one quad in their order.
    const uint32_t key = stored && ((uint32_t)slot & 3u) == (uint32_t)k ? (uint32_t)(slot >> 2) : ~(uint32_t)k;
    const uint32_t key2 = xor_bits<2 * LPR>(key);
    const uint32_t key1 = xor_bits<LPR>(key), key3 = xor_bits<LPR>(key2);  // in all lanes: an && would leave some out
    const bool whole = key == key1 && key == key2 && key == key3;
    if (!stored) continue;
    // slot = (block * tiles + tile of the block) * 16 + token; a (block, head) has tiles.d tiles.
    const uint32_t tile = (uint32_t)(slot >> 4);
    const int t = (int)(slot & 15);
    const uint32_t blk = udiv(tile, a.tiles);
    const int64_t at = (((int64_t)blk * a.kv_heads + h) * a.tiles.d + (tile - blk * a.tiles.d)) * (10 * D);
    if (!is_v) {
      char* o = a.k_pool + at;
      *reinterpret_cast<uint32_t*>(o + t * (D / 2) + 4 * c) = word;
      if ((c & 3) == 0) *reinterpret_cast<uint32_t*>(o + 8 * D + (t * (D / kGroup) + c / 4) * 4) = meta;
    } else {
      char* o = a.v_pool + at;
      const int quad = t >> 2;
      char* data = o + quad * 2 * D + 16 * c;
      char* m = o + 8 * D + (quad * (D / kGroup) + c / 4) * 16;
      if (whole) {
        *reinterpret_cast<uint32_t*>(data + 4 * k) = quad_word;
        if ((c & 3) == 0 && k < 2) {  // tokens 0, 2 and 1, 3
          *reinterpret_cast<uint32_t*>(m + 4 * k) = __builtin_amdgcn_perm(meta2, meta, 0x05040100u);
          *reinterpret_cast<uint32_t*>(m + 8 + 4 * k) = __builtin_amdgcn_perm(meta2, meta, 0x07060302u);
        }
      } else {
        const int tk = t & 3;
#pragma unroll
        for (int y = 0; y < 4; ++y) data[4 * y + tk] = (char)(word >> (8 * y));
        if ((c & 3) == 0) {
          m += 2 * ((tk & 1) * 2 + (tk >> 1));
          *reinterpret_cast<uint16_t*>(m) = (uint16_t)scale_h;
          *reinterpret_cast<uint16_t*>(m + 8) = (uint16_t)low_h;
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Gather: out[b, h, t, :] = the values of position t of row b for t < lens[b], zero otherwise.
// ---------------------------------------------------------------------------
// One thread per 8 dims of 4 tokens (a quad) of one head, of K (grid.y 0) or V (1): V's words hold 4 tokens. Bound by the bytes it
// writes: bf16 16 rows to 1500 of 20 x 64, 149 MB, 23.5 us (6.3 TB/s).
template <int DT, int D>
__global__ __launch_bounds__(256) void gather_int4_kernel(const char* k_pool, const char* v_pool, const int32_t* tables,
                                                          int64_t tstride, const int32_t* lens, char* k_out, char* v_out,
                                                          uint32_t total, DivU32 quads, DivU32 heads, DivU32 tiles,
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
      const uint32_t tile = (uint32_t)t0 >> 4, blk_i = udiv(tile, tiles), in = tile - blk_i * tiles.d;
      const uint32_t blk = (uint32_t)tables[(int64_t)b * tstride + blk_i];
      if (blk < (uint32_t)nb) {
        const char* p = (is_v ? v_pool : k_pool) + (((int64_t)blk * heads.d + h) * tiles.d + in) * (10 * D);
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

// A wave-uniform word of a table that the kernel does not write: a scalar load.
__device__ __forceinline__ int32_t scalar_word(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
}

// Keys query qi of row b sees.
__device__ __forceinline__ int visible(const Int4Attn& p, int b, int qi) {
  const int len = scalar_word(p.lens + b) - (p.causal ? p.qlen - 1 - qi : 0);
  return min(max(len, 0), p.max_ctx);
}

// One workgroup per (row, query, head, key chunk), everything in fp32: 16-key tiles go to its waves in turn.
// Scores: lane (g, r) takes a quarter of key r's dims. Values: lane m takes dims 2m and 2m + 1 of D / 2 lanes' worth of
// quads. For fp32 rows, whose results are held to fp32's rounding: values are low + scale * code in fp32 before their products
// (codes first, scale after the sum, cancels: 1.4e-7 of the results' rms from float64 at 4 keys, now 0.65e-7). Bound by its vector
// operations: 4 rows x 2000 keys, 8 heads x 64, 8.0 us.
template <int D>
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
    load8<SKV_F32>(q, threadIdx.x, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) s_q[8 * threadIdx.x + e] = f[e];
  }
  __syncthreads();
  float qf[8 * ND];
#pragma unroll
  for (int e = 0; e < 8 * ND; ++e) qf[e] = s_q[g * 8 * ND + e];
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
    const uint32_t km = *reinterpret_cast<const uint32_t*>(kt + 8 * D + (r * (D / kGroup) + g * 8 * ND / kGroup) * 4);
    const float k_scale = half_bits(km & 0xffffu), k_low = half_bits(km >> 16);
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(kt + r * (D / 2) + (g * ND + i) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s = fmaf(qf[8 * i + 2 * e], fmaf(k_scale, (float)((w >> (4 * e)) & 15u), k_low), s);
        s = fmaf(qf[8 * i + 2 * e + 1], fmaf(k_scale, (float)((w >> (4 * e + 16)) & 15u), k_low), s);
      }
    }
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
  reinterpret_cast<float*>(p.o + (int64_t)b * p.osb + (int64_t)qi * p.osq + (int64_t)h * p.osh)[d] = out;
}

// 16-bit rows on the matrix cores. One workgroup per (row, KV head, 16 queries, key chunk): the queries are those of the
// head's whole group, so its keys are read once for all of them; its waves take 32-key steps in turn and join at the end.
// Codes become fp16 in two operations: shifted and masked under the exponent of 16 they are 16 + code exactly.
//   S^T = K Q^T: lane (g, r) unpacks 8 dims of key r, the operand of one product per 32 dims that share a scale, whose
//     results (keys 4 g + i of query r) take that scale in fp32; it reaches them from the lane of the 16 that loaded it. One
//     more product adds low and takes off 16 scale, against the sums of q over each 32 dims: K is exact.
//   O^T = V^T P^T: the lane's 8 weights are the operand P^T (keys 4 g + 0, 2, 1, 3 of both tiles), and it unpacks those keys'
//     dims [r D / 16, + D / 16) of V, one operand per dim. There the scale belongs to the contraction, so V's own operand takes
//     it: scale * (16 + code) + z in one fma, z = fp16(-24 scale), is the value about the group's middle, rounded once (2^-11
//     of it, what a cache in fp16 rounds too). The rest, low - 16 scale - z, is the group's own and one product more.
// Both products run in fp16 whatever the rows' type: queries are first scaled by a power of two that brings their greatest
// element to [0.5, 1), which the scores' factor takes back. Weights (times 2^6, clear of fp16's subnormals) go in as a
// rounded head and its rounded remainder; their sum is one more row of the product.
// fp16, 300 keys: 2.7e-4 of the results' rms from float64, where rounding exact ones is 2.1e-4 (with K's scale in its operand
// as well 3.6e-4, with weights rounded once 3.3e-4, with low - 16 scale rounded into the fma 25e-4).
// What bounds it: HBM and the vector operations alike on long rows (about 3.3 an element at head_dim 128, half of them to unpack),
// for few keys the chain lengths -> table -> keys -> join. bf16 unless said, 32 / 8 heads x 128: 32 rows of 1000..16384 keys 83 us
// (4.3 TB/s), fp16 one row of 131072 keys 34 us (5.0 TB/s); 20 heads x 64: 16 x 4096 keys 27 us (3.9 TB/s), 64 rows of 1..452 keys 12.8.
constexpr float kLazyMaxLog2 = 8.f;  // the accumulators are rescaled when a maximum grows by more than this
constexpr float kWeightLog2 = 6.f;   // weights below 2^(8 + 6)

__device__ __forceinline__ uint32_t pk_fma(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2v, a), __builtin_bit_cast(half2v, b),
                                                                __builtin_bit_cast(half2v, c)));
}
// 16 + code of nibbles K and K + 4 of w. mask and base are kCodeMask and kCodeBase in registers, which lets one instruction
// do both.
constexpr uint32_t kCodeMask = 0x03c003c0u, kCodeBase = 0x4c004c00u;
template <int K>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, uint32_t mask, uint32_t base) {
  const uint32_t x = K == 0 ? w << 6 : (K == 1 ? w << 2 : (K == 2 ? w >> 2 : w >> 6));
  return (x & mask) | base;
}
// All 8 codes of w with one shift, for a product that can take off different bases: 1024 + code of dims 0, 1, 4, 5 (nibbles 0,
// 4, 2, 6), 64 + code of dims 2, 3, 6, 7.
struct CodeRegs {
  uint32_t low, base_low, high, base_high;
};
__device__ __forceinline__ uint4 code_row(uint32_t w, const CodeRegs& c) {
  const uint32_t x = w >> 8;
  return make_uint4((w & c.low) | c.base_low, (w & c.high) | c.base_high, (x & c.low) | c.base_low, (x & c.high) | c.base_high);
}
// z of a pair of scales, and what remains of their groups' values: low - 16 scale - z as (low + 8 scale) - (24 scale + z),
// whose second part is exact.
__device__ __forceinline__ uint32_t code_zero(uint32_t scale) { return pk_fma(scale, 0xce00ce00u, 0x80008000u); }
__device__ __forceinline__ uint32_t middles(uint32_t low, uint32_t scale, uint32_t z) {
  const uint32_t mid = pk_fma(scale, 0x48004800u, low), err = pk_fma(scale, 0x4e004e00u, z);
  return pk_fma(err, 0xbc00bc00u, mid);
}
// a + b * (x of lane L of this lane's 16).
template <int L>
__device__ __forceinline__ float fma_row_lane(float x, float b, float a) {
  return fmaf(__int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x150 + L, 0xf, 0xf, true)), b, a);
}

// The dwords of a key's row, ND consecutive ones per lane group as loaded, dealt out so that lane group g of word G holds one
// of group G's four (dword 4 G + g; with two words in the order 0, 2, 1, 3).
template <int ND>
__device__ __forceinline__ void deal_words(uint32_t (&w)[ND]) {
  auto swap32 = [](uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
  };
  auto swap16 = [](uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0], b = r[1];
  };
  if constexpr (ND == 4) {
    swap32(w[0], w[2]);
    swap32(w[1], w[3]);
    swap16(w[0], w[1]);
    swap16(w[2], w[3]);
  } else if constexpr (ND == 2) {
    swap32(w[0], w[1]);
  }
}

template <int N>
struct Words {
  uint32_t w[N];
};
template <int N>
__device__ __forceinline__ Words<N> load_words(__amdgpu_buffer_rsrc_t tile, uint32_t off) {
  Words<N> r;
  if constexpr (N == 4) {
    const uint4 v = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(tile, off, 0, 0));
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(tile, off, 0, 0));
    r.w[0] = v.x, r.w[1] = v.y;
  } else {
    r.w[0] = __builtin_amdgcn_raw_buffer_load_b32(tile, off, 0, 0);
  }
  return r;
}

// One tile of a pool: loads at 32-bit lane offsets from a scalar base (with plain pointers the compiler kept the sums of pool and
// lane offset, two vector registers each, and added the tile's offset to them every step).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_at(const char* pool, uint64_t at, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(pool + at), (short)0, bytes, kBufWord3);
}

// What a wave holds of one step: two 16-key tiles.
template <int ND>
struct Step4 {
  Words<ND> k[2];      // dwords ND g .. of key r
  Words<ND> v[2];
  uint32_t ks[2];      // (scale, low) of the lane's place in the row's [4 keys][ND]
  uint32_t kr[2];      // (scale, low) of key r, group g
  uint4 vm[2];         // scales and lows of quad g, the group of the lane's dims
};

struct Int4Divs {
  DivU32 kv_heads, qtiles, group, tiles;
};

// The sum of x over the 4 lane groups (a permlane swap of a register with itself leaves a lane's own value in one result, its
// partner's in the other).
__device__ __forceinline__ float sum_groups(float x) {
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r16[0]) + __uint_as_float(r16[1]);
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r32[0]) + __uint_as_float(r32[1]);
}
__device__ __forceinline__ float max_groups(float x) {
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = max_score(__uint_as_float(r16[0]), __uint_as_float(r16[1]));
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max_score(__uint_as_float(r32[0]), __uint_as_float(r32[1]));
}

template <int DT, int D>
__global__ __launch_bounds__(64 * kAttnWaves, D == 128 ? 4 : 5) void attention_int4_mfma_kernel(Int4Attn p, Int4Divs dv) {
  constexpr int WAVES = kAttnWaves;
  constexpr int ND = D / 32;
  constexpr int NB = D / 16;     // 16-row blocks of the result
  constexpr int STEP = 2 * kTile;
  constexpr int ACC = D + 4;     // floats of a query's accumulators in LDS
  extern __shared__ __attribute__((aligned(16))) float s_mem[];  // [waves][queries] (max, sum), then [waves][queries][ACC]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int g = lane >> 4, r = lane & 15;
  const int rest = (int)udiv(blockIdx.x, dv.kv_heads);
  const int kvh = (int)blockIdx.x - rest * p.kv_heads;
  const int b = (int)udiv(rest, dv.qtiles);
  const int qt = rest - b * (int)dv.qtiles.d;
  const int chunk = blockIdx.y;
  const int rows = p.group * p.qlen;       // queries of the KV head
  const int count = min(16, rows - qt * 16);  // of this workgroup
  const int last_q = (int)udiv(qt * 16 + count - 1, dv.group);
  // The queries' loads go out first: vector loads return in order, and the keys' behind them are what takes long.
  const int x = min(qt * 16 + r, rows - 1);
  const int qi = (int)udiv(x, dv.group), h = kvh * p.group + x - qi * p.group;
  uint4 q_raw[ND];
  {
    const char* q = p.q + (int64_t)b * p.qsb + (int64_t)qi * p.qsq + (int64_t)h * p.qsh;
#pragma unroll
    for (int i = 0; i < ND; ++i)  // dims 32 i + 8 times deal_words' order of g
      q_raw[i] = *reinterpret_cast<const uint4*>(q + 16 * (4 * i + (ND == 2 ? (g & 1) * 2 + (g >> 1) : g)));
  }
  const int lim = p.nb > 0 ? visible(p, b, last_q) : 0;  // keys any of its queries sees
  const int t_begin = chunk * p.chunk, t_end = min(lim, t_begin + p.chunk);
  if (t_begin >= lim && chunk > 0) return;
  const int32_t* trow = p.tables + (int64_t)(p.trows ? scalar_word(p.trows + b) : b) * p.tstride;
  const int last_tile = (t_end - 1) >> 4;

  // The two tiles of a step. One behind a block id outside the pool reads block 0 instead and counts for nothing.
  struct Tiles {
    uint64_t at[2];
    bool ok[2];
  };
  const uint64_t head_at = (uint64_t)kvh * p.tiles * (10 * D);
  const uint32_t block_bytes = (uint32_t)(p.kv_heads * p.tiles * (10 * D));
  auto find = [&](int t0) __attribute__((always_inline)) -> Tiles {
    Tiles r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t tile = (uint32_t)min((t0 >> 4) + i, last_tile);
      const uint32_t blk_i = udiv(tile, dv.tiles);
      const uint32_t blk = (uint32_t)scalar_word(trow + blk_i);
      r.ok[i] = blk < (uint32_t)p.nb;
      r.at[i] = head_at + (uint64_t)(r.ok[i] ? blk : 0u) * block_bytes + (tile - blk_i * dv.tiles.d) * (10 * D);
    }
    return r;
  };
  using Step = Step4<ND>;
  const uint32_t k_off = r * (D / 2) + g * (D / 8), kr_off = 8 * D + (r * ND + g * ND / 4) * 4;
  const uint32_t ks_off = 8 * D + (g * 4 * ND + r % (4 * ND)) * 4;
  const uint32_t v_off = g * 2 * D + r * (D / 8), vm_off = 8 * D + (g * ND + r * ND / 16) * 16;
  Step cur;
  auto load_k = [&](const Tiles& t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __amdgpu_buffer_rsrc_t k = tile_at(p.k_pool, t.at[i], 10 * D);
      cur.k[i] = load_words<ND>(k, k_off);
      cur.ks[i] = load_words<1>(k, ks_off).w[0];
      cur.kr[i] = load_words<1>(k, kr_off).w[0];
    }
  };
  auto load_v = [&](const Tiles& t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __amdgpu_buffer_rsrc_t v = tile_at(p.v_pool, t.at[i], 10 * D);
      cur.v[i] = load_words<ND>(v, v_off);
      cur.vm[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(v, vm_off, 0, 0));
    }
  };
  // The registers of a step's K take the next step's as soon as they are read, and V's theirs: each load has the other half of a
  // step to arrive in. With a second set of registers instead, waves spilled or were half as many (32 x 16384 keys: 108 and 93 us
  // against 84). Tiles are looked up two steps ahead; those past the end are the last tile again.
  Tiles where{}, then{};
  int t0 = t_begin + wave * STEP;
  if (t0 < t_end) {
    where = find(t0);
    then = find(t0 + WAVES * STEP);
    load_k(where);
    load_v(where);
  }

  const int len0 = scalar_word(p.lens + b);
  auto seen = [&](int q) __attribute__((always_inline)) {
    return min(max(len0 - (p.causal ? p.qlen - 1 - q : 0), 0), p.max_ctx);
  };
  const int mine = min(seen(qi), t_end);   // keys of this chunk this lane's query sees end here
  const int least = min(seen((int)udiv(qt * 16, dv.group)), t_end);
  // Q^T: lane (query r, g) holds 8 dims of product G.
  uint4 qf[ND], qs;
  float c;  // of the scores; positive and finite, as the maximum is taken over unscaled ones and -infinity marks a masked key
  const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
  {
    float f[ND][8], top = 0.f;
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      unpack16<DT>(q_raw[i], f[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max_score(top, fabsf(f[i][e]));
    }
    top = max_groups(top);
    const int ex = top > 0.f && top < __builtin_huge_valf() ? __builtin_amdgcn_frexp_expf(top) : 0;
    c = fminf(fmaxf(ldexpf(fabsf(p.scale_log2), ex), 1.17549435e-38f), 3.4028234664e38f);
    // Of the group whose (scale, low) the lane's kr holds: its sum of q, and of q times the codes' bases.
    float sum = 0.f, based = 0.f;
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      uint32_t w[4];
      float part[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = pack2<SKV_F16>(ldexpf(f[i][2 * e], -ex), ldexpf(f[i][2 * e + 1], -ex)) ^ flip;
        part[e & 1] += lo16<SKV_F16>(w[e]) + hi16<SKV_F16>(w[e]);
      }
      qf[i] = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
      for (int e = 0; e < 2; ++e) part[e] = sum_groups(part[e]);
      if (g * ND / 4 == i) sum = part[0] + part[1], based = -1024.f * part[0] - 64.f * part[1];
    }
    sum *= ND / 4.f;  // 4 / ND lane groups hold one group
    based *= ND / 4.f;
    auto head = [](float v) { return lo16<SKV_F16>(pack2<SKV_F16>(v, 0.f)); };
    const float s0 = head(sum), b0 = head(based), b1 = head(based - b0);
    qs = make_uint4(pack2<SKV_F16>(s0, sum - s0), pack2<SKV_F16>(b0, b1), pack2<SKV_F16>(based - b0 - b1, 0.f), 0u);
  }
  uint32_t code_mask = kCodeMask, code_base = kCodeBase;
  CodeRegs rows_c{0x000f000fu, 0x64006400u, 0x00f000f0u, 0x54005400u};
  asm volatile("" : "+s"(code_mask), "+v"(code_base));
  asm volatile("" : "+s"(rows_c.low), "+s"(rows_c.high), "+v"(rows_c.base_low), "+v"(rows_c.base_high));

  float m = kNegInf, ref = 0.f;
  f32x4 acc[NB], rest_acc = f32x4{0.f, 0.f, 0.f, 0.f};  // rows 4 g: the middles' part of the lane's group; 4 g + 1: the weights' sum
#pragma unroll
  for (int i = 0; i < NB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bool sum_row = (r & 3) == 1;

  while (t0 < t_end) {
    const bool ok0 = where.ok[0], ok1 = where.ok[1];
    const Tiles later = find(t0 + 2 * WAVES * STEP);
    f32x4 s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t low = __builtin_amdgcn_perm(cur.kr[i], cur.kr[i], 0x03020302u);
      const uint32_t scale = __builtin_amdgcn_perm(cur.kr[i], cur.kr[i], 0x01000100u);
      const float sf = lo16<SKV_F16>(cur.ks[i]);
      s[i] = mfma_16x16x32<SKV_F16>(make_uint4(low, scale, scale, 0u), qs, f32x4{0.f, 0.f, 0.f, 0.f});
      f32x4 t[ND];
      deal_words<ND>(cur.k[i].w);
#pragma unroll
      for (int e = 0; e < ND; ++e) {
        const uint32_t w = cur.k[i].w[e];
        t[e] = mfma_16x16x32<SKV_F16>(code_row(w, rows_c), qf[e], f32x4{0.f, 0.f, 0.f, 0.f});
      }
      auto scaled = [&](auto e_c) __attribute__((always_inline)) {
        constexpr int E = decltype(e_c)::value;
        if constexpr (E < ND) {
          s[i][0] = fma_row_lane<E>(sf, t[E][0], s[i][0]);
          s[i][1] = fma_row_lane<ND + E>(sf, t[E][1], s[i][1]);
          s[i][2] = fma_row_lane<2 * ND + E>(sf, t[E][2], s[i][2]);
          s[i][3] = fma_row_lane<3 * ND + E>(sf, t[E][3], s[i][3]);
        }
      };
      scaled(std::integral_constant<int, 0>{});
      scaled(std::integral_constant<int, 1>{});
      scaled(std::integral_constant<int, 2>{});
      scaled(std::integral_constant<int, 3>{});
    }
    load_k(then);
    __builtin_amdgcn_sched_barrier(0);
    // A step with a key that some query does not see, or behind an invalid block id (wave-uniform).
    if (t0 + STEP > least || !(ok0 && ok1)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // What a slot past the row's end holds may be anything: those keys' scales and offsets become zeros, as do those
        // of a tile behind an invalid block id.
        const int base = t0 + kTile * i + 4 * g;
        const int end = (i == 0 ? ok0 : ok1) ? t_end : 0;
        const bool z0 = base >= end, z1 = base + 1 >= end, z2 = base + 2 >= end, z3 = base + 3 >= end;
        const uint32_t m02 = (z0 ? 0u : 0xffffu) | (z2 ? 0u : 0xffff0000u), m13 = (z1 ? 0u : 0xffffu) | (z3 ? 0u : 0xffff0000u);
        cur.vm[i].x &= m02, cur.vm[i].y &= m13, cur.vm[i].z &= m02, cur.vm[i].w &= m13;
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = base + e < min(mine, end) ? s[i][e] : kNegInf;
      }
    }
    float mx = kNegInf;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = max_score(mx, s[i][e]);
    if (__builtin_amdgcn_ballot_w64(mx * c > m + kLazyMaxLog2) != 0) {  // wave-uniform
      mx = max_groups(mx);
      const float mn = max_score(m, mx * c);
      ref = mn == kNegInf ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
      for (int i = 0; i < NB; ++i) acc[i] *= alpha;
      rest_acc *= alpha;
      m = mn;
    }
    float w[8];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[4 * i + e] = __builtin_amdgcn_exp2f(fmaf(s[i][e], c, kWeightLog2 - ref));
    uint32_t head[4], tail[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = 4 * (e >> 1) + (e & 1);  // keys 0, 2 and 1, 3 of each tile
      head[e] = pack2<SKV_F16>(w[k], w[k + 2]);
      tail[e] = pack2<SKV_F16>(fmaf(lo16<SKV_F16>(head[e]), -1.f, w[k]), fmaf(hi16<SKV_F16>(head[e]), -1.f, w[k + 2]));
    }
    const uint4 pt[2] = {make_uint4(head[0], head[1], head[2], head[3]), make_uint4(tail[0], tail[1], tail[2], tail[3])};
    uint32_t z02[2], z13[2], mid[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      z02[i] = code_zero(cur.vm[i].x), z13[i] = code_zero(cur.vm[i].y);
      mid[2 * i] = middles(cur.vm[i].z, cur.vm[i].x, z02[i]);
      mid[2 * i + 1] = middles(cur.vm[i].w, cur.vm[i].y, z13[i]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) mid[e] = sum_row ? 0x3c003c00u : mid[e];
    const uint4 rest_a = make_uint4(mid[0], mid[1], mid[2], mid[3]);
#pragma unroll
    for (int o = 0; o < 2; ++o) rest_acc = mfma_16x16x32<SKV_F16>(rest_a, pt[o], rest_acc);
#pragma unroll
    for (int y = 0; y < ND; ++y) {
      const uint32_t wa = cur.v[0].w[y], wb = cur.v[1].w[y];
      const uint4 even = make_uint4(
          pk_fma(code_pair<0>(wa, code_mask, code_base), cur.vm[0].x, z02[0]), pk_fma(code_pair<2>(wa, code_mask, code_base), cur.vm[0].y, z13[0]),
          pk_fma(code_pair<0>(wb, code_mask, code_base), cur.vm[1].x, z02[1]), pk_fma(code_pair<2>(wb, code_mask, code_base), cur.vm[1].y, z13[1]));
      const uint4 odd = make_uint4(
          pk_fma(code_pair<1>(wa, code_mask, code_base), cur.vm[0].x, z02[0]), pk_fma(code_pair<3>(wa, code_mask, code_base), cur.vm[0].y, z13[0]),
          pk_fma(code_pair<1>(wb, code_mask, code_base), cur.vm[1].x, z02[1]), pk_fma(code_pair<3>(wb, code_mask, code_base), cur.vm[1].y, z13[1]));
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        acc[2 * y] = mfma_16x16x32<SKV_F16>(even, pt[o], acc[2 * y]);
        acc[2 * y + 1] = mfma_16x16x32<SKV_F16>(odd, pt[o], acc[2 * y + 1]);
      }
    }
    load_v(then);
    __builtin_amdgcn_sched_barrier(0);
    t0 += WAVES * STEP;
    where = then;
    then = later;
  }
  const float l = rest_acc[1];
#pragma unroll
  for (int i = 0; i < NB; ++i) acc[i] += rest_acc[0];
  // Lane (g, query r) holds dims (4 g + i) D / 16 + block in acc[block][i].
  float2* s_ml = reinterpret_cast<float2*>(s_mem);
  float* s_acc = s_mem + 2 * WAVES * count;
  if (r < count) {
    if (g == 0) s_ml[wave * count + r] = make_float2(m, l);
    float* a = s_acc + (wave * count + r) * ACC + g * (D / 4);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < NB; ++e) a[i * NB + e] = acc[e][i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count * (D / 2); i += 64 * WAVES) {
    const int y = i / (D / 2), d = 2 * (i % (D / 2));
    float mm = s_ml[y].x;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) mm = max_score(mm, s_ml[w * count + y].x);
    const float base = mm == kNegInf ? 0.f : mm;
    float sum = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float2 ml = s_ml[w * count + y];
      const float f = __builtin_amdgcn_exp2f(ml.x - base);
      const float2 v = *reinterpret_cast<const float2*>(s_acc + (w * count + y) * ACC + d);
      sum = fmaf(ml.y, f, sum);
      a0 = fmaf(v.x, f, a0);
      a1 = fmaf(v.y, f, a1);
    }
    const int xq = qt * 16 + y, oq = (int)udiv(xq, dv.group), oh = kvh * p.group + xq - oq * p.group;
    if (p.nchunk > 1 && seen(oq) > p.chunk) {
      float* rec = p.part + ((((int64_t)b * p.qlen + oq) * p.heads + oh) * p.nchunk + chunk) * (D + kPad);
      *reinterpret_cast<float2*>(rec + kPad + d) = make_float2(a0, a1);
      if (d == 0) *reinterpret_cast<float2*>(rec) = make_float2(mm, sum);
    } else if (chunk == 0) {  // its keys lie in the first chunk
      const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
      *reinterpret_cast<uint32_t*>(p.o + (int64_t)b * p.osb + (int64_t)oq * p.osq + (int64_t)oh * p.osh + 2 * d) =
          pack2<DT>(a0 * inv, a1 * inv);
    }
  }
}

// Rows of several chunks: one workgroup per (row, query, head) joins the chunks' partials, D / 4 lanes a partial, 1024 / D
// partials at once: 4-5 us, most of it the launch (one thread per dim over 128 chunks 59).
template <int DT, int D>
__global__ __launch_bounds__(256) void merge_int4_kernel(Int4Attn p) {
  constexpr int LANES = D / 4, SETS = 256 / LANES;
  __shared__ __attribute__((aligned(16))) float s_acc[SETS][D];
  __shared__ float s_red[8];
  const int h = blockIdx.x % p.heads;
  const int rest = blockIdx.x / p.heads;
  const int qi = rest % p.qlen, b = rest / p.qlen;
  const int len = visible(p, b, qi);
  const int n = (len + p.chunk - 1) / p.chunk;
  if (n <= 1) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* rec = p.part + (((int64_t)b * p.qlen + qi) * p.heads + h) * p.nchunk * (D + kPad);
  float mm = kNegInf;
  for (int c = threadIdx.x; c < n; c += 256) mm = max_score(mm, rec[(int64_t)c * (D + kPad)]);
  mm = max_score(mm, xor_lane<1>(mm));
  mm = max_score(mm, xor_lane<2>(mm));
  mm = max_score(mm, xor_lane<4>(mm));
  mm = max_score(mm, xor_lane<8>(mm));
  mm = max_score(mm, xor_lane<16>(mm));
  mm = max_score(mm, xor_lane<32>(mm));
  if (lane == 0) s_red[wave] = mm;
  __syncthreads();
  mm = max_score(max_score(s_red[0], s_red[1]), max_score(s_red[2], s_red[3]));
  const float ref = mm == kNegInf ? 0.f : mm;
  const int set = threadIdx.x / LANES, d = (threadIdx.x % LANES) * 4;
  float l = 0.f;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int c = set; c < n; c += SETS) {
    const float* r = rec + (int64_t)c * (D + kPad);
    const float f = __builtin_amdgcn_exp2f(r[0] - ref);
    l = fmaf(r[1], f, l);
    acc += f * *reinterpret_cast<const f32x4*>(r + kPad + d);
  }
  *reinterpret_cast<f32x4*>(&s_acc[set][d]) = acc;
  // Each set's sum once: its lanes hold the same.
  __shared__ float s_sum[SETS];
  if (d == 0) s_sum[set] = l;
  __syncthreads();
  if (threadIdx.x >= D) return;
  float out = 0.f, sum = 0.f;
#pragma unroll
  for (int i = 0; i < SETS; ++i) {
    out += s_acc[i][threadIdx.x];
    sum += s_sum[i];
  }
  out = sum > 0.f || sum != sum ? out / sum : 0.f;
  char* o = p.o + (int64_t)b * p.osb + (int64_t)qi * p.osq + (int64_t)h * p.osh;
  if constexpr (DT == SKV_F32)
    reinterpret_cast<float*>(o)[threadIdx.x] = out;
  else
    reinterpret_cast<uint16_t*>(o)[threadIdx.x] = (uint16_t)pack2<DT>(out, 0.f);
}

// ---------------------------------------------------------------------------
// Host.
// ---------------------------------------------------------------------------
constexpr int kChunkUnit = 64;  // chunks are multiples of this many keys

// Workgroups a call has before its keys are split.
int64_t attn4_items(int32_t batch, int32_t q_len, int32_t heads, int32_t kv_heads, int32_t dtype) {
  if (dtype == SKV_F32) return (int64_t)batch * q_len * heads;
  return (int64_t)batch * cdiv((int64_t)(heads / kv_heads) * q_len, 16) * kv_heads;
}

// Key chunk of a call of `items` workgroups before its keys are split: none for short rows (the second launch that joins the
// parts costs 2.5 us) and many items; else one workgroup per compute unit, of 128 to 1024 keys. bf16, one request of
// 8 / 20 KV heads x 128 / 64, us by chunk (the rule's in brackets):
//   8 x 2000 keys     [128] 8.8   256 9.4   512 11.1  unsplit 19.0
//   8 x 8000          128 11.7  [256] 9.7   512 11.5  1024 14.7
//   8 x 32000         256 20.1   512 18.1 [1024] 17.4  2048 24.4
//   20 x 600 (64)     128 7.8    256 8.3   512 9.6    [unsplit] 7.4
//   128 x 1000        256 12.5   512 12.0  [unsplit] 12.2;  320 x 1000 (64) 256 14.2  512 14.2  [unsplit] 12.7
//   256 x 1000..16384 512 95.9 [1024] 87.8  2048 85.8  4096 96.5;  512 x 200..2000 512 31.1  1024 31.4  [unsplit] 28.0
int32_t pick_chunk4(int64_t items, int32_t max_ctx) {
  const int64_t ctx = max_ctx > 0 ? max_ctx : 1;
  if (ctx <= 768 || (ctx <= 1024 && items >= 128) || (ctx <= 2048 && items >= 512))
    return (int32_t)(cdiv(ctx, kChunkUnit) * kChunkUnit);
  const int64_t even = cdiv(items * ctx / 256, kChunkUnit) * kChunkUnit;
  return (int32_t)(even < 128 ? 128 : (even > 1024 ? 1024 : even));
}

template <int DT, int D>
void launch_attn4(const Int4Attn& p, hipStream_t stream) {
  const uint32_t items = (uint32_t)((int64_t)p.batch * p.qlen * p.heads);
  if constexpr (DT != SKV_F32) {
    const int rows = p.group * p.qlen, qtiles = (rows + 15) / 16;
    const uint32_t lds = (uint32_t)(kAttnWaves * (rows < 16 ? rows : 16) * (2 + D + 4) * sizeof(float));
    const Int4Divs dv{make_div((uint32_t)p.kv_heads), make_div((uint32_t)qtiles), make_div((uint32_t)p.group),
                      make_div((uint32_t)p.tiles)};
    hipLaunchKernelGGL((attention_int4_mfma_kernel<DT, D>), dim3((uint32_t)(p.batch * qtiles * p.kv_heads), p.nchunk),
                       dim3(64 * kAttnWaves), lds, stream, p, dv);
  } else {
    hipLaunchKernelGGL((attention_int4_kernel<D>), dim3(items, p.nchunk), dim3(64 * kAttnWaves), 0, stream, p);
  }
  if (p.nchunk > 1) hipLaunchKernelGGL((merge_int4_kernel<DT, D>), dim3(items), dim3(256), 0, stream, p);
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

uint32_t blocks_of(uint32_t total) { return (uint32_t)(cdiv(total, 256) < 32767 ? cdiv(total, 256) : 32767); }

template <int DT, int D>
void launch_append4(Int4Append a, const RotaryAppend& q, hipStream_t stream) {
  a.blocks = blocks_of(a.total);
  const dim3 grid(a.blocks + blocks_of(q.total));
  if (a.r.interleaved)
    hipLaunchKernelGGL((append_int4_kernel<DT, D, true>), grid, dim3(256), 0, stream, a, q);
  else
    hipLaunchKernelGGL((append_int4_kernel<DT, D, false>), grid, dim3(256), 0, stream, a, q);
}
template <int DT>
void launch_append4_d(int d, const Int4Append& a, const RotaryAppend& q, hipStream_t stream) {
  if (d == 32)
    launch_append4<DT, 32>(a, q, stream);
  else if (d == 64)
    launch_append4<DT, 64>(a, q, stream);
  else
    launch_append4<DT, 128>(a, q, stream);
}

struct Int4Gather {
  const char *k_pool, *v_pool;
  const int32_t* tables;
  int64_t tstride;
  const int32_t* lens;
  char *k_out, *v_out;
  uint32_t total;
  DivU32 quads, heads, tiles;
  int32_t nb, max_len;
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
  if (nb * (bs / kTile) > (int64_t)1 << 29) return fail(SKV_EINVAL, "%s: pool of %lld x %d tokens is too large", who, (long long)nb, bs);
  // The attention counts a block's bytes in 32 bits.
  if ((int64_t)kv_heads * (bs / kTile) * (10 * d) >= (int64_t)1 << 31)
    return fail(SKV_EINVAL, "%s: a block of %d heads x %d tokens x %d dims is too large", who, kv_heads, bs, d);
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
  RotaryAppend qa{};  // q rows alone: no K or V heads
  const int epl = 16 / eb;
  const int64_t lanes = 2 * (int64_t)num_kv_heads * (head_dim / 8), pairs = head_dim / (2 * epl);
  const int64_t q_pairs = q ? num_heads * pairs : 1;
  if (lanes >= (int64_t)1 << 28 || q_pairs >= (int64_t)1 << 28) return fail(SKV_EINVAL, "%s: too many heads", who);
  a.per_quad = make_div((uint32_t)(4 * lanes));
  a.tiles = make_div((uint32_t)(block_size / kTile));
  a.kv_heads = num_kv_heads;
  a.k_pool = (char*)k_pool;
  a.v_pool = (char*)v_pool;
  a.num_slots = (int64_t)num_blocks * block_size;
  a.r = {cos_sin, positions, num_positions, rot_dim, interleaved ? 1 : 0};
  qa.per_tok = make_div((uint32_t)q_pairs);
  qa.pairs = make_div((uint32_t)pairs);
  qa.q_heads = q ? num_heads : 0;
  qa.r = a.r;
  // Indices of a launch stay below 2^31: longer batches go in slices of tokens.
  const int64_t most = lanes > q_pairs ? lanes : q_pairs;
  const int64_t slice = (((int64_t)1 << 31) - 1) / (4 * most) * 4;
  for (int64_t n0 = 0; n0 < n_tokens; n0 += slice) {
    const int64_t n = n_tokens - n0 < slice ? n_tokens - n0 : slice;
    auto rows = [&](const void* p, int64_t sn, int64_t sh) {
      return Rows{p ? (const char*)p + n0 * sn * eb : nullptr, sn * eb, sh * eb};
    };
    a.k = rows(k_new, k_stride_n, k_stride_h);
    a.v = rows(v_new, v_stride_n, v_stride_h);
    a.ko = rows(k_out, ko_stride_n, ko_stride_h);
    a.slots = qa.slots = slot_mapping + n0;
    a.r.positions = qa.r.positions = positions ? positions + n0 : nullptr;
    a.n = (uint32_t)n;
    a.total = (uint32_t)(cdiv(n, 4) * 4 * lanes);
    if (q) {
      qa.q = rows(q, q_stride_n, q_stride_h);
      qa.qo = rows(q_out, qo_stride_n, qo_stride_h);
      qa.total = (uint32_t)(n * q_pairs);
    }
    switch (dtype) {
      case SKV_F32: launch_append4_d<SKV_F32>(head_dim, a, qa, (hipStream_t)stream); break;
      case SKV_F16: launch_append4_d<SKV_F16>(head_dim, a, qa, (hipStream_t)stream); break;
      default: launch_append4_d<SKV_BF16>(head_dim, a, qa, (hipStream_t)stream); break;
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
                       make_div((uint32_t)quads), make_div((uint32_t)num_kv_heads), make_div((uint32_t)(block_size / kTile)), num_blocks, max_len};
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
  if (batch <= 0 || q_len <= 0 || num_heads <= 0 || num_kv_heads <= 0) return kChunkUnit;
  return pick_chunk4(attn4_items(batch, q_len, num_heads, num_kv_heads, dtype), max_ctx);
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
  if (max_ctx > 1 << 30 || chunk_tokens > 1 << 30)
    return fail(SKV_EINVAL, "%s: max_ctx %d or chunk_tokens %d past 2^30", who, max_ctx, chunk_tokens);
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
