// Causal attention of packed prompts over their own keys: softmax(q K^T scale) V per sequence, query i of a sequence seeing
// its keys 0..i, grouped heads. Sequences lie one behind the other in the rows, without padding.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "skv_common.h"
#include "skv_device.h"

using namespace skv;

namespace {

struct PromptAttn {
  const char *q, *k, *v;
  char* o;
  int64_t qsn, qsh, ksn, ksh, vsn, vsh, osn, osh;  // bytes
  const int32_t* cu;
  float scale_log2;
  int32_t n, seqs, heads, group, row_bytes;
};

template <int DT>
using elt_t = typename std::conditional<DT == SKV_F32, float,
                                        typename std::conditional<DT == SKV_F16, _Float16, __bf16>::type>::type;

// Sequence s as [begin, end), within the rows whatever cu holds.
__device__ __forceinline__ void seq_range(const PromptAttn& p, int s, int& begin, int& end) {
  begin = min(max(p.cu[s], 0), p.n);
  end = min(max(p.cu[s + 1], begin), p.n);
}

// One query by one wave, its head's keys one after the other in fp32: lane l holds dims l and l + 64.
template <int DT, int D>
__device__ __forceinline__ void query_slow(const PromptAttn& p, int row, int begin, int h) {
  constexpr int N = D > 64 ? D / 64 : 1;
  const int lane = threadIdx.x & 63;
  const bool on = lane < p.row_bytes / (int)sizeof(elt_t<DT>);
  const int kvh = h / p.group;
  const elt_t<DT>* q = reinterpret_cast<const elt_t<DT>*>(p.q + (int64_t)row * p.qsn + (int64_t)h * p.qsh);
  float qf[N], acc[N], m = kNegInf, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    qf[i] = on ? (float)q[lane + 64 * i] : 0.f;
    acc[i] = 0.f;
  }
  for (int t = begin; t <= row; ++t) {
    const elt_t<DT>* k = reinterpret_cast<const elt_t<DT>*>(p.k + (int64_t)t * p.ksn + (int64_t)kvh * p.ksh);
    const elt_t<DT>* v = reinterpret_cast<const elt_t<DT>*>(p.v + (int64_t)t * p.vsn + (int64_t)kvh * p.vsh);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (on) s = fmaf(qf[i], (float)k[lane + 64 * i], s);
    s = group_sum<64>(s) * p.scale_log2;
    const float mx = max_score(m, s);
    const float ref = mx == kNegInf ? 0.f : mx;
    const float a = __builtin_amdgcn_exp2f(m - ref), w = __builtin_amdgcn_exp2f(s - ref);
    l = fmaf(l, a, w);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (on) acc[i] = fmaf(w, (float)v[lane + 64 * i], acc[i] * a);
    m = mx;
  }
  if (!on) return;
  elt_t<DT>* o = reinterpret_cast<elt_t<DT>*>(p.o + (int64_t)row * p.osn + (int64_t)h * p.osh);
#pragma unroll
  for (int i = 0; i < N; ++i) o[lane + 64 * i] = (elt_t<DT>)(l > 0.f || l != l ? acc[i] / l : 0.f);
}

// ---------------------------------------------------------------------------
// 16-bit rows on the matrix cores: one workgroup owns 32 * QW consecutive queries of one head, 32 per wave, and walks the keys
// up to its last query in tiles of KT staged in LDS (double-buffered, one barrier per tile). KW = 2: two waves share 32 queries,
// each with half of every tile's keys, and join at the end.
//   S^T = K Q^T in 32 x 32 products: a lane holds 16 keys' scores of one query per product, whose softmax weights are, in
//   place, the operand of O^T = V^T P^T: contraction element (half f, j) of a 16-key step stands for key 4 f + j, 8 + 4 f + j - 4
//   in both operands. V^T comes from the row-major LDS rows through the transpose load.
// The running maximum and sum and the accumulators are fp32; the weights are rounded to the rows' type for their product
// (by half a step each, 2^-8 or 2^-11, as the result is), their sum takes them unrounded.
// What bounds it: the matrix cores (55 % of the clocks) and the vector operations of the softmax (47 %), which two waves per SIMD
// overlap in part. bf16: 16384 tokens, 32 / 8 heads x 128, 2.07-2.2 ms (1000-1060 TFLOP/s, the library's 8192^3 product 1402);
// 20 heads x 64 0.75-0.8 ms (870-910); 8 x 448 tokens 14.7 us.
// ---------------------------------------------------------------------------
constexpr float kLazyMaxLog2 = 8.f;  // the accumulators are rescaled when a maximum grows by more than this

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16* lds_v4;
__device__ __forceinline__ uint2 lds_tr16(const char* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4) const_cast<char*>(p)));
}

__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, xor_lane<1>(x));
  x = fmaxf(x, xor_lane<2>(x));
  x = fmaxf(x, xor_lane<4>(x));
  x = fmaxf(x, xor_lane<8>(x));
  x = fmaxf(x, xor_lane<16>(x));
  return fmaxf(x, xor_lane<32>(x));
}

// The (sequence, query tile) of a work index. Sequence s has its places from start(s) = floor(cu[s] / M) + s on, which leaves
// each its ceil(length / M) tiles and takes n / M + seqs in all, so that the 64 sequences around an index are found by a search
// over cu instead of a sum over all that come before (128 queries a workgroup, bf16 20 heads x 64, 1024 prompts of 30 tokens:
// 237 us with the sum, 157 with the search; 4096 of one token 1277 and 412). Within the 64, tiles with more keys come first, so that the workgroups that take longest do not start last. False for a
// place without a tile.
template <int M>
__device__ __forceinline__ bool find_tile(const PromptAttn& p, int index, int& begin, int& len, int& tile) {
  const int lane = threadIdx.x & 63;
  int s0 = 0;
  for (int span = (p.seqs + 63) / 64; span > 1;) {  // groups of 64 that may hold the index, from s0 on
    const int step = (span + 63) / 64;
    bool at_or_before = false;
    if (lane * step < span) {
      const int s = s0 + 64 * lane * step;
      at_or_before = min(max(p.cu[s], 0), p.n) / M + s <= index;
    }
    const int last = __builtin_popcountll(__builtin_amdgcn_ballot_w64(at_or_before)) - 1;
    if (last < 0) return false;
    s0 += 64 * last * step;
    span = min(step, span - last * step);
  }
  int b = 0, e = 0;
  if (s0 + lane < p.seqs) seq_range(p, s0 + lane, b, e);
  index -= __builtin_amdgcn_readfirstlane(b) / M + s0;
  const int n = (e - b + M - 1) / M;
  // Tiles with a number of t or more, over the 64 sequences (fewer than 2^24 in a launch, which floats count).
  auto from = [&](int t) __attribute__((always_inline)) {
    return __builtin_amdgcn_readfirstlane((int)group_sum<64>((float)max(n - t, 0)));
  };
  if (index < 0 || index >= from(0)) return false;
  int lo = 0, hi = __builtin_amdgcn_readfirstlane((int)wave_max((float)n)), ahead = 0;
  while (hi - lo > 1) {  // from(lo) > index >= from(hi) = ahead
    const int mid = (lo + hi) / 2, f = from(mid);
    if (f > index)
      lo = mid;
    else
      hi = mid, ahead = f;
  }
  // The (index - ahead)-th sequence of those that have a tile number lo.
  const uint64_t have = __builtin_amdgcn_ballot_w64(n > lo);
  const int before = __builtin_popcountll(have & ((1ull << lane) - 1));
  const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(n > lo && before == index - ahead));
  begin = __builtin_amdgcn_readlane(b, l);
  len = __builtin_amdgcn_readlane(e, l) - begin;
  tile = lo;
  return true;
}

template <int DT, int D, int QW, int KW, int KT>
__global__ __launch_bounds__(64 * QW * KW, 2) void prompt_kernel(PromptAttn p) {
  constexpr int M = 32 * QW;
  constexpr int KB = KT / 32 / KW;          // 32-key blocks of a tile that a wave takes
  constexpr int VPR = D / 8;                // 16-byte vectors per row
  constexpr int RPP = 64 * QW * KW / VPR;   // rows a pass of the workgroup loads
  constexpr int PASSES = RPP > KT ? 1 : KT / RPP;
  // LDS rows are padded so that neither the 16 rows of a K load (16 bytes each) nor the 4 rows of a V^T load (64 bytes each)
  // meet in a bank.
  constexpr int KROW = D * 2 + 16, VROW = D * 2 + (D == 32 ? 0 : 64);
  constexpr int KS = D / 16;                // contraction steps of a score product
  constexpr int DB = D / 32;                // 32-dim blocks of the result
  constexpr int KBUF = KT * KROW, VBUF = KT * VROW;
  constexpr int JOIN = KW == 1 ? 0 : QW * 64 * (16 * DB + 2) * 4;  // the second key half's state
  constexpr int LDS = 2 * (KBUF + VBUF) > JOIN ? 2 * (KBUF + VBUF) : JOIN;
  __shared__ __attribute__((aligned(16))) char s_mem[LDS];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int qw = wave % QW, kw = wave / QW;
  const int n = lane & 31, f = lane >> 5;
  // Heads vary fastest, the heads of a die (workgroup index modulo 8) being neighbours that share K/V.
  const int H = p.heads;
  int h = (int)(blockIdx.x % (uint32_t)H);
  if ((H & 7) == 0) h = (h & 7) * (H >> 3) + (h >> 3);
  int begin, len, tile;
  if (!find_tile<M>(p, (int)(blockIdx.x / (uint32_t)H), begin, len, tile)) return;
  const int kvh = h / p.group;
  const int first = tile * M + qw * 32;     // the wave's first query in its sequence
  const int keys = min(len, tile * M + M);  // keys of the workgroup
  const int wave_keys = first < len ? min(len, first + 32) : 0;

  // The maximum is taken over unscaled scores, so the scale has to be positive: a negative one goes into q's signs, and 0
  // becomes the least normal number, whose scores' weights are 1 as well.
  const float c = fmaxf(fabsf(p.scale_log2), 1.17549435e-38f);
  const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
  // Q^T operand: lane (query n, half f) holds dims 16 ks + 8 f .. + 7.
  uint4 qf[KS];
  {
    const char* row = p.q + (int64_t)(begin + min(first + n, len - 1)) * p.qsn + (int64_t)h * p.qsh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint4 x = 32 * ks + 16 * f < p.row_bytes ? *reinterpret_cast<const uint4*>(row + 32 * ks + 16 * f)
                                                     : make_uint4(0u, 0u, 0u, 0u);
      qf[ks] = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
    }
  }

  const char* kbase = p.k + (int64_t)begin * p.ksn + (int64_t)kvh * p.ksh;
  const char* vbase = p.v + (int64_t)begin * p.vsn + (int64_t)kvh * p.vsh;
  const int ld_row = threadIdx.x / VPR, ld_col = (threadIdx.x % VPR) * 16;
  const bool loads = ld_row < KT;  // with D = 32 a pass may hold more rows than a tile
  uint4 kr[PASSES], vr[PASSES];
  // Byte offsets of the lane's vectors within a tile; head_dim 16 leaves the upper half of 32 dims zeros.
  uint32_t koff[PASSES], voff[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const bool on = loads && ld_col < p.row_bytes;
    koff[i] = on ? (uint32_t)((ld_row + i * RPP) * (int)p.ksn + ld_col) : kBufOutOfRange;
    voff[i] = on ? (uint32_t)((ld_row + i * RPP) * (int)p.vsn + ld_col) : kBufOutOfRange;
  }
  // Loads of the tile at key t0; rows past the sequence read zeros (rows of stride 0 are all the first row).
  auto issue = [&](const char* base, int64_t stride, int t0, const uint32_t (&off)[PASSES], uint4 (&r)[PASSES])
                   __attribute__((always_inline)) {
    const int left = len - t0;  // may be 0 or less: nothing is read
    const int64_t bytes = left > 0 ? (int64_t)(min(left, KT) - 1) * stride + p.row_bytes : 0;
    const __amdgpu_buffer_rsrc_t res =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + (int64_t)t0 * stride), (short)0, (int)bytes, kBufWord3);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) r[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(res, off[i], 0, 0));
  };
  auto issue_k = [&](int t0) __attribute__((always_inline)) { issue(kbase, p.ksn, t0, koff, kr); };
  auto issue_v = [&](int t0) __attribute__((always_inline)) { issue(vbase, p.vsn, t0, voff, vr); };
  auto stage_k = [&](int buf) __attribute__((always_inline)) {
    if (!loads) return;
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
      *reinterpret_cast<uint4*>(s_mem + buf * KBUF + (ld_row + i * RPP) * KROW + ld_col) = kr[i];
  };
  auto stage_v = [&](int buf) __attribute__((always_inline)) {
    if (!loads) return;
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
      *reinterpret_cast<uint4*>(s_mem + 2 * KBUF + buf * VBUF + (ld_row + i * RPP) * VROW + ld_col) = vr[i];
  };
  const char* lk0 = s_mem + (32 * KB * kw + n) * KROW + 16 * f;
  // V^T: lane 4 kk + q of a 16-lane group addresses key kk, dims 4 q .. + 3 of the group's 16 dims.
  const char* lv0 = s_mem + 2 * KBUF + (32 * KB * kw + 4 * f + ((lane & 15) >> 2)) * VROW + 8 * (lane & 3) +
                    32 * ((lane >> 4) & 1);
  auto scores = [&](int buf, f32x16 (&s)[KB]) __attribute__((always_inline)) {
    const char* lk = lk0 + buf * KBUF;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        s[kb] = mfma_32x32x16<DT>(*reinterpret_cast<const uint4*>(lk + 32 * kb * KROW + 32 * ks), qf[ks], s[kb]);
    }
  };

  float m = kNegInf, ref = 0.f, l = 0.f;
  f32x16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;

  // Tile t's scores are computed during tile t - 1, beside its softmax: the products of the one and the exponentials of the other
  // need not wait for each other. So K is staged a tile ahead of V.
  issue_k(0);
  issue_v(0);
  stage_k(0);
  issue_k(KT);
  __syncthreads();
  f32x16 s[KB], s_next[KB];
  scores(0, s);
  stage_v(0);
  stage_k(1);
  issue_k(2 * KT);
  issue_v(KT);
  lds_barrier();
  for (int t0 = 0, buf = 0; t0 < keys; t0 += KT, buf ^= 1) {
    // Tile t0 + 128's K goes where tile t0's was, tile t0 + 64's V where tile t0 - 64's was: the last barrier is behind their reads.
    if (t0 > 0) {
      stage_v(buf);
      stage_k(buf ^ 1);
      issue_k(t0 + 2 * KT);
      issue_v(t0 + KT);
      lds_barrier();
    }
    const int k0 = t0 + 32 * KB * kw;  // the wave's first key of the tile
    if (k0 < wave_keys) {              // wave-uniform
      if (k0 + 32 * KB > first + 1) {  // wave-uniform: a key that some query does not see
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[kb][i] = k0 + 32 * kb + 8 * (i >> 2) + 4 * f + (i & 3) <= first + n ? s[kb][i] : kNegInf;
      }
      float mx = kNegInf;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = max_score(mx, s[kb][i]);
      if (__builtin_amdgcn_ballot_w64(mx * c > m + kLazyMaxLog2) != 0) {  // wave-uniform
        const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        mx = max_score(__uint_as_float(r32[0]), __uint_as_float(r32[1]));
        const float mn = max_score(m, mx * c);
        ref = mn == kNegInf ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] *= alpha;
        l *= alpha;
        m = mn;
      }
      scores(buf ^ 1, s_next);
      uint4 pt[2 * KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        float w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], c, -ref));
#pragma unroll
        for (int i = 0; i < 16; i += 4) l += (w[i] + w[i + 1]) + (w[i + 2] + w[i + 3]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          pt[2 * kb + i] = make_uint4(pack2<DT>(w[8 * i], w[8 * i + 1]), pack2<DT>(w[8 * i + 2], w[8 * i + 3]),
                                      pack2<DT>(w[8 * i + 4], w[8 * i + 5]), pack2<DT>(w[8 * i + 6], w[8 * i + 7]));
      }
      const char* lv = lv0 + buf * VBUF;
#pragma unroll
      for (int ks = 0; ks < 2 * KB; ++ks) {
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const uint2 a = lds_tr16(lv + 16 * ks * VROW + 64 * db), b = lds_tr16(lv + (16 * ks + 8) * VROW + 64 * db);
          acc[db] = mfma_32x32x16<DT>(make_uint4(a.x, a.y, b.x, b.y), pt[ks], acc[db]);
        }
      }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) s[kb] = s_next[kb];
    }
  }
  lds_barrier();

  if constexpr (KW == 2) {
    // The second key half hands its state to the first, a float of each lane after the other; the tiles are done with.
    float* join = reinterpret_cast<float*>(s_mem) + qw * 64 * (16 * DB + 2) + lane;
    if (kw == 1) {
      join[0] = m;
      join[64] = l;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) join[64 * (2 + 16 * db + i)] = acc[db][i];
    }
    lds_barrier();
    if (kw == 1) return;
    const float m1 = join[0];
    const float mm = max_score(m, m1);
    const float base = mm == kNegInf ? 0.f : mm;
    const float f0 = __builtin_amdgcn_exp2f(m - base), f1 = __builtin_amdgcn_exp2f(m1 - base);
    l = l * f0 + join[64] * f1;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[db][i] = acc[db][i] * f0 + join[64 * (2 + 16 * db + i)] * f1;
  }
  if (first >= len) return;  // wave-uniform
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
  const float sum = __uint_as_float(r32[0]) + __uint_as_float(r32[1]);
  // A key that a query does not see has weight 0 in the tile's product, and 0 times an infinite or NaN value is NaN: a wave with
  // such a result, and such a value among the keys of its last tile, computes its queries again one at a time.
  float all = 0.f;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) all += fabsf(acc[db][i]);
  if (__builtin_amdgcn_ballot_w64(!(all < __builtin_huge_valf())) != 0) {
    bool bad = false;
    for (int t = first; t < min(len, (wave_keys + KT - 1) / KT * KT); ++t) {
      const elt_t<DT>* v = reinterpret_cast<const elt_t<DT>*>(vbase + (int64_t)t * p.vsn);
      for (int d = lane; 2 * d < p.row_bytes; d += 64) bad |= !(fabsf((float)v[d]) < __builtin_huge_valf());
    }
    if (__builtin_amdgcn_ballot_w64(bad) != 0) {
      for (int qi = first; qi < min(len, first + 32); ++qi) query_slow<DT, D>(p, begin + qi, begin, h);
      return;
    }
  }
  if (first + n >= len) return;
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  char* o = p.o + (int64_t)(begin + first + n) * p.osn + (int64_t)h * p.osh;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; i += 4)  // dims 32 db + 8 (i / 4) + 4 f .. + 3
      if (64 * db + 4 * i < p.row_bytes)
        *reinterpret_cast<uint2*>(o + 64 * db + 4 * i + 8 * f) =
            make_uint2(pack2<DT>(acc[db][i] * inv, acc[db][i + 1] * inv), pack2<DT>(acc[db][i + 2] * inv, acc[db][i + 3] * inv));
}

// ---------------------------------------------------------------------------
// fp32 rows on the matrix cores: one workgroup per (head, 16 queries), its waves take the keys in turns of 16 and join at the
// end. Everything stays in registers: the contraction index an element stands for only has to agree between the operands, so
// lane (g, r) loads whole pieces of rows (key r, dims g D / 4 .. + D / 4 - 1; keys 4 g + e, dims r D / 16 .. + D / 16 - 1), and the
// scores come out as the operand that the second product takes. What bounds it: the 16 x 16 x 4 products, 32 clocks each (1500
// tokens, 12 heads x 64 52 us, 67 of the library's 154 TFLOP/s; one wave per query took 860).
// ---------------------------------------------------------------------------
constexpr int kWaves32 = 4;

template <int D>
__global__ __launch_bounds__(64 * kWaves32) void prompt_f32_kernel(PromptAttn p) {
  constexpr int KD = D / 4, VD = D / 16;  // floats of a lane's piece of a K row and of a V row
  __shared__ float s_ml[kWaves32][2][16];
  __shared__ float s_acc[kWaves32][16][D + 4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int g = lane >> 4, r = lane & 15;
  const int h = (int)(blockIdx.x % (uint32_t)p.heads);
  int begin, len, tile;
  if (!find_tile<16>(p, (int)(blockIdx.x / (uint32_t)p.heads), begin, len, tile)) return;
  const int kvh = h / p.group;
  const int first = tile * 16, keys = min(len, first + 16);
  const char* kbase = p.k + (int64_t)begin * p.ksn + (int64_t)kvh * p.ksh + g * KD * 4;
  const char* vbase = p.v + (int64_t)begin * p.vsn + (int64_t)kvh * p.vsh;
  float q[KD], kr[KD], vr[4][VD];
  load_floats<KD>(reinterpret_cast<const float*>(p.q + (int64_t)(begin + min(first + r, len - 1)) * p.qsn + (int64_t)h * p.qsh) +
                      g * KD, q);
  // Rows past the sequence are its last row, whose weight is then 0.
  auto load_k = [&](int t0) __attribute__((always_inline)) {
    load_floats<KD>(reinterpret_cast<const float*>(kbase + (int64_t)min(t0 + r, len - 1) * p.ksn), kr);
  };
  auto load_v = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float* v = reinterpret_cast<const float*>(vbase + (int64_t)min(t0 + 4 * g + e, len - 1) * p.vsn) + r * VD;
      if constexpr (VD >= 4) {
        load_floats<VD>(v, vr[e]);
      } else {
#pragma unroll
        for (int i = 0; i < VD; ++i) vr[e][i] = v[i];
      }
    }
  };
  f32x4 acc[VD];
#pragma unroll
  for (int i = 0; i < VD; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = kNegInf, l = 0.f;
  int t0 = 16 * wave;
  if (t0 < keys) {
    load_k(t0);
    load_v(t0);
  }
  for (; t0 < keys; t0 += 16 * kWaves32) {
    f32x4 s0 = f32x4{0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
    for (int e = 0; e < KD; e += 2) {
      s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[e], q[e], s0, 0, 0, 0);
      s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[e + 1], q[e + 1], s1, 0, 0, 0);
    }
    load_k(t0 + 16 * kWaves32);
    float s[4], mx = m;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[e] = t0 + 4 * g + e <= first + r ? (s0[e] + s1[e]) * p.scale_log2 : kNegInf;
      mx = max_score(mx, s[e]);
    }
    mx = max_score(mx, xor_lane<16>(mx));
    mx = max_score(mx, xor_lane<32>(mx));
    const float ref = mx == kNegInf ? 0.f : mx;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    l *= alpha;
#pragma unroll
    for (int i = 0; i < VD; ++i) acc[i] *= alpha;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[e] = __builtin_amdgcn_exp2f(s[e] - ref);
      l += s[e];
    }
    m = mx;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < VD; ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[e][i], s[e], acc[i], 0, 0, 0);
    load_v(t0 + 16 * kWaves32);
  }
  l += xor_lane<16>(l);
  l += xor_lane<32>(l);
  // Lane (g, r) holds query r, dims (4 g + e) D / 16 + i in acc[i][e].
  if (g == 0) {
    s_ml[wave][0][r] = m;
    s_ml[wave][1][r] = l;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int i = 0; i < VD; ++i) s_acc[wave][r][(4 * g + e) * VD + i] = acc[i][e];
  __syncthreads();
  // As in prompt_kernel: a result that is not finite beside such a value among keys that some query does not see.
  bool off = false;
  for (int i = threadIdx.x; i < 16 * D; i += 64 * kWaves32) {
    const int qi = i / D, d = i % D;
    if (first + qi >= len) continue;
    float mm = s_ml[0][0][qi];
#pragma unroll
    for (int w = 1; w < kWaves32; ++w) mm = max_score(mm, s_ml[w][0][qi]);
    const float ref = mm == kNegInf ? 0.f : mm;
    float lt = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves32; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_ml[w][0][qi] - ref);
      lt = fmaf(s_ml[w][1][qi], f, lt);
      o = fmaf(s_acc[w][qi][d], f, o);
    }
    o = lt > 0.f || lt != lt ? o / lt : 0.f;
    off |= !(fabsf(o) < __builtin_huge_valf());
    reinterpret_cast<float*>(p.o + (int64_t)(begin + first + qi) * p.osn + (int64_t)h * p.osh)[d] = o;
  }
  if (!__syncthreads_or(off)) return;
  bool bad = false;
  for (int t = first; t < keys; ++t) {
    const float* v = reinterpret_cast<const float*>(vbase + (int64_t)t * p.vsn);
    for (int d = lane; d < D; d += 64) bad |= !(fabsf(v[d]) < __builtin_huge_valf());
  }
  if (__builtin_amdgcn_ballot_w64(bad) == 0) return;
  for (int qi = first + wave; qi < keys; qi += kWaves32) query_slow<SKV_F32, D>(p, begin + qi, begin, h);
}

template <int DT, int D, int QW, int KW, int KT>
void launch_tiles(const PromptAttn& p, hipStream_t stream) {
  const int tiles = p.n / (32 * QW) + p.seqs;  // at least the sum of ceil(length / M)
  hipLaunchKernelGGL((prompt_kernel<DT, D, QW, KW, KT>), dim3((uint32_t)tiles * (uint32_t)p.heads), dim3(64 * QW * KW), 0, stream, p);
}
// Three forms, by what the host knows: rows, sequences and heads. bf16, us of the form with 128 queries / the one named:
//   Short sequences, up to 128 rows on average: 64 queries a workgroup and 32 keys a tile, whose small LDS lets more
//     workgroups run at once, each with less padding. 20 heads x 64: 1024 x 30 tokens 157 / 98, 256 x 60 43 / 35, 256 x 120
//     90 / 90, 64 x 200 40 / 46; 32 / 8 heads x 128: 256 x 60 139 / 105, 2048 and 200 x 10 105 / 74, 2048..1 (16) 80 / 82.
//   Few workgroups of 128 (up to 1.5 a compute unit; two fit on one) are as slow as the one with the most keys: two waves share
//     32 queries' keys. Heads x 128: 32 x 512 tokens (128 workgroups) 15.9 / 12.4, 8 x 4096 (256) 81 / 61, 6 x 6428 (306) 126 / 95,
//     20 x 3 prompts of 700 (340) 22 / 24, 12 x 4096 (384) 88 / 76, 28 x 2048 (448) 51 / 53, 32 x 2048 (512) 53 / 55; x 64: 20 x
//     2048 (320) 32 / 24, 20 x 100 6.0 / 5.1 (the short form 5.6), 20 x 8 of 30 4.3 / 4.3 (3.8): the short form up to 64 on average.
template <int DT, int D>
void launch_prompt(const PromptAttn& p, hipStream_t stream) {
  const bool few = 2 * cdiv(p.n, 128) * p.heads <= 3 * compute_units();
  if (p.n <= (few ? 64 : 128) * (int64_t)p.seqs)
    launch_tiles<DT, D, 2, 1, 32>(p, stream);
  else if (few)
    launch_tiles<DT, D, 2, 2, 64>(p, stream);
  else
    launch_tiles<DT, D, 4, 1, 64>(p, stream);
}
template <int D>
void launch_prompt_f32(const PromptAttn& p, hipStream_t stream) {
  const int tiles = p.n / 16 + p.seqs;
  hipLaunchKernelGGL((prompt_f32_kernel<D>), dim3((uint32_t)tiles * (uint32_t)p.heads), dim3(64 * kWaves32), 0, stream, p);
}
template <int DT>
void launch_prompt_d(int d, const PromptAttn& p, hipStream_t stream) {
  if constexpr (DT != SKV_F32) {
    if (d == 128)
      launch_prompt<DT, 128>(p, stream);
    else if (d == 64)
      launch_prompt<DT, 64>(p, stream);
    else
      launch_prompt<DT, 32>(p, stream);
  } else {
    if (d == 128)
      launch_prompt_f32<128>(p, stream);
    else if (d == 64)
      launch_prompt_f32<64>(p, stream);
    else if (d == 32)
      launch_prompt_f32<32>(p, stream);
    else
      launch_prompt_f32<16>(p, stream);
  }
}

}  // namespace

extern "C" int skv_prompt_attention(const void* q, int64_t q_stride_n, int64_t q_stride_h, const void* k,
                                    int64_t k_stride_n, int64_t k_stride_h, const void* v, int64_t v_stride_n,
                                    int64_t v_stride_h, const int32_t* cu_seqlens, void* out, int64_t o_stride_n,
                                    int64_t o_stride_h, int32_t n_tokens, int32_t num_seqs, int32_t num_heads,
                                    int32_t num_kv_heads, int32_t head_dim, float scale, int32_t dtype, void* stream) {
  const char* who = "skv_prompt_attention";
  const int eb = elt_bytes(dtype);
  if (eb == 0) return fail(SKV_EDTYPE, "%s: unknown dtype %d", who, dtype);
  if (head_dim != 16 && head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(SKV_EINVAL, "%s: head_dim %d not in {16,32,64,128}", who, head_dim);
  if (n_tokens < 0 || num_seqs < 0 || num_heads <= 0 || num_heads > 65535 || num_kv_heads <= 0 || num_heads % num_kv_heads)
    return fail(SKV_EINVAL, "%s: bad sizes n=%d seqs=%d heads=%d kv_heads=%d", who, n_tokens, num_seqs, num_heads, num_kv_heads);
  if (n_tokens == 0 || num_seqs == 0) return SKV_OK;
  if (!q || !k || !v || !out || !cu_seqlens) return fail(SKV_EINVAL, "%s: null pointer argument", who);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(SKV_EALIGN, "%s: q, k, v and out must be 16-byte aligned", who);
  const int epl = 16 / eb;
  if ((q_stride_n | q_stride_h | k_stride_n | k_stride_h | v_stride_n | v_stride_h | o_stride_n | o_stride_h) % epl)
    return fail(SKV_EALIGN, "%s: strides must be multiples of %d elements", who, epl);
  // A tile's rows are read through 32-bit offsets, which no row may leave: up to 16 MiB from one to the next.
  for (int64_t st : {k_stride_n, v_stride_n})
    if (st < 0 || st * eb >= (int64_t)1 << 24)
      return fail(SKV_EINVAL, "%s: row stride %lld of k or v is negative or past 16 MiB", who, (long long)st);
  const int64_t tiles = n_tokens / (dtype == SKV_F32 ? 16 : 64) + (int64_t)num_seqs;  // the most any form launches per head
  if (tiles * num_heads >= (int64_t)1 << 24)
    return fail(SKV_EINVAL, "%s: launch too large (%d rows, %d sequences, %d heads)", who, n_tokens, num_seqs, num_heads);
  const PromptAttn p{(const char*)q, (const char*)k, (const char*)v, (char*)out,
                     q_stride_n * eb, q_stride_h * eb, k_stride_n * eb, k_stride_h * eb,
                     v_stride_n * eb, v_stride_h * eb, o_stride_n * eb, o_stride_h * eb,
                     cu_seqlens, scale * kLog2e, n_tokens, num_seqs, num_heads, num_heads / num_kv_heads, head_dim * eb};
  switch (dtype) {
    case SKV_F32: launch_prompt_d<SKV_F32>(head_dim, p, (hipStream_t)stream); break;
    case SKV_F16: launch_prompt_d<SKV_F16>(head_dim, p, (hipStream_t)stream); break;
    default: launch_prompt_d<SKV_BF16>(head_dim, p, (hipStream_t)stream); break;
  }
  return check_launch(who);
}
