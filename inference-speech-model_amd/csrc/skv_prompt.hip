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
  int32_t n, seqs, heads, group;
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
  const bool on = lane < D;
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

// One wave per (query, head), any sequence: the simple form.
template <int DT, int D>
__global__ __launch_bounds__(256) void prompt_simple_kernel(PromptAttn p) {
  const uint32_t item = blockIdx.x * 4u + (threadIdx.x >> 6);
  const int row = (int)(item / (uint32_t)p.heads), h = (int)(item % (uint32_t)p.heads);
  if (row >= p.n) return;
  for (int s = 0; s < p.seqs; ++s) {
    int begin, end;
    seq_range(p, s, begin, end);
    if (row >= begin && row < end) {
      query_slow<DT, D>(p, row, begin, h);
      return;
    }
  }
}

// ---------------------------------------------------------------------------
// 16-bit rows on the matrix cores: one workgroup of 4 waves owns 128 * QB consecutive queries of one head, 32 * QB per wave,
// and walks the keys up to its last query in tiles of 64 staged in LDS (double-buffered, one barrier per tile).
//   S^T = K Q^T in 32 x 32 products: a lane holds 16 keys' scores of one query per product, whose softmax weights are, in
//   place, the operand of O^T = V^T P^T: contraction element (half f, j) of a 16-key step stands for key 4 f + j, 8 + 4 f + j - 4
//   in both operands. V^T comes from the row-major LDS rows through the transpose load.
// The running maximum and sum and the accumulators are fp32; the weights are rounded to the rows' type for their product
// (relative 2^-9 or 2^-12 each, as the result is), their sum takes them unrounded.
// ---------------------------------------------------------------------------
constexpr int kKeys = 64;            // keys of a staged tile
constexpr float kLazyMaxLog2 = 8.f;  // the accumulators are rescaled when a maximum grows by more than this

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16* lds_v4;
__device__ __forceinline__ uint2 lds_tr16(const char* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4) const_cast<char*>(p)));
}

// The (sequence, query tile) of a work index: sequences have ceil(length / M) tiles each. False past the last one.
template <int M>
__device__ __forceinline__ bool find_tile(const PromptAttn& p, int index, int& begin, int& len, int& tile) {
  const int lane = threadIdx.x & 63;
  int run = 0;
  for (int s0 = 0; s0 < p.seqs; s0 += 64) {
    int b = 0, e = 0;
    if (s0 + lane < p.seqs) seq_range(p, s0 + lane, b, e);
    const int n = (e - b + M - 1) / M;
    int sum = n;  // inclusive prefix sum over the lanes
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(sum, o);
      if (lane >= o) sum += up;
    }
    const uint64_t behind = __builtin_amdgcn_ballot_w64(run + sum > index);
    if (behind) {
      const int l = __builtin_ctzll(behind);
      begin = __builtin_amdgcn_readlane(b, l);
      len = __builtin_amdgcn_readlane(e, l) - begin;
      tile = index - (run + __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(n, l));
      return true;
    }
    run += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

template <int DT, int D, int QB>
__global__ __launch_bounds__(256, 2) void prompt_kernel(PromptAttn p, int tiles) {
  constexpr int M = 128 * QB;
  constexpr int VPR = D / 8;           // 16-byte vectors per row
  constexpr int RPP = 256 / VPR;       // rows a pass of the workgroup loads
  constexpr int PASSES = kKeys / RPP;
  constexpr int KROW = D * 2 + 16;     // LDS rows: 16 bytes of padding spread the rows over the banks
  constexpr int KS = D / 16;           // contraction steps of a score product
  constexpr int DB = D / 32;           // 32-dim blocks of the result
  constexpr int BUF = 2 * kKeys * KROW;
  __shared__ __attribute__((aligned(16))) char s_kv[2][BUF];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int n = lane & 31, f = lane >> 5;
  // Heads vary fastest, the heads of a die (workgroup index modulo 8) being neighbours that share K/V; tiles go from the
  // last, which has the most keys, to the first.
  const int H = p.heads;
  int h = (int)(blockIdx.x % (uint32_t)H);
  if ((H & 7) == 0) h = (h & 7) * (H >> 3) + (h >> 3);
  int begin, len, tile;
  if (!find_tile<M>(p, tiles - 1 - (int)(blockIdx.x / (uint32_t)H), begin, len, tile)) return;
  const int kvh = h / p.group;
  const int q0 = tile * M + wave * (32 * QB);  // the wave's first query in its sequence
  const int keys = min(len, tile * M + M);     // keys of the workgroup
  const int wave_keys = q0 < len ? min(len, q0 + 32 * QB) : 0;

  // The maximum is taken over unscaled scores, so the scale has to be positive: a negative one goes into q's signs, and 0
  // becomes the least normal number, whose scores' weights are 1 as well.
  const float c = fmaxf(fabsf(p.scale_log2), 1.17549435e-38f);
  const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
  // Q^T operand: lane (query n, half f) holds dims 16 ks + 8 f .. + 7.
  uint4 qf[QB][KS];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int qi = min(q0 + 32 * qb + n, len - 1);
    const char* row = p.q + (int64_t)(begin + qi) * p.qsn + (int64_t)h * p.qsh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint4 x = *reinterpret_cast<const uint4*>(row + 32 * ks + 16 * f);
      qf[qb][ks] = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
    }
  }

  const char* kbase = p.k + (int64_t)begin * p.ksn + (int64_t)kvh * p.ksh;
  const char* vbase = p.v + (int64_t)begin * p.vsn + (int64_t)kvh * p.vsh;
  const int ld_row = threadIdx.x / VPR, ld_col = (threadIdx.x % VPR) * 16;
  uint4 kr[PASSES], vr[PASSES];
  // Loads of the tile at key t0; rows past the sequence read zeros.
  auto issue = [&](int t0) __attribute__((always_inline)) {
    const int left = len - t0;  // may be 0 or less: nothing is read
    const int64_t kb = left > 0 ? (int64_t)(min(left, kKeys) - 1) * p.ksn + D * 2 : 0;
    const int64_t vb = left > 0 ? (int64_t)(min(left, kKeys) - 1) * p.vsn + D * 2 : 0;
    const __amdgpu_buffer_rsrc_t kres = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(kbase + (int64_t)t0 * p.ksn), (short)0, (int)kb, kBufWord3);
    const __amdgpu_buffer_rsrc_t vres = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(vbase + (int64_t)t0 * p.vsn), (short)0, (int)vb, kBufWord3);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int row = ld_row + i * RPP;
      kr[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(kres, row * (int)p.ksn + ld_col, 0, 0));
      vr[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(vres, row * (int)p.vsn + ld_col, 0, 0));
    }
  };
  auto stage = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      char* t = &s_kv[buf][0] + (ld_row + i * RPP) * KROW + ld_col;
      *reinterpret_cast<uint4*>(t) = kr[i];
      *reinterpret_cast<uint4*>(t + kKeys * KROW) = vr[i];
    }
  };

  float m[QB], ref[QB], l[QB];
  f32x16 acc[QB][DB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    m[qb] = kNegInf, ref[qb] = 0.f, l[qb] = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[qb][db][i] = 0.f;
  }

  issue(0);
  stage(0);
  issue(kKeys);
  __syncthreads();
  for (int t0 = 0, buf = 0; t0 < keys; t0 += kKeys, buf ^= 1) {
    if (t0 + kKeys < keys) stage(buf ^ 1);
    issue(t0 + 2 * kKeys);
    if (t0 < wave_keys) {  // wave-uniform
      const char* lk = &s_kv[buf][0] + n * KROW + 16 * f;
      // V^T: lane 4 kk + q of a 16-lane group addresses key kk, dims 4 q .. + 3 of the group's 16 dims.
      const char* lv = &s_kv[buf][0] + kKeys * KROW + (4 * f + ((lane & 15) >> 2)) * KROW + 8 * (lane & 3) + 32 * ((lane >> 4) & 1);
      f32x16 s[QB][2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[qb][kb][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint4 a = *reinterpret_cast<const uint4*>(lk + 32 * kb * KROW + 32 * ks);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) s[qb][kb] = mfma_32x32x16<DT>(a, qf[qb][ks], s[qb][kb]);
        }
      }
      uint4 pt[QB][4];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const int first = q0 + 32 * qb;  // every query of the block sees the keys up to it
        if (t0 + kKeys > first + 1) {    // wave-uniform
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              s[qb][kb][i] = t0 + 32 * kb + 8 * (i >> 2) + 4 * f + (i & 3) <= first + n ? s[qb][kb][i] : kNegInf;
        }
        float mx = kNegInf;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = max_score(mx, s[qb][kb][i]);
        if (__builtin_amdgcn_ballot_w64(mx * c > m[qb] + kLazyMaxLog2) != 0) {  // wave-uniform
          const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
          mx = max_score(__uint_as_float(r32[0]), __uint_as_float(r32[1]));
          const float mn = max_score(m[qb], mx * c);
          ref[qb] = mn == kNegInf ? 0.f : mn;
          const float alpha = __builtin_amdgcn_exp2f(m[qb] - ref[qb]);
#pragma unroll
          for (int db = 0; db < DB; ++db) acc[qb][db] *= alpha;
          l[qb] *= alpha;
          m[qb] = mn;
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          float w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = __builtin_amdgcn_exp2f(fmaf(s[qb][kb][i], c, -ref[qb]));
#pragma unroll
          for (int i = 0; i < 16; i += 4) l[qb] += (w[i] + w[i + 1]) + (w[i + 2] + w[i + 3]);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            pt[qb][2 * kb + i] = make_uint4(pack2<DT>(w[8 * i], w[8 * i + 1]), pack2<DT>(w[8 * i + 2], w[8 * i + 3]),
                                            pack2<DT>(w[8 * i + 4], w[8 * i + 5]), pack2<DT>(w[8 * i + 6], w[8 * i + 7]));
        }
      }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const uint2 a = lds_tr16(lv + 16 * ks * KROW + 64 * db), b = lds_tr16(lv + (16 * ks + 8) * KROW + 64 * db);
          const uint4 vt = make_uint4(a.x, a.y, b.x, b.y);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) acc[qb][db] = mfma_32x32x16<DT>(vt, pt[qb][ks], acc[qb][db]);
        }
      }
    }
    lds_barrier();
  }

#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int first = q0 + 32 * qb;
    if (first >= len) break;  // wave-uniform
    const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(l[qb]), __float_as_uint(l[qb]), false, false);
    const float sum = __uint_as_float(r32[0]) + __uint_as_float(r32[1]);
    // A key that a query does not see has weight 0 in the tile's product, and 0 times an infinite or NaN value is NaN: a
    // block with such a result, and such a value among its own keys, is computed again one query at a time.
    float all = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) all += fabsf(acc[qb][db][i]);
    if (__builtin_amdgcn_ballot_w64(!(all < __builtin_huge_valf())) != 0) {
      bool bad = false;
      for (int t = first; t < min(len, (wave_keys + kKeys - 1) / kKeys * kKeys); ++t) {
        const elt_t<DT>* v = reinterpret_cast<const elt_t<DT>*>(vbase + (int64_t)t * p.vsn);
        for (int d = lane; d < D; d += 64) bad |= !(fabsf((float)v[d]) < __builtin_huge_valf());
      }
      if (__builtin_amdgcn_ballot_w64(bad) != 0) {
        for (int qi = first; qi < min(len, first + 32); ++qi) query_slow<DT, D>(p, begin + qi, begin, h);
        continue;
      }
    }
    if (first + n >= len) continue;
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    char* o = p.o + (int64_t)(begin + first + n) * p.osn + (int64_t)h * p.osh;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4)  // dims 32 db + 8 (i / 4) + 4 f .. + 3
        *reinterpret_cast<uint2*>(o + 64 * db + 4 * i + 8 * f) =
            make_uint2(pack2<DT>(acc[qb][db][i] * inv, acc[qb][db][i + 1] * inv),
                       pack2<DT>(acc[qb][db][i + 2] * inv, acc[qb][db][i + 3] * inv));
  }
}

template <int DT, int D, int QB>
void launch_tiles(const PromptAttn& p, hipStream_t stream) {
  const int tiles = p.n / (128 * QB) + p.seqs;  // at least the sum of ceil(length / M)
  hipLaunchKernelGGL((prompt_kernel<DT, D, QB>), dim3((uint32_t)tiles * (uint32_t)p.heads), dim3(256), 0, stream, p, tiles);
}

template <int DT>
void launch_prompt(int d, const PromptAttn& p, hipStream_t stream) {
  if constexpr (DT != SKV_F32) {
    if (d == 64) return launch_tiles<DT, 64, 1>(p, stream);
    if (d == 128) return launch_tiles<DT, 128, 1>(p, stream);
  }
  const dim3 grid((uint32_t)cdiv((int64_t)p.n * p.heads, 4));
  if (d == 16)
    hipLaunchKernelGGL((prompt_simple_kernel<DT, 16>), grid, dim3(256), 0, stream, p);
  else if (d == 32)
    hipLaunchKernelGGL((prompt_simple_kernel<DT, 32>), grid, dim3(256), 0, stream, p);
  else if (d == 64)
    hipLaunchKernelGGL((prompt_simple_kernel<DT, 64>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((prompt_simple_kernel<DT, 128>), grid, dim3(256), 0, stream, p);
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
  if ((int64_t)n_tokens * num_heads >= (int64_t)1 << 25)
    return fail(SKV_EINVAL, "%s: launch too large (tokens * heads = %lld)", who, (long long)n_tokens * num_heads);
  const PromptAttn p{(const char*)q, (const char*)k, (const char*)v, (char*)out,
                     q_stride_n * eb, q_stride_h * eb, k_stride_n * eb, k_stride_h * eb,
                     v_stride_n * eb, v_stride_h * eb, o_stride_n * eb, o_stride_h * eb,
                     cu_seqlens, scale * kLog2e, n_tokens, num_seqs, num_heads, num_heads / num_kv_heads};
  switch (dtype) {
    case SKV_F32: launch_prompt<SKV_F32>(head_dim, p, (hipStream_t)stream); break;
    case SKV_F16: launch_prompt<SKV_F16>(head_dim, p, (hipStream_t)stream); break;
    default: launch_prompt<SKV_BF16>(head_dim, p, (hipStream_t)stream); break;
  }
  return check_launch(who);
}
