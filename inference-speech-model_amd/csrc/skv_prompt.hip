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

template <int DT>
void launch_prompt(int d, const PromptAttn& p, hipStream_t stream) {
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
