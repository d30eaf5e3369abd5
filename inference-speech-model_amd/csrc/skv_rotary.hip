// Rotary append: q and k rotated by their positions, k and v written into the paged pools, one launch.
//
//   y[i] = x[i] cos - x[i + rot/2] sin,  y[i + rot/2] = x[i + rot/2] cos + x[i] sin   (or pairs 2i, 2i + 1)
//
// in fp32, rounded to the rows' type once. Three products and a sum per element against 4 (fp32: 8) bytes moved: the launch
// is bound by its bytes (bf16 8192 tokens, 32 / 8 heads x 128: 35 us, 6.4 TB/s), a decode step's by the launch and the chain
// position -> angles -> store (64 tokens: 4 us).
#include <hip/hip_runtime.h>

#include "skv_common.h"
#include "skv_rotary.h"

using namespace skv;

namespace {

template <int DT, bool INTERLEAVED>
__global__ __launch_bounds__(256) void append_rotary_kernel(RotaryAppend a) {
  rotate_rows<DT, INTERLEAVED>(a, blockIdx.x * 256u + threadIdx.x, gridDim.x * 256u);
}

template <int DT>
void launch(const RotaryAppend& a, hipStream_t stream) {
  const uint32_t blocks = (uint32_t)(cdiv(a.total, 256) < 65535 ? cdiv(a.total, 256) : 65535);
  if (a.r.interleaved)
    hipLaunchKernelGGL((append_rotary_kernel<DT, true>), dim3(blocks), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((append_rotary_kernel<DT, false>), dim3(blocks), dim3(256), 0, stream, a);
}

}  // namespace

extern "C" int skv_append_rotary(const void* q, int64_t q_stride_n, int64_t q_stride_h, const void* k_new,
                                 int64_t k_stride_n, int64_t k_stride_h, const void* v_new, int64_t v_stride_n,
                                 int64_t v_stride_h, void* q_out, int64_t qo_stride_n, int64_t qo_stride_h, void* k_out,
                                 int64_t ko_stride_n, int64_t ko_stride_h, void* k_pool, void* v_pool,
                                 const int64_t* slot_mapping, const int64_t* positions, const float* cos_sin,
                                 int64_t num_positions, int32_t rot_dim, int32_t interleaved, int32_t n_tokens,
                                 int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int64_t num_slots,
                                 int32_t dtype, void* stream) {
  const char* who = "skv_append_rotary";
  const int eb = elt_bytes(dtype);
  if (eb == 0) return fail(SKV_EDTYPE, "%s: unknown dtype %d", who, dtype);
  const int epl = 16 / eb;
  if (n_tokens < 0 || num_kv_heads <= 0 || head_dim <= 0 || num_slots < 0 || num_positions < 0 || (q && num_heads <= 0))
    return fail(SKV_EINVAL, "%s: bad sizes n=%d heads=%d kv_heads=%d head_dim=%d slots=%lld positions=%lld", who, n_tokens,
                num_heads, num_kv_heads, head_dim, (long long)num_slots, (long long)num_positions);
  if (head_dim % (2 * epl) || rot_dim <= 0 || rot_dim > head_dim || rot_dim % (2 * epl))
    return fail(SKV_EINVAL, "%s: head_dim %d and rot_dim %d (at most head_dim) must be multiples of %d", who, head_dim,
                rot_dim, 2 * epl);
  if (n_tokens == 0) return SKV_OK;
  if (!k_new || !v_new || !k_pool || !v_pool || !slot_mapping || !positions || !cos_sin || (q == nullptr) != (q_out == nullptr))
    return fail(SKV_EINVAL, "%s: null pointer argument (q and q_out go together)", who);
  if (!aligned16(q) || !aligned16(k_new) || !aligned16(v_new) || !aligned16(q_out) || !aligned16(k_out) ||
      !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(cos_sin))
    return fail(SKV_EALIGN, "%s: pointers must be 16-byte aligned", who);
  int64_t odd = k_stride_n | k_stride_h | v_stride_n | v_stride_h;
  if (q) odd |= q_stride_n | q_stride_h | qo_stride_n | qo_stride_h;
  if (k_out) odd |= ko_stride_n | ko_stride_h;
  if (odd % epl) return fail(SKV_EALIGN, "%s: strides must be multiples of %d elements", who, epl);
  RotaryAppend a{};
  const int64_t heads = (q ? num_heads : 0) + 2 * (int64_t)num_kv_heads, pairs = head_dim / (2 * epl);
  if (heads * pairs >= (int64_t)1 << 30) return fail(SKV_EINVAL, "%s: a token of %lld heads is too large", who, (long long)heads);
  a.per_tok = make_div((uint32_t)(heads * pairs));
  a.pairs = make_div((uint32_t)pairs);
  a.q_heads = q ? num_heads : 0;
  a.kv_heads = num_kv_heads;
  a.head_bytes = (uint32_t)(head_dim * eb);
  a.k_pool = (char*)k_pool;
  a.v_pool = (char*)v_pool;
  a.num_slots = num_slots;
  a.r = {cos_sin, positions, num_positions, rot_dim, interleaved ? 1 : 0};
  // Indices of a launch stay below 2^31: longer batches go in slices of tokens.
  const int64_t slice = (((int64_t)1 << 31) - 1) / (heads * pairs);
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
    a.r.positions = positions + n0;
    a.total = (uint32_t)(n * heads * pairs);
    switch (dtype) {
      case SKV_F32: launch<SKV_F32>(a, (hipStream_t)stream); break;
      case SKV_F16: launch<SKV_F16>(a, (hipStream_t)stream); break;
      default: launch<SKV_BF16>(a, (hipStream_t)stream); break;
    }
    const int rc = check_launch(who);
    if (rc != SKV_OK) return rc;
  }
  return SKV_OK;
}
