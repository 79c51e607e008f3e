// Attention of packed prompts over themselves.
#include "oc_attn_row.cuh"

namespace {

using namespace oc;

// The document of query row t: binary search in cu (docs + 1 entries); -1 if none.
__device__ __forceinline__ int find_doc(const int32_t* cu, int docs, int64_t t) {
  if (docs < 1 || t < cu[0] || t >= cu[docs]) return -1;
  int lo = 0, hi = docs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One warp per (query row, head).
template <typename T>
__global__ void __launch_bounds__(32) prompt_row_kernel(const oc_prompt_args a) {
  __shared__ float qs[kRowMaxDim];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, hk = h / a.group, lane = threadIdx.x;
  const T* q = static_cast<const T*>(a.q) + t * a.q_tok_stride + h * a.q_head_stride;
  for (int d = lane; d < a.head_dim; d += 32) qs[d] = to_f32(q[d]);
  __syncwarp();
  const int doc = a.cu_q ? find_doc(a.cu_q, a.docs, t) : 0;
  int64_t k0 = 0;
  int n = 0, pos = 0, prefix = 0;
  if (doc >= 0) {
    const int64_t q0 = a.cu_q ? a.cu_q[doc] : 0, q1 = a.cu_q ? a.cu_q[doc + 1] : a.tokens;
    k0 = a.cu_q ? a.cu_k[doc] : 0;
    int64_t k1 = a.cu_q ? a.cu_k[doc + 1] : a.key_tokens;
    if (k0 < 0 || k1 < k0 || k1 > a.key_tokens) {
      if (lane == 0) raise_status(a.status, OC_STATUS_POSITION);
      k0 = k1 = 0;
    }
    n = (int)(k1 - k0);
    pos = (int)(t - q0 + n - (q1 - q0));
    prefix = a.prefix_lens ? a.prefix_lens[doc] : 0;
  }
  const T* k = static_cast<const T*>(a.k) + k0 * a.k_tok_stride + hk * a.k_head_stride;
  const T* v = static_cast<const T*>(a.v) + k0 * a.v_tok_stride + hk * a.v_head_stride;
  T* out = static_cast<T*>(a.out) + t * a.out_tok_stride + h * a.out_head_stride;
  const float lse = attend_row<T>(
      qs, a.head_dim, RowScore{a.scale, a.softcap, a.slopes ? -a.slopes[h] : 0.f}, 1.f, 0, n,
      [&](int j) { return !(j < prefix || ((j <= pos || !a.causal) && (a.window == 0 || j > pos - a.window))); },
      [&](int j) { return k + j * a.k_tok_stride; }, [&](int j) { return v + j * a.v_tok_stride; },
      [&](int j) { return fabsf((float)(pos - j)); }, [&](int d, float x) { out[d] = from_f32<T>(x); });
  if (a.lse && lane == 0) a.lse[t * a.lse_tok_stride + h] = lse;
}

template <typename T>
int launch_rows(const oc_prompt_args& a, void* stream) {
  return launch_pdl(prompt_row_kernel<T>, dim3((unsigned)a.tokens, (unsigned)(a.kv_heads * a.group)), 32, 0, stream, a);
}

}  // namespace

extern "C" int oc_prompt_attention(const oc_prompt_args* args, void* stream) {
  if (!args) return OC_ERR_INVALID;
  const oc_prompt_args& a = *args;
  if (a.tokens < 0 || a.key_tokens < 0 || a.docs < 0 || a.kv_heads < 1 || a.group < 1 || a.head_dim < 1 ||
      a.window < 0 || a.num_sms < 1 || !(a.softcap >= 0.f) || (int64_t)a.kv_heads * a.group > 65535)
    return OC_ERR_INVALID;
  if (a.tokens == 0) return OC_OK;
  if (!a.q || !a.out || (a.cu_q && !a.cu_k) || (a.key_tokens && (!a.k || !a.v))) return OC_ERR_INVALID;
  if (a.tokens > 0x7fffffff || a.key_tokens > 0x7fffffff) return OC_ERR_TOO_LARGE;
  if (a.head_dim > kRowMaxDim) return OC_ERR_UNSUPPORTED;
  switch (a.dtype) {
    case OC_F32: return launch_rows<float>(a, stream);
    case OC_F16: return launch_rows<__half>(a, stream);
    case OC_BF16: return launch_rows<__nv_bfloat16>(a, stream);
    default: return OC_ERR_UNSUPPORTED;
  }
}
