// Exact attention of one new token per sequence over its pages.
#include "oc_attn_row.cuh"

namespace {

using namespace oc;

// One warp per (sequence, query head).
template <typename T, typename C>
__global__ void __launch_bounds__(32) decode_row_kernel(const oc_paged_decode_args a) {
  __shared__ float qs[kRowMaxDim];
  pdl_launch_dependents();
  pdl_wait();
  const int seq = blockIdx.y, h = blockIdx.x, hk = h / a.group, lane = threadIdx.x;
  const T* q = static_cast<const T*>(a.q) + seq * a.q_seq_stride + h * a.q_head_stride;
  for (int d = lane; d < a.head_dim; d += 32) qs[d] = to_f32(q[d]);
  __syncwarp();
  int n = a.seq_lens[seq];
  const int64_t room = (int64_t)a.max_blocks * a.block_size;
  if (n < 0 || n > room) {
    if (lane == 0) raise_status(a.status, OC_STATUS_POSITION);
    n = n < 0 ? 0 : (int)room;
  }
  const int first = a.window > 0 && n > a.window ? n - a.window : 0;
  const int32_t* table = a.block_tables + seq * a.block_table_stride;
  auto row = [&](const void* cache, int64_t bs, int64_t hs, int64_t ts, int j) -> const C* {
    const int64_t page = table[j / a.block_size];
    if (page < 0 || page >= a.num_blocks) {
      raise_status(a.status, OC_STATUS_BAD_PAGE);
      return nullptr;
    }
    return static_cast<const C*>(cache) + page * bs + hk * hs + (j % a.block_size) * ts;
  };
  T* out = static_cast<T*>(a.out) + seq * a.out_seq_stride + h * a.out_head_stride;
  const float lse = attend_row<C>(
      qs, a.head_dim, RowScore{a.scale * a.k_scale, a.softcap, a.slopes ? a.slopes[h] : 0.f}, a.v_scale, first, n,
      [](int) { return false; },
      [&](int j) { return row(a.k_cache, a.kc_block_stride, a.kc_head_stride, a.kc_tok_stride, j); },
      [&](int j) { return row(a.v_cache, a.vc_block_stride, a.vc_head_stride, a.vc_tok_stride, j); },
      [&](int j) { return (float)(j - (n - 1)); }, [&](int d, float x) { out[d] = from_f32<T>(x); });
  if (a.lse && lane == 0) a.lse[(int64_t)seq * a.kv_heads * a.group + h] = lse;
}

template <typename T, typename C>
int launch_rows(const oc_paged_decode_args& a, void* stream) {
  return launch_pdl(decode_row_kernel<T, C>, dim3((unsigned)(a.kv_heads * a.group), (unsigned)a.num_seqs), 32, 0,
                    stream, a);
}

}  // namespace

extern "C" size_t oc_paged_decode_workspace_bytes(const oc_paged_decode_args*) { return 0; }

extern "C" int oc_paged_decode_attention(const oc_paged_decode_args* args, void* stream) {
  if (!args) return OC_ERR_INVALID;
  const oc_paged_decode_args& a = *args;
  if (a.num_seqs < 0 || a.kv_heads < 1 || a.group < 1 || a.head_dim < 1 || a.block_size < 1 || a.max_blocks < 0 ||
      a.window < 0 || a.num_sms < 1 || a.num_blocks < 0 || !(a.softcap >= 0.f))
    return OC_ERR_INVALID;
  if (a.num_seqs == 0) return OC_OK;
  if (!a.q || !a.out || !a.seq_lens || (a.max_blocks && (!a.block_tables || !a.k_cache || !a.v_cache)))
    return OC_ERR_INVALID;
  if (a.head_dim > kRowMaxDim) return OC_ERR_UNSUPPORTED;
  if (a.num_seqs > 65535) return OC_ERR_TOO_LARGE;
  if (a.cache_dtype != a.dtype && a.cache_dtype != OC_F8E4M3) return OC_ERR_UNSUPPORTED;
  const bool f8 = a.cache_dtype == OC_F8E4M3;
  switch (a.dtype) {
    case OC_F32: return f8 ? launch_rows<float, fp8_t>(a, stream) : launch_rows<float, float>(a, stream);
    case OC_F16: return f8 ? launch_rows<__half, fp8_t>(a, stream) : launch_rows<__half, __half>(a, stream);
    case OC_BF16:
      return f8 ? launch_rows<__nv_bfloat16, fp8_t>(a, stream) : launch_rows<__nv_bfloat16, __nv_bfloat16>(a, stream);
    default: return OC_ERR_UNSUPPORTED;
  }
}
