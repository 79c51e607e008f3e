// Rotary embedding of a step's (or a prompt's) q and k, and the append of k
// and v to the paged cache, in one launch.
//
//   y_a = x_a c - x_b s,  y_b = x_b c + x_a s   for each pair (a, b) of the
//   first rotary_dim columns, c / s from float32 tables at the token's
//   position, in float32, rounded once;  cache[table[seq, pos / bs], h,
//   pos % bs] = round(k / k_scale).
//
// Every element is read once and written once (k twice where k_out is asked
// for): memory bound for prompts, launch latency for steps.
#include "oc_ops.cuh"

namespace {

using namespace oc;

template <typename T, int N, bool ALIGNED>
__device__ __forceinline__ void load_vec(const T* p, int n, float (&x)[N]) {
  if constexpr (ALIGNED) {
    const Vec<T, N> v = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32(v.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = i < n ? to_f32(p[i]) : 0.f;
  }
}

template <typename T, int N, bool ALIGNED>
__device__ __forceinline__ void store_vec(T* p, int n, const float (&x)[N]) {
  if constexpr (ALIGNED) {
    Vec<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v.e[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Vec<T, N>*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = from_f32<T>(x[i]);
  }
}

template <typename C, int N, bool ALIGNED>
__device__ __forceinline__ void store_cache(C* p, int n, const float (&x)[N], float scale) {
  if constexpr (sizeof(C) == 1) {
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = __fdiv_rn(x[i], scale);
    store_vec<C, N, ALIGNED>(p, n, y);
  } else {
    store_vec<C, N, ALIGNED>(p, n, x);
  }
}

// One thread: one vector of columns (two, a pair of vectors rotary_dim / 2
// apart, in the half layout) of one token, over the heads ty, ty + HL, ...:
// the position, the page lookup and the table entries are read once for all
// heads.  blockDim = (columns, heads side by side, tokens).
template <typename T, typename C, int N, bool ALIGNED, bool INTER>
__global__ void __launch_bounds__(256) rotary_append_kernel(const oc_rotary_args a, int head_lanes, int columns) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = (int64_t)blockIdx.x * blockDim.z + threadIdx.z;
  if (t >= a.tokens) return;
  const int64_t pos = a.positions_64 ? static_cast<const int64_t*>(a.positions)[t]
                                     : (int64_t) static_cast<const int32_t*>(a.positions)[t];
  const bool first = threadIdx.x == 0 && threadIdx.y == 0 && blockIdx.y == 0;
  const int half = a.rotary_dim / 2;
  int64_t row = pos;
  if (half && (pos < 0 || pos >= a.table_rows)) {
    if (first) raise_status(a.status, OC_STATUS_POSITION);
    row = 0;
  }
  // the token's slot
  int64_t page = -1;
  int slot = 0;
  if (a.k_cache) {
    const int64_t seq = a.seq_ids ? a.seq_ids[t] : t;
    if (seq >= 0) {
      const int64_t col = pos / a.block_size;
      if (pos < 0 || seq >= a.num_seqs || col >= a.max_blocks || row != pos) {
        if (first) raise_status(a.status, OC_STATUS_POSITION);
      } else {
        page = a.block_tables[seq * a.block_table_stride + col];
        slot = (int)(pos - col * a.block_size);
        if (page < 0 || page >= a.num_blocks) {
          if (first) raise_status(a.status, OC_STATUS_BAD_PAGE);
          page = -1;
        }
      }
    }
  }
  const T* qt = static_cast<const T*>(a.q) + t * a.q_tok_stride;
  T* qo = static_cast<T*>(a.q_out) + t * a.qo_tok_stride;
  const T* kt = static_cast<const T*>(a.k) + t * a.k_tok_stride;
  T* ko = a.k_out ? static_cast<T*>(a.k_out) + t * a.ko_tok_stride : nullptr;
  const T* vt = static_cast<const T*>(a.v) + t * a.v_tok_stride;
  C* kc = page >= 0 ? static_cast<C*>(a.k_cache) + page * a.kc_block_stride + (int64_t)slot * a.kc_tok_stride : nullptr;
  C* vc = page >= 0 ? static_cast<C*>(a.v_cache) + page * a.vc_block_stride + (int64_t)slot * a.vc_tok_stride : nullptr;
  const int nh = a.q_heads + a.kv_heads * (a.v ? 2 : 1);

  for (int i = threadIdx.x; i < columns; i += blockDim.x) {
    // columns [lo, lo + n) and, in the half layout, their partners [hi, hi + n)
    int lo, hi = -1, n;
    bool turn = true;
    const int turning = INTER ? (a.rotary_dim + N - 1) / N : (half + N - 1) / N;
    if (i < turning) {
      lo = i * N;
      n = min(N, (INTER ? a.rotary_dim : half) - lo);
      if (!INTER) hi = half + lo;
    } else {
      lo = a.rotary_dim + (i - turning) * N;
      n = min(N, a.head_dim - lo);
      turn = false;
    }
    float c[N], s[N];
    if (turn) {
      const float* ct = a.cos_tab + row * half + (INTER ? lo / 2 : lo);
      const float* st = a.sin_tab + row * half + (INTER ? lo / 2 : lo);
#pragma unroll
      for (int j = 0; j < (INTER ? N / 2 : N); ++j) {
        const bool in = ALIGNED || (INTER ? 2 * j < n : j < n);
        c[j] = in ? ct[j] : 1.f;
        s[j] = in ? st[j] : 0.f;
        if (a.flags & OC_ROTARY_INVERSE) s[j] = -s[j];
      }
    }
#pragma unroll 4
    for (int h = blockIdx.y * blockDim.y + threadIdx.y; h < nh; h += head_lanes) {
      const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.kv_heads;
      const int hk = is_q ? h : is_k ? h - a.q_heads : h - a.q_heads - a.kv_heads;
      const T* src = is_q ? qt + hk * a.q_head_stride : is_k ? kt + hk * a.k_head_stride : vt + hk * a.v_head_stride;
      float x[N], y[N];
      load_vec<T, N, ALIGNED>(src + lo, n, x);
      if (!INTER && hi >= 0) load_vec<T, N, ALIGNED>(src + hi, n, y);
      if (turn && (is_q || is_k)) {
        if constexpr (INTER) {
#pragma unroll
          for (int j = 0; j < N / 2; ++j) {
            const float u = x[2 * j], w = x[2 * j + 1];
            x[2 * j] = u * c[j] - w * s[j];
            x[2 * j + 1] = w * c[j] + u * s[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const float u = x[j], w = y[j];
            x[j] = u * c[j] - w * s[j];
            y[j] = w * c[j] + u * s[j];
          }
        }
      }
      if (is_q) {
        T* dst = qo + hk * a.qo_head_stride;
        store_vec<T, N, ALIGNED>(dst + lo, n, x);
        if (!INTER && hi >= 0) store_vec<T, N, ALIGNED>(dst + hi, n, y);
      } else {
        if (is_k && ko) {
          T* dst = ko + hk * a.ko_head_stride;
          store_vec<T, N, ALIGNED>(dst + lo, n, x);
          if (!INTER && hi >= 0) store_vec<T, N, ALIGNED>(dst + hi, n, y);
        }
        if (kc) {
          C* dst = is_k ? kc + hk * a.kc_head_stride : vc + hk * a.vc_head_stride;
          const float scale = is_k ? a.k_scale : a.v_scale;
          store_cache<C, N, ALIGNED>(dst + lo, n, x, scale);
          if (!INTER && hi >= 0) store_cache<C, N, ALIGNED>(dst + hi, n, y, scale);
        }
      }
    }
  }
}

template <typename T, typename C, int N, bool ALIGNED, bool INTER>
int launch(const oc_rotary_args& a, void* stream) {
  const int half = a.rotary_dim / 2;
  const int turning = INTER ? (a.rotary_dim + N - 1) / N : (half + N - 1) / N;
  const int columns = turning + (a.head_dim - a.rotary_dim + N - 1) / N;
  const int bx = columns < 256 ? columns : 256;
  const int nh = a.q_heads + a.kv_heads * (a.v ? 2 : 1);
  // heads per thread: as many as keep every SM full (1024 threads), one for small calls
  const int64_t threads = a.tokens * columns * nh, full = (int64_t)a.num_sms * 2048;
  int per = (int)(threads / full);
  per = per < 1 ? 1 : per > 12 ? 12 : per;
  int lanes = (nh + per - 1) / per;
  int by = 256 / bx < lanes ? 256 / bx : lanes;
  if (by < 1) by = 1;
  int gy = (lanes + by - 1) / by;
  lanes = by * gy;
  int bz = 256 / (bx * by);
  if (bz < 1) bz = 1;
  if (bz > 64) bz = 64;
  const int64_t gx = (a.tokens + bz - 1) / bz;
  if (gx > 0x7fffffff || gy > 65535) return OC_ERR_TOO_LARGE;
  return launch_pdl(rotary_append_kernel<T, C, N, ALIGNED, INTER>, dim3((unsigned)gx, (unsigned)gy),
                    dim3((unsigned)bx, (unsigned)by, (unsigned)bz), 0, stream, a, lanes, columns);
}

// 16-byte vectors of T where every row starts at a multiple of 16 bytes and
// the rotated part splits into whole vectors; else elements one by one.
template <typename T, typename C>
int dispatch(const oc_rotary_args& a, void* stream) {
  constexpr int N = 16 / sizeof(T);
  const bool inter = a.flags & OC_ROTARY_INTERLEAVED;
  const int half = a.rotary_dim / 2;
  bool vec = a.head_dim % N == 0 && a.rotary_dim % N == 0 && (inter || half % N == 0);
  auto ok = [&](const void* p, int64_t s0, int64_t s1, int64_t s2, size_t bytes) {
    if (p) vec = vec && aligned_to(p, bytes) && s0 % N == 0 && s1 % N == 0 && s2 % N == 0;
  };
  ok(a.q, a.q_tok_stride, a.q_head_stride, 0, 16);
  ok(a.q_out, a.qo_tok_stride, a.qo_head_stride, 0, 16);
  ok(a.k, a.k_tok_stride, a.k_head_stride, 0, 16);
  ok(a.v, a.v_tok_stride, a.v_head_stride, 0, 16);
  ok(a.k_out, a.ko_tok_stride, a.ko_head_stride, 0, 16);
  ok(a.k_cache, a.kc_block_stride, a.kc_head_stride, a.kc_tok_stride, N * sizeof(C));
  ok(a.v_cache, a.vc_block_stride, a.vc_head_stride, a.vc_tok_stride, N * sizeof(C));
  if (vec) return inter ? launch<T, C, N, true, true>(a, stream) : launch<T, C, N, true, false>(a, stream);
  return inter ? launch<T, C, 2, false, true>(a, stream) : launch<T, C, 1, false, false>(a, stream);
}

}  // namespace

extern "C" int oc_rotary_append_paged(const oc_rotary_args* args, void* stream) {
  if (!args) return OC_ERR_INVALID;
  const oc_rotary_args& a = *args;
  if (a.tokens < 0 || a.head_dim < 1 || a.q_heads < 0 || a.kv_heads < 0 || a.rotary_dim < 0 || (a.rotary_dim & 1) ||
      a.rotary_dim > a.head_dim || a.num_sms < 1)
    return OC_ERR_INVALID;
  if (a.tokens == 0 || a.q_heads + a.kv_heads == 0) return OC_OK;
  if (!a.positions || (a.q_heads && (!a.q || !a.q_out)) || (a.kv_heads && (!a.k || (!a.k_out && !a.k_cache))) ||
      (a.rotary_dim && (!a.cos_tab || !a.sin_tab || a.table_rows < 1)))
    return OC_ERR_INVALID;
  if (a.k_cache && (!a.v_cache || !a.v || !a.kv_heads || !a.block_tables || a.block_size < 1 || a.max_blocks < 0 ||
                    a.num_seqs < 0 || a.num_blocks < 0))
    return OC_ERR_INVALID;
  if (!a.k_cache && (a.v || a.v_cache)) return OC_ERR_INVALID;
  const int cache = a.k_cache ? a.cache_dtype : a.dtype;
  if (cache != a.dtype && cache != OC_F8E4M3) return OC_ERR_UNSUPPORTED;
  const bool f8 = cache == OC_F8E4M3;
  switch (a.dtype) {
    case OC_F32: return f8 ? dispatch<float, fp8_t>(a, stream) : dispatch<float, float>(a, stream);
    case OC_F16: return f8 ? dispatch<__half, fp8_t>(a, stream) : dispatch<__half, __half>(a, stream);
    case OC_BF16:
      return f8 ? dispatch<__nv_bfloat16, fp8_t>(a, stream) : dispatch<__nv_bfloat16, __nv_bfloat16>(a, stream);
    default: return OC_ERR_UNSUPPORTED;
  }
}
