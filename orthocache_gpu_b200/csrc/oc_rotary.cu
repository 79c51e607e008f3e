// Rotary embedding of a step's (or a prompt's) q and k, and the append of k
// and v to the paged cache, in one launch.
//
//   y_a = x_a c - x_b s,  y_b = x_b c + x_a s   for each pair (a, b) of the
//   first rotary_dim columns, c / s from float32 tables at the token's
//   position, in float32, rounded once;  cache[table[seq, pos / bs], h,
//   pos % bs] = round(k (1 / k_scale)).
//
// Every element is read once and written once (k twice where k_out is asked
// for): memory bound for prompts, launch latency for steps.
//
// Measured on one B200: one token of 32 + 4 heads of 64, 2.5 us in a graph and
// 5.9 us a call, which is the host's time; 64 tokens of 32 + 8 heads of 128,
// 3.2 us in a graph.  8191 tokens of 32 + 8 heads of 128 in bfloat16 with an
// 8-bit cache, 37 us (5.1 TB/s of 189 MB): instructions are issued in 60% of
// the cycles, and the conversions to 8 bits take as many as the rotation.
#include "oc_ops.cuh"
#include "oc_ptx.cuh"

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
    if constexpr (sizeof(T) == 1) {
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const auto two = __nv_cvt_float2_to_fp8x2(float2{x[i], x[i + 1]}, __NV_SATFINITE, __NV_E4M3);
        v.e[i].b = (uint8_t)(two & 0xff);
        v.e[i + 1].b = (uint8_t)(two >> 8);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v.e[i] = from_f32<T>(x[i]);
    }
    *reinterpret_cast<Vec<T, N>*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = from_f32<T>(x[i]);
  }
}

template <typename C, int N, bool ALIGNED>
__device__ __forceinline__ void store_cache(C* p, int n, const float (&x)[N], float inv_scale) {
  if constexpr (sizeof(C) == 1) {
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = x[i] * inv_scale;
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
  const float k_inv = 1.f / a.k_scale, v_inv = 1.f / a.v_scale;

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
          const float scale = is_k ? k_inv : v_inv;
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

// ------------------------------------------------------------------ prompts
// Enough tokens for every warp of the machine: the loads of the kernel above,
// at most a few per thread between two stores, leave HBM half idle, so here
// each warp keeps its input on the way ahead of it: a ring of kStages bulk
// copies of up to 4 KB (a run of heads of q, k or v, which lie side by side),
// 192 KB an SM.  A warp takes an equal run of those pieces, token after token.
// Lane (head, column) holds its column's table entries; those, the page and
// the position of the next tokens are read while this one is worked on.
constexpr int kStages = 3, kStageBytes = 4096, kStreamWarps = 16;

// JOINED: q, k and v of a token lie side by side and make one piece.
template <typename T, typename C, int N, bool INTER, bool JOINED>
__global__ void __launch_bounds__(kStreamWarps * 32, 1)
    rotary_stream_kernel(const __grid_constant__ oc_rotary_args a, int columns) {
  constexpr int NT = INTER ? N / 2 : N;  // table entries of a vector
  extern __shared__ __align__(128) char ring[];
  __shared__ __align__(8) uint64_t bars[kStreamWarps][kStages];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t my_bar = smem_u32(bars[warp]), my_ring = smem_u32(ring) + warp * kStages * kStageBytes;
  const char* const mine = ring + warp * kStages * kStageBytes;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(my_bar + 8 * i, 1);
    mbar_init_fence();
  }
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait();

  // a token's pieces: runs of at most `most` heads of q, of k, of v, or all of them
  const int row = a.head_dim * (int)sizeof(T), most = kStageBytes / row;
  const int hq = a.q_heads, hk = a.kv_heads, heads = hq + hk * (a.v ? 2 : 1);
  const int nq = (hq + most - 1) / most, nk = (hk + most - 1) / most;
  const int pieces = JOINED ? 1 : nq + nk * (a.v ? 2 : 1);
  struct Piece {
    int part, h0, heads;  // 0 q, 1 k, 2 v; the piece's first head in the part, and how many
  };
  auto piece_of = [&](int i) {
    Piece p;
    p.part = JOINED || i < nq ? 0 : i < nq + nk ? 1 : 2;
    p.h0 = (p.part == 0 ? i : p.part == 1 ? i - nq : i - nq - nk) * most;
    p.heads = min(most, (JOINED ? heads : p.part == 0 ? hq : hk) - p.h0);
    return p;
  };
  const int64_t warps = (int64_t)gridDim.x * kStreamWarps, me = (int64_t)blockIdx.x * kStreamWarps + warp;
  const int64_t begin = a.tokens * pieces * me / warps, end = a.tokens * pieces * (me + 1) / warps;
  if (begin >= end) return;
  int64_t t = begin / pieces;
  int i = (int)(begin - t * pieces);
  int64_t ld_t = t, ld_left = end - begin;
  int ld_piece = i, ld_stage = 0;
  auto issue = [&]() {  // the next piece's copy
    if (ld_left <= 0) return;
    --ld_left;
    if (lane == 0) {
      const Piece p = piece_of(ld_piece);
      const char* src = static_cast<const char*>(p.part == 0 ? a.q : p.part == 1 ? a.k : a.v);
      const int64_t stride = p.part == 0 ? a.q_tok_stride : p.part == 1 ? a.k_tok_stride : a.v_tok_stride;
      const uint32_t bar = my_bar + 8 * ld_stage, bytes = (uint32_t)(p.heads * row);
      mbar_arrive_expect_tx(bar, bytes);
      bulk_load(my_ring + ld_stage * kStageBytes, src + ld_t * stride * (int64_t)sizeof(T) + (int64_t)p.h0 * row, bytes, bar);
    }
    ld_stage = ld_stage + 1 == kStages ? 0 : ld_stage + 1;
    if (++ld_piece == pieces) {
      ld_piece = 0;
      ++ld_t;
    }
  };

  // this lane's column
  const int half = a.rotary_dim / 2, turning = (INTER ? a.rotary_dim : half) / N;
  const int col = lane % columns, hl = lane / columns, side = 32 / columns;
  const bool active = hl < side, turn = col < turning, paired = !INTER && turn;
  const int lo = turn ? col * N : a.rotary_dim + (col - turning) * N;
  const int shift = a.k_cache ? __ffs(a.block_size) - 1 : 0;
  const float sign = a.flags & OC_ROTARY_INVERSE ? -1.f : 1.f;
  const float k_inv = 1.f / a.k_scale, v_inv = 1.f / a.v_scale;

  struct Place {
    int64_t pos, seq;
  };
  auto place_of = [&](int64_t t) {
    Place p = {0, -1};  // beyond the last token: a place that exists and appends nothing
    if (t < a.tokens) {
      p.pos = a.positions_64 ? static_cast<const int64_t*>(a.positions)[t]
                             : (int64_t) static_cast<const int32_t*>(a.positions)[t];
      if (a.k_cache) p.seq = a.seq_ids ? a.seq_ids[t] : t;
    }
    return p;
  };
  struct Token {
    float c[NT], s[NT];
    int page, slot;  // page -2: no append
  };
  auto look = [&](Place p) {
    Token k;
    const bool inside = half == 0 || (p.pos >= 0 && p.pos < a.table_rows);
    bool bad = !inside;
    k.page = -2;
    k.slot = 0;
    if (p.seq >= 0) {
      const int64_t column = p.pos >> shift;
      if (inside && p.pos >= 0 && p.seq < a.num_seqs && column < a.max_blocks) {
        k.page = a.block_tables[p.seq * a.block_table_stride + column];
        k.page = k.page < 0 || k.page >= a.num_blocks ? -1 : k.page;
        k.slot = (int)(p.pos & (a.block_size - 1));
      } else {
        bad = true;
      }
    }
    if (bad && lane == 0) raise_status(a.status, OC_STATUS_POSITION);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      k.c[j] = 1.f;
      k.s[j] = 0.f;
    }
    if (turn) {
      const float* ct = a.cos_tab + (inside ? p.pos : 0) * half + (INTER ? lo / 2 : lo);
      const float* st = a.sin_tab + (inside ? p.pos : 0) * half + (INTER ? lo / 2 : lo);
      constexpr int W = NT < 4 ? NT : 4;
#pragma unroll
      for (int j = 0; j < NT; j += W) {
        const Vec<float, W> cv = *reinterpret_cast<const Vec<float, W>*>(ct + j);
        const Vec<float, W> sv = *reinterpret_cast<const Vec<float, W>*>(st + j);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          k.c[j + e] = cv.e[e];
          k.s[j + e] = sv.e[e] * sign;
        }
      }
    }
    return k;
  };

#pragma unroll
  for (int s = 0; s < kStages; ++s) issue();
  const Place p0 = place_of(t), p1 = place_of(t + 1);
  Token now = look(p0), next = look(p1);
  Place ahead = place_of(t + 2);
  int stage = 0;
  uint32_t parity = 0;
  bool late = false;
  int64_t left = end - begin;
  for (; left > 0; --left) {
    if (now.page == -1 && lane == 0) raise_status(a.status, OC_STATUS_BAD_PAGE);
    const Piece p = piece_of(i);
    late = !__all_sync(0xffffffffu, mbar_wait_bounded(my_bar + 8 * stage, parity >> stage & 1, kPolls));
    if (late) break;
    parity ^= 1u << stage;
    const char* in = mine + stage * kStageBytes;
    // where a head goes: out (q, or the copy of k), and the cache; of the piece's part, or looked up head by head
    T* out = nullptr;
    C* cache = nullptr;
    int64_t out_head = 0, cache_head = 0;
    float inv = 1.f;
    auto place = [&](int part) {
      if (part == 0) {
        out = static_cast<T*>(a.q_out) + t * a.qo_tok_stride + lo;
        out_head = a.qo_head_stride;
        cache = nullptr;
      } else if (part == 1) {
        out = a.k_out ? static_cast<T*>(a.k_out) + t * a.ko_tok_stride + lo : nullptr;
        out_head = a.ko_head_stride;
        cache = now.page >= 0 ? static_cast<C*>(a.k_cache) + now.page * a.kc_block_stride + now.slot * a.kc_tok_stride + lo
                              : nullptr;
        cache_head = a.kc_head_stride;
        inv = k_inv;
      } else {
        out = nullptr;
        cache = now.page >= 0 ? static_cast<C*>(a.v_cache) + now.page * a.vc_block_stride + now.slot * a.vc_tok_stride + lo
                              : nullptr;
        cache_head = a.vc_head_stride;
        inv = v_inv;
      }
    };
    if (!JOINED) place(p.part);
    if (active) {
#pragma unroll 2
      for (int h = hl; h < p.heads; h += side) {
        const int part = !JOINED ? p.part : h < hq ? 0 : h < hq + hk ? 1 : 2;
        const int head = !JOINED ? p.h0 + h : part == 0 ? h : part == 1 ? h - hq : h - hq - hk;
        if (JOINED) place(part);
        const T* src = reinterpret_cast<const T*>(in + h * row) + lo;
        const Vec<T, N> xv = *reinterpret_cast<const Vec<T, N>*>(src);
        Vec<T, N> yv = {};
        if (paired) yv = *reinterpret_cast<const Vec<T, N>*>(src + half);
        float x[N], y[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          x[j] = to_f32(xv.e[j]);
          y[j] = to_f32(yv.e[j]);
        }
        if (turn && part != 2) {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            float& u = INTER ? x[2 * j] : x[j];
            float& w = INTER ? x[2 * j + 1] : y[j];
            const float u0 = u, w0 = w;
            u = u0 * now.c[j] - w0 * now.s[j];
            w = w0 * now.c[j] + u0 * now.s[j];
          }
        }
        if (out) {
          T* dst = out + head * out_head;
          store_vec<T, N, true>(dst, N, x);
          if (paired) store_vec<T, N, true>(dst + half, N, y);
        }
        if (cache) {
          C* dst = cache + head * cache_head;
          store_cache<C, N, true>(dst, N, x, inv);
          if (paired) store_cache<C, N, true>(dst + half, N, y, inv);
        }
      }
    }
    __syncwarp();  // every lane has read the stage before it is filled again
    issue();
    stage = stage + 1 == kStages ? 0 : stage + 1;
    if (++i == pieces) {
      i = 0;
      ++t;
      now = next;
      next = look(ahead);
      ahead = place_of(t + 2);
    }
  }
  if (late) {  // report it, and let this warp's copies land before the CTA's memory is reused
    if (lane == 0) raise_status(a.status, OC_STATUS_TIMEOUT);
#pragma unroll 1
    for (int i = 0; i < kStages && i < left; ++i) {
      mbar_wait_bounded(my_bar + 8 * stage, parity >> stage & 1, kLandPolls);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
  }
}

// The heads of a token side by side, whole vectors, 32 columns at most, and a token for every warp.
template <typename T, int N, bool INTER>
bool streams(const oc_rotary_args& a, int& columns) {
  const int half = a.rotary_dim / 2;
  columns = (INTER ? a.rotary_dim : half) / N + (a.head_dim - a.rotary_dim) / N;
  auto dense = [&](const void* p, int64_t head_stride, int heads) { return !p || heads == 1 || head_stride == a.head_dim; };
  return columns <= 32 && a.head_dim * (int)sizeof(T) <= kStageBytes && a.tokens >= (int64_t)a.num_sms * kStreamWarps &&
         dense(a.q, a.q_head_stride, a.q_heads) && dense(a.k, a.k_head_stride, a.kv_heads) &&
         dense(a.v, a.v_head_stride, a.kv_heads) && aligned_to(a.cos_tab, 16) && aligned_to(a.sin_tab, 16) && half % 4 == 0;
}

template <typename T, typename C, int N, bool INTER>
int launch_aligned(const oc_rotary_args& a, void* stream) {
  int columns;
  if (!streams<T, N, INTER>(a, columns)) return launch<T, C, N, true, INTER>(a, stream);
  constexpr int smem = kStreamWarps * kStages * kStageBytes;
  // parts of one projection's output, small enough for one piece a token (25147 tokens of 8 + 2 heads
  // of 128: 53 us apart, 40 joined)
  const bool joined = a.q && a.k && a.v && a.q_tok_stride == a.k_tok_stride && a.q_tok_stride == a.v_tok_stride &&
                      static_cast<const T*>(a.q) + a.q_heads * a.head_dim == a.k &&
                      static_cast<const T*>(a.k) + a.kv_heads * a.head_dim == a.v &&
                      (int64_t)(a.q_heads + 2 * a.kv_heads) * a.head_dim * sizeof(T) <= kStageBytes;
  auto kernel = joined ? rotary_stream_kernel<T, C, N, INTER, true> : rotary_stream_kernel<T, C, N, INTER, false>;
  static std::atomic<uint64_t> ready[2];
  if (!allow_smem(reinterpret_cast<const void*>(kernel), ready[joined], smem)) return OC_ERR_CUDA;
  const int64_t ctas = (a.tokens + kStreamWarps - 1) / kStreamWarps;
  return launch_pdl(kernel, dim3((unsigned)(ctas < a.num_sms ? ctas : a.num_sms)), dim3(kStreamWarps * 32), smem, stream,
                    a, columns);
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
  if (vec) return inter ? launch_aligned<T, C, N, true>(a, stream) : launch_aligned<T, C, N, false>(a, stream);
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
  if (a.k_cache && (!a.v_cache || !a.v || !a.kv_heads || !a.block_tables || a.block_size < 1 || (a.block_size & (a.block_size - 1)) ||
                    a.max_blocks < 0 ||
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
