// Attention of packed prompts over themselves.
//
//   s_ij = cap(scale q_i.k_j) - slope |p_i - j|,  o_i = sum_j 2^(s_ij - m_i) v_j / sum_j 2^(s_ij - m_i)
//
// over the keys that the mask leaves.  4 D operations per query-key pair
// against one exponential: on this part a 128 x 128 tile takes 1024 cycles of
// the tensor cores at D = 128 (512 at D = 64) and 1024 cycles of the
// exponential unit (16 a cycle), so the two are kept busy at the same time:
// a CTA works on two tiles of 128 queries in turn, and while one tile's scores
// go through the softmax the tensor cores multiply for the other.  (Short
// documents and windows at up to 64 columns: two CTAs an SM, a tile each.)
//
// Roles: 4 + 4 softmax warps (a thread per query row), one warp that issues
// the matrix instructions, one that issues the copies.  Q, K and V arrive by
// TMA in 128-byte-swizzled panels of 64 columns; S = Q K^T and O += P V
// accumulate in tensor memory (S0 S1 O0 O1, at most 512 columns); P overwrites S in 16
// bits and is the second product's operand from there, V is read as it lies
// (contiguous in D).  O is rescaled only when a row's maximum has grown by
// 2^8: almost never after the first tiles.  Key tiles that the mask hides from
// all 128 queries are neither copied nor multiplied.
//
// A key that the mask hides weighs 0, but 0 times an infinity or NaN in its
// value (or in a neighbouring document that shares the tile) is not 0; rows
// whose sum comes out not finite are therefore computed again from the
// definition, over their visible keys only.
//
// P is rounded to 16 bits, since a matrix instruction takes both operands in one
// type; the sum that normalises is that of the rounded weights, in float32.
// Against 64 bits an output is then off by 0.0021 (bfloat16, 8192 tokens) where
// one rounding alone gives 0.0016.
//
// Measured on one B200: 8192 tokens, causal, 32 heads of 128 in bfloat16, 439
// us in a graph (1250 TFLOP/s; one call after another under the power cap,
// 516), tensor cores and exponential unit each 62% busy: what is left is the
// hand-over between the two and the first and last tiles of a CTA.  4099
// tokens in 7 documents, capped scores, a window of 1024, 16 heads of 128: 45
// us: the cap's polynomial is 6 packed operations for two scores, and the 2.2
// CTAs an SM end unevenly: tiles go out longest first within a document, but
// documents in their order.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>
#include <type_traits>

#include "oc_attn_row.cuh"
#include "oc_tc.cuh"

namespace {

using namespace oc;

// ------------------------------------------------------------------ documents and masks
// One document: query rows [q0, q1), keys [k0, k0 + n); query row r sits at r - q0 + shift.
struct Doc {
  int64_t q0, q1, k0;
  int n, shift, prefix;
};

// Rows outside every document form documents -1 (before the first) and docs (after the last), without keys.
__device__ __forceinline__ Doc get_doc(const oc_prompt_args& a, int d) {
  Doc r = {0, a.tokens, 0, (int)a.key_tokens, 0, 0};
  if (a.cu_q) {
    r.q0 = d < 0 ? 0 : a.cu_q[d];
    r.q1 = d >= a.docs ? a.tokens : a.cu_q[d + 1];
    bool bad = r.q0 < 0 || r.q1 < r.q0 || r.q1 > a.tokens;
    r.n = 0;
    if (d >= 0 && d < a.docs) {
      r.k0 = a.cu_k[d];
      const int64_t k1 = a.cu_k[d + 1];
      bad = bad || r.k0 < 0 || k1 < r.k0 || k1 > a.key_tokens;
      r.n = (int)(k1 - r.k0);
    }
    if (bad) {
      raise_status(a.status, OC_STATUS_POSITION);
      r.q0 = min(max(r.q0, (int64_t)0), a.tokens);
      r.q1 = min(max(r.q1, r.q0), a.tokens);
      r.k0 = 0;
      r.n = 0;
    }
  }
  r.shift = r.n - (int)(r.q1 - r.q0);
  r.prefix = a.prefix_lens && d >= 0 && d < a.docs ? min(max(a.prefix_lens[d], 0), r.n) : 0;
  return r;
}

// Keys that a query at position p sees: [lo, hi) and [0, prefix).
struct Sight {
  int lo, hi;
};
__device__ __forceinline__ Sight sight_of(const oc_prompt_args& a, const Doc& d, int p) {
  const int64_t lo = a.window > 0 ? (int64_t)p - a.window + 1 : 0;  // p may be negative: fewer keys than queries
  return Sight{lo < 0 ? 0 : (int)lo, a.causal ? min(p + 1, d.n) : d.n};
}

// ------------------------------------------------------------------ the tiled kernel
constexpr int kBM = 128;       // queries of a tile; one or two tiles a CTA
constexpr int kBN = 128;       // keys of a tile

template <int DP, int TILES_>
struct Tile {
  static constexpr int PANEL = kBN * 128;      // bytes of 128 rows of 64 columns
  static constexpr int PANELS = DP / 64;
  static constexpr int BYTES = PANEL * PANELS;  // of a Q, K or V tile
  static constexpr int TILES = TILES_;                  // of queries, a CTA
  static constexpr int PER_SM = 3 - TILES;              // resident CTAs
  static constexpr int STAGES = DP == 64 && TILES == 2 ? 8 : 5;  // 4 at least: copies are awaited a tile ahead
  static constexpr int SMEM = (TILES + STAGES) * BYTES + 1024;
  static constexpr int MATRIX = 4 * TILES, COPY = MATRIX + 1;  // warps, after the softmax warps of every tile; two more idle
  static constexpr int THREADS = 32 * (MATRIX + 4);
  static constexpr int COLUMNS = 512 / PER_SM;          // of tensor memory: the tiles' scores, then their outputs
  static constexpr int OUT = 128 * TILES;
};

struct Maps {
  CUtensorMap q, k, v;
  int q_swap, k_swap, v_swap;  // dimensions are (columns, head, row), or (columns, row, head)
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
// a + the two 16-bit numbers of a word: an addition of mixed types each, without conversions (a causal prompt of 8192
// tokens, 32 heads of 128: 448 -> 441 us; capped, a window of 1024: 79 -> 75).
template <bool BF16>
__device__ __forceinline__ float2 add16(float2 a, uint32_t two) {
  float2 r;
  if constexpr (BF16)
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; add.rn.f32.bf16 %0, l, %3; add.rn.f32.bf16 %1, h, %4;}"
        : "=f"(r.x), "=f"(r.y)
        : "r"(two), "f"(a.x), "f"(a.y));
  else
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; add.rn.f32.f16 %0, l, %3; add.rn.f32.f16 %1, h, %4;}"
        : "=f"(r.x), "=f"(r.y)
        : "r"(two), "f"(a.x), "f"(a.y));
  return r;
}

// k tanh(r x) of 128 scores.  |r x| <= 5/8 for the whole warp, the rule with
// caps of some tens: x times an even polynomial, fitted to the smallest largest
// absolute error (3e-8), on the multiply units, with k and the powers of r in
// the coefficients (6 packed operations for two scores; the coefficients are
// made anew for each tile, since 10 more registers held across tiles spill); else
// 1 - 2 / (1 + 2^(2 x log2 e)), two operations of the exponential unit a score
// (absolute error some 1e-7).
__device__ __forceinline__ void cap_scores(float* s, float r, float k) {
  float tops[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 128; i += 2) tops[i >> 1 & 3] = max3_abs(tops[i >> 1 & 3], s[i], s[i + 1]);
  const float top = max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[3]);
  if (__all_sync(0xffffffffu, fabsf(top * r) <= 0.625f)) {
    float f;
    asm volatile("mul.f32 %0, %1, %2;" : "=f"(f) : "f"(k), "f"(r));  // volatile: not moved out of the loop over tiles
    const float r2 = r * r;
    const float2 c0 = both(0.999999463558197f * f), c1 = both(-0.33330482244491577f * (f *= r2)),
                 c2 = both(0.13291031122207642f * (f *= r2)), c3 = both(-0.051362860947847366f * (f *= r2)),
                 c4 = both(0.014530060812830925f * (f *= r2));
#pragma unroll
    for (int i = 0; i < 128; i += 2) {
      const float2 v = {s[i], s[i + 1]}, q = mul2(v, v);
      float2 p = fma2(q, c4, c3);
      p = fma2(q, p, c2);
      p = fma2(q, p, c1);
      p = fma2(q, p, c0);
      p = mul2(p, v);
      s[i] = p.x;
      s[i + 1] = p.y;
    }
  } else {
    const float z = 2.f * kLog2e * r;
#pragma unroll
    for (int i = 0; i < 128; ++i) {
      float y;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + ex2(s[i] * z)));
      s[i] = fmaf(-2.f * k, y, k);
    }
  }
}

// GENERAL: scores are capped, biased or scaled by a factor that is not
// positive; else the scale is folded into the exponential.  LSE: the logarithm
// of the sum is asked for.
template <typename T, int DP, int TILES, bool GENERAL, bool LSE>
__global__ void __launch_bounds__(Tile<DP, TILES>::THREADS, Tile<DP, TILES>::PER_SM)
    prompt_kernel(const __grid_constant__ oc_prompt_args a, const __grid_constant__ Maps maps) {
  using L = Tile<DP, TILES>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ char raw[];
  __shared__ __align__(8) uint64_t bars[2 * L::STAGES + 11];
  __shared__ uint32_t tmem_at;
  __shared__ Doc s_doc;
  __shared__ int s_tile;  // which TILES query tiles of the document; -1: none

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t bar0 = smem_u32(bars);
  auto kv_full = [&](int s) { return bar0 + 8 * s; };
  auto kv_empty = [&](int s) { return bar0 + 8 * (L::STAGES + s); };
  auto q_full = [&](int t) { return bar0 + 8 * (2 * L::STAGES + t); };
  auto s_full = [&](int t) { return bar0 + 8 * (2 * L::STAGES + 2 + t); };
  auto p_full = [&](int t) { return bar0 + 8 * (2 * L::STAGES + 4 + t); };
  auto o_full = [&](int t) { return bar0 + 8 * (2 * L::STAGES + 6 + t); };
  auto p_most = [&](int t) { return bar0 + 8 * (2 * L::STAGES + 8 + t); };  // P of the tile's first 96 keys

  const uint32_t stopped = bar0 + 8 * (2 * L::STAGES + 10);  // the products in flight when a wait ran out have ended
  if (warp == L::MATRIX && lane == 0) {
    mbar_init(stopped, 1);
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(q_full(t), 1);
      mbar_init(s_full(t), 1);
      mbar_init(p_full(t), 4);
      mbar_init(p_most(t), 4);
      mbar_init(o_full(t), 1);
    }
    mbar_init_fence();
  }
  if (warp == L::COPY) tmem_alloc(smem_u32(&tmem_at), L::COLUMNS);
  pdl_launch_dependents();
  pdl_wait();
  // the query tiles of this CTA, the document's last first (causal: the longest)
  if (warp == 0) {
    int before = 0, doc = -2, tile = -1;
    for (int d0 = a.cu_q ? -1 : 0; d0 <= a.docs && tile < 0; d0 += 32) {
      const int d = d0 + lane;
      int n = 0;
      if (d <= a.docs && (a.cu_q || d == 0)) {
        const Doc x = get_doc(a, d);
        n = (int)((x.q1 - x.q0 + TILES * kBM - 1) / (TILES * kBM));
      }
      int up = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += y;
      }
      const int at = (int)blockIdx.y - before - (up - n);
      const unsigned hit = __ballot_sync(0xffffffffu, at >= 0 && at < n);
      if (hit) {
        const int who = __ffs(hit) - 1;
        doc = d0 + who;
        tile = __shfl_sync(0xffffffffu, n - 1 - at, who);
      }
      before += __shfl_sync(0xffffffffu, up, 31);
    }
    if (lane == 0) {
      s_tile = tile;
      if (tile >= 0) s_doc = get_doc(a, doc);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_at, 0);
  const int pair = __shfl_sync(0xffffffffu, s_tile, 0);
  if (pair >= 0) {
    // through a shuffle: warp-uniform for the compiler, so that the matrix warp works in uniform registers
    Doc doc;
    doc.q0 = __shfl_sync(0xffffffffu, s_doc.q0, 0);
    doc.q1 = __shfl_sync(0xffffffffu, s_doc.q1, 0);
    doc.k0 = __shfl_sync(0xffffffffu, s_doc.k0, 0);
    doc.n = __shfl_sync(0xffffffffu, s_doc.n, 0);
    doc.shift = __shfl_sync(0xffffffffu, s_doc.shift, 0);
    doc.prefix = __shfl_sync(0xffffffffu, s_doc.prefix, 0);
    const int h = blockIdx.x, hk = h / a.group;
    const int64_t row0 = doc.q0 + (int64_t)pair * TILES * kBM;  // first query row of tile 0
    const int rows = (int)min((int64_t)TILES * kBM, doc.q1 - row0);
    const int key_tiles = (doc.n + kBN - 1) / kBN;
    // key tiles that some query of tile t sees: [lo, hi) of t, and those below `shared` (the prefix)
    const int shared = (doc.prefix + kBN - 1) / kBN;
    int from[2] = {key_tiles, key_tiles}, to[2] = {0, 0};
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const int n = min(kBM, rows - t * kBM), p = (int)(row0 - doc.q0) + t * kBM + doc.shift;
      const Sight first = sight_of(a, doc, p), last = sight_of(a, doc, p + n - 1);
      if (n > 0 && last.hi > first.lo) {
        from[t] = first.lo / kBN;
        to[t] = (last.hi + kBN - 1) / kBN;
      }
    }
    const int from_any = min(from[0], from[1]), to_any = max(to[0], to[1]);
    auto need = [&](int t, int j) {
      if (t >= TILES) return false;
      return (j < shared && rows > t * kBM) || (j >= (t ? from[1] : from[0]) && j < (t ? to[1] : to[0]));
    };
    auto next = [&](int j) {  // the next key tile that one of the two needs
      ++j;
      if (j >= shared && j < from_any) j = from_any;
      return j < shared || j < to_any ? j : key_tiles;
    };
    const int start = next(-1);
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (ok) ok = mbar_wait_bounded(bar, parity, kPolls);
      return ok;
    };

    auto wait_all = [&](uint32_t bar, uint32_t parity) {  // the same answer for the whole warp
      const bool arrived = mbar_wait_bounded(bar, parity, kPolls);
      // once a wait has run out, it stays so; through the vote, which keeps `ok` uniform for the compiler (a plain
      // conjunction: 77 tokens 7.7 us a call, 5.7 so)
      ok = __all_sync(0xffffffffu, arrived && ok);
      return ok;
    };

    // registers: 8 warps x 32 x 208 + 4 x 32 x 88 = 384 x 168, or 4 x 32 x 208 + 4 x 32 x 48 = 256 x 128, what the CTA
    // was launched with
    if (warp >= L::MATRIX) {
      if constexpr (TILES == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      else asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
      if (warp == L::COPY) {
        // ------------------------------------------------------------ copies
        if (lane == 0) {
          auto tile_in = [&](const CUtensorMap* map, int swap, int head, int64_t row, uint32_t dst, uint32_t bar) {
            mbar_arrive_expect_tx(bar, L::BYTES);
#pragma unroll
            for (int p = 0; p < L::PANELS; ++p)
              tma_load_3d(dst + p * L::PANEL, map, p * 64, swap ? (int)row : head, swap ? head : (int)row, bar);
          };
          int idx = 0;
          auto stage_in = [&](const CUtensorMap* map, int swap, int j) {
            const int s = idx % L::STAGES;
            if (!wait(kv_empty(s), ((idx / L::STAGES) & 1) ^ 1)) return;
            tile_in(map, swap, hk, doc.k0 + (int64_t)j * kBN, base + (TILES + s) * L::BYTES, kv_full(s));
            ++idx;
          };
          if (start < key_tiles) {
            tile_in(&maps.q, maps.q_swap, h, row0, base, q_full(0));
            stage_in(&maps.k, maps.k_swap, start);
            if (TILES == 2 && rows > kBM) tile_in(&maps.q, maps.q_swap, h, row0 + kBM, base + L::BYTES, q_full(1));
            for (int j = start; j < key_tiles && ok;) {
              stage_in(&maps.v, maps.v_swap, j);
              j = next(j);
              if (j < key_tiles) stage_in(&maps.k, maps.k_swap, j);
            }
          }
          // every copy has landed before the CTA's memory is given back
          if (start < key_tiles) {
            mbar_wait_bounded(q_full(0), 0, kLandPolls);
            if (TILES == 2 && rows > kBM) mbar_wait_bounded(q_full(1), 0, kLandPolls);
          }
          for (int i = idx > L::STAGES ? idx - L::STAGES : 0; i < idx; ++i)
            mbar_wait_bounded(kv_full(i % L::STAGES), (i / L::STAGES) & 1, kLandPolls);
        }
        __syncwarp();
      } else if (warp == L::MATRIX) {
        // ------------------------------------------------------------ matrix instructions
        if (start < key_tiles) {
          constexpr uint32_t qk = instr_desc(kBM, kBN, BF16, false), pv = instr_desc(kBM, DP, BF16, true);
          constexpr uint32_t hi = smem_desc_hi(1024);
          const bool one = elect_one();
          const uint32_t q_lo = smem_desc_lo(base, 16), k_lo = smem_desc_lo(base + TILES * L::BYTES, 16),
                         v_lo = smem_desc_lo(base + TILES * L::BYTES, L::PANEL);
          int done[2] = {0, 0};  // tiles whose P V has been issued
          auto scores = [&](int t, int stage) {
            if (one) {
              const uint32_t qa = q_lo + t * (L::BYTES >> 4), ka = k_lo + stage * (L::BYTES >> 4);
#pragma unroll
              for (int k = 0; k < DP / 16; ++k) {
                const uint32_t off = ((k / 4) * L::PANEL + (k % 4) * 32) >> 4;
                tc_mma_ss(tmem + t * 128, qa + off, ka + off, hi, qk, k > 0);
              }
              tc_commit(s_full(t));
            }
          };
          // P V, of the first 96 keys as soon as their P is there
          auto values = [&](int t, int stage) {
            const uint32_t va = v_lo + stage * (L::BYTES >> 4);
            if (!wait_all(p_most(t), done[t] & 1)) return;
            tc_fence_after();
            if (one) {
#pragma unroll
              for (int k = 0; k < 6; ++k)
                tc_mma_ts(tmem + L::OUT + t * 128, tmem + t * 128 + k * 8, va + ((k * 2048) >> 4), hi, pv,
                          done[t] > 0 || k > 0);
            }
            if (!wait_all(p_full(t), done[t] & 1)) return;
            tc_fence_after();
            if (one) {
#pragma unroll
              for (int k = 6; k < 8; ++k)
                tc_mma_ts(tmem + L::OUT + t * 128, tmem + t * 128 + k * 8, va + ((k * 2048) >> 4), hi, pv, true);
              tc_commit(o_full(t));
            }
            ++done[t];
          };
          auto free_stage = [&](int stage) {
            if (one) tc_commit(kv_empty(stage));
          };
          wait_all(kv_full(0), 0);
#pragma unroll
          for (int t = 0; t < TILES; ++t)
            if (ok && rows > t * kBM && wait_all(q_full(t), 0) && need(t, start)) scores(t, 0);
          free_stage(0);
          // A wait, even for a barrier that has completed, takes some 200 cycles next to operands that stream from
          // shared memory: those for copies are made one tile ahead, while the unit is busy.
          int last = -1, sv = 1, sk = 2;  // stage of the last V; of V(j), of K(next j)
          uint32_t ring = 1u;             // bit s: the phase of stage s that completes next
          auto arrive = [&](int s) {
            wait_all(kv_full(s), ring >> s & 1);
            ring ^= 1u << s;
          };
          int jn = next(start);
          arrive(sv);
          if (jn < key_tiles) arrive(sk);
          bool has[2] = {need(0, start), need(1, start)};
          for (int j = start; j < key_tiles && ok;) {
            const bool more = jn < key_tiles;
            const int jm = more ? next(jn) : key_tiles;
            const int mv = sk + 1 == L::STAGES ? 0 : sk + 1, mk = mv + 1 == L::STAGES ? 0 : mv + 1;
            const bool then[2] = {more && need(0, jn), more && need(1, jn)};
            if (ok && has[0]) values(0, sv);
            if (ok && then[0]) scores(0, sk);
            if (more) arrive(mv);
            if (jm < key_tiles) arrive(mk);
            if (ok && has[1]) values(1, sv);
            free_stage(sv);
            if (ok && then[1]) scores(1, sk);
            if (more) free_stage(sk);
            last = sv;
            sv = mv;
            sk = mk;
            has[0] = then[0];
            has[1] = then[1];
            j = jn;
            jn = jm;
          }
          // the last arrival that the matrix unit owes a barrier of this CTA: of the phase that V filled
          if (ok && last >= 0) wait_all(kv_empty(last), (ring >> last & 1) ^ 1);
          if (!ok) {  // no product may outlive the CTA's shared and tensor memory
            if (one) tc_commit(stopped);
            mbar_wait_bounded(stopped, 0, kLandPolls);
          }
        }
        __syncwarp();
      }
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
      // ------------------------------------------------------------ softmax: a thread per query row
      const int t = warp >> 2, r = t * kBM + (warp & 3) * 32 + lane;  // row of the pair
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t s_at = tmem + lanes + t * 128, o_at = tmem + lanes + L::OUT + t * 128;
      const bool active = rows > t * kBM;
      if (active) {
        const bool mine = r < rows;
        const int p = (int)(row0 - doc.q0) + r + doc.shift;
        const Sight see = sight_of(a, doc, p);
        const float slope = a.slopes ? a.slopes[h] : 0.f, slope2 = slope * kLog2e;
        // GENERAL: scores become log2 units at once; else they stay products and c is applied in the exponent
        const float c = GENERAL ? 1.f : a.scale * kLog2e;
        const float inv_cap = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
        float m = -INFINITY, l = 0.f;
        float le = 0.f;  // LSE: the sum of the weights before rounding
        float odd = 0.f;  // becomes NaN if a score or a result is not finite
        int done = 0;
        for (int j = next(-1); j < key_tiles; j = next(j)) {
          if (!need(t, j)) continue;
          if (!wait_all(s_full(t), done & 1)) break;
          tc_fence_after();
          uint32_t u[128];
          float* s = reinterpret_cast<float*>(u);
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_ld32(s_at + i * 32, u + i * 32);
          tmem_wait_ld();
          const int k0 = j * kBN;
          float offset = 0.f;  // what the scores of this tile lack, the same for all of them
          if constexpr (GENERAL) {
            if (a.softcap > 0.f) {
              cap_scores(s, inv_cap, a.softcap * kLog2e);
            } else {
#pragma unroll
              for (int i = 0; i < 128; i += 2) {
                const float2 v = mul2(float2{s[i], s[i + 1]}, both(a.scale * kLog2e));
                s[i] = v.x;
                s[i + 1] = v.y;
              }
            }
            if (a.slopes) {
              if (__all_sync(0xffffffffu, p >= k0 + kBN - 1)) {  // no key after the query: the bias is linear
                offset = -slope2 * (float)(p - k0);
#pragma unroll
                for (int i = 0; i < 128; i += 2) {
                  const float2 v = fma2(float2{(float)i, (float)(i + 1)}, both(slope2), float2{s[i], s[i + 1]});
                  s[i] = v.x;
                  s[i + 1] = v.y;
                }
              } else {
                const float d0 = (float)(p - k0);
#pragma unroll
                for (int i = 0; i < 128; ++i) s[i] = fmaf(-slope2, fabsf(d0 - (float)i), s[i]);
              }
            }
          }
          // the mask, where it cuts this tile for some row of the warp: the upper end, then what lies between the
          // prefix and the lower end
          const bool whole = k0 + kBN <= doc.prefix || (k0 >= see.lo && k0 + kBN <= see.hi);
          if (!__all_sync(0xffffffffu, whole)) {
            const int pre = doc.prefix - k0, hi = max(see.hi - k0, pre), lo = see.lo - k0;
            if (__any_sync(0xffffffffu, hi < kBN)) {
#pragma unroll
              for (int i = 0; i < 128; ++i) s[i] = i < hi ? s[i] : -INFINITY;
            }
            if (__any_sync(0xffffffffu, lo > max(pre, 0))) {
#pragma unroll
              for (int i = 0; i < 128; ++i) s[i] = i >= lo || i < pre ? s[i] : -INFINITY;
            }
          }
          float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int i = 4; i + 1 < 128; i += 2) top[(i >> 1) & 3] = max3(top[(i >> 1) & 3], s[i], s[i + 1]);
          const float mt = max3(max3(top[0], top[1], top[2]), top[3], top[3]) + offset;
          odd = mt != mt ? NAN : odd;
          // the maximum moves when it has grown by 2^8: sums are in float32 and p stays below 2^8
          const bool grow = (mt - m) * c > 8.f;
          if (__any_sync(0xffffffffu, grow)) {
            const float m_new = grow ? mt : m;
            const float back = grow ? (m == -INFINITY ? 0.f : ex2((m - m_new) * c)) : 1.f;
            m = m_new;
            l *= back;
            if (LSE) le *= back;
            if (done > 0) {
              if (!wait_all(o_full(t), (done - 1) & 1)) break;
              tc_fence_after();
#pragma unroll
              for (int i = 0; i < DP / 32; ++i) {
                uint32_t o[32];
                tmem_ld32(o_at + i * 32, o);
                tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * back);
                tmem_st32(o_at + i * 32, o);
              }
              tmem_wait_st();
            }
          }
          const float mc = m == -INFINITY ? 0.f : m * c;
          const float2 c2 = both(c), mc2 = both(offset - mc);
          float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}}, exact = {0.f, 0.f};
          // 32 keys at a time: P goes out while the next are computed
          auto weigh = [&](int x) {
            uint32_t q[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float2 e = fma2(float2{s[x * 32 + 2 * i], s[x * 32 + 2 * i + 1]}, c2, mc2);
              e.x = ex2(e.x);
              e.y = ex2(e.y);
              q[i] = pack16<BF16>(e.x, e.y);
              // the sum is that of the rounded weights, the ones that the values get: a row with one large weight
              // loses nothing
              if (LSE) exact = add2(exact, e);
              sum[i & 1] = add16<BF16>(sum[i & 1], q[i]);
            }
            tmem_st16(s_at + x * 16, q);
          };
          auto hand_over = [&](uint32_t bar) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
          };
#pragma unroll
          for (int x = 0; x < 3; ++x) weigh(x);
          hand_over(p_most(t));
          weigh(3);
          hand_over(p_full(t));
          sum[0] = add2(sum[0], sum[1]);
          l += sum[0].x + sum[0].y;
          if (LSE) le += exact.x + exact.y;
          ++done;
        }
        // ---------------------------------------------------------- output
        if (ok && done > 0) wait_all(o_full(t), (done - 1) & 1);
        tc_fence_after();
        if (ok) {
          // no weight at all: 0 where nothing is visible; where every visible score is -inf the definition decides
          if (l == 0.f && (see.hi > see.lo || doc.prefix > 0)) odd = NAN;
          const float inv = l == 0.f ? 0.f : 1.f / l;
          T* out = static_cast<T*>(a.out) + (row0 + r) * a.out_tok_stride + (int64_t)h * a.out_head_stride;
#pragma unroll
          for (int i = 0; i < DP / 32; ++i) {
            uint32_t o[32];
            if (done > 0) {
              tmem_ld32(o_at + i * 32, o);
              tmem_wait_ld();
            }
            if (l == 0.f) {
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] = 0;
            }
#pragma unroll
            for (int x = 0; x < 32; x += 8) {
              Vec<T, 8> v;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float y = __uint_as_float(o[x + e]) * inv;
                odd = fmaf(y, 0.f, odd);
                v.e[e] = from_f32<T>(y);
              }
              const int d = i * 32 + x;
              if (mine && d < a.head_dim) *reinterpret_cast<Vec<T, 8>*>(out + d) = v;
            }
          }
          if (LSE && mine)
            a.lse[(row0 + r) * a.lse_tok_stride + h] =
                l == 0.f ? -INFINITY : ((m == -INFINITY ? 0.f : m * c) + log2f(le)) * kLn2;
          // rows that are not finite, again from the definition (their tile of Q is no longer needed)
          unsigned again = __ballot_sync(0xffffffffu, mine && !(odd == 0.f));
          float* qs = reinterpret_cast<float*>(raw + (base - smem_u32(raw)) + t * L::BYTES + (warp & 3) * 1024);
          while (again) {
            const int who = __ffs(again) - 1;
            again &= again - 1;
            const int64_t row = row0 + t * kBM + (warp & 3) * 32 + who;
            const int pw = __shfl_sync(0xffffffffu, p, who);
            const Sight sw = sight_of(a, doc, pw);
            const T* q = static_cast<const T*>(a.q) + row * a.q_tok_stride + (int64_t)h * a.q_head_stride;
            __syncwarp();
            for (int d = lane; d < a.head_dim; d += 32) qs[d] = to_f32(q[d]);
            __syncwarp();
            const T* k = static_cast<const T*>(a.k) + doc.k0 * a.k_tok_stride + (int64_t)hk * a.k_head_stride;
            const T* v = static_cast<const T*>(a.v) + doc.k0 * a.v_tok_stride + (int64_t)hk * a.v_head_stride;
            T* o = static_cast<T*>(a.out) + row * a.out_tok_stride + (int64_t)h * a.out_head_stride;
            const float lse = attend_row<T, 128, false, false>(
                qs, a.head_dim, RowScore{a.scale, a.softcap, -slope}, 1.f, 0, doc.n,
                [&](int x) { return !(x < doc.prefix || (x >= sw.lo && x < sw.hi)); },
                [&](int x) { return k + x * a.k_tok_stride; }, [&](int x) { return v + x * a.v_tok_stride; },
                [&](int x) { return fabsf((float)(pw - x)); }, [&](int d, float x) { o[d] = from_f32<T>(x); });
            if (LSE && lane == 0) a.lse[row * a.lse_tok_stride + h] = lse;
          }
        }
      }
    }
    if (!ok && lane == 0) raise_status(a.status, OC_STATUS_TIMEOUT);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == L::COPY) tmem_free(tmem, L::COLUMNS);
}

// ------------------------------------------------------------------ any type, any alignment
// One warp per (query row, head), every key read for that row alone: right for
// anything and slow, 8192 causal tokens, 32 / 8 heads of 128 in float32 take 149
// ms, where elementary operations on whole matrices take 43.
template <typename T, int DMAX, bool WIDE>
__global__ void __launch_bounds__(32) prompt_row_kernel(const __grid_constant__ oc_prompt_args a) {
  __shared__ float qs[kRowMaxDim];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, hk = h / a.group, lane = threadIdx.x;
  const T* q = static_cast<const T*>(a.q) + t * a.q_tok_stride + h * a.q_head_stride;
  for (int d = lane; d < a.head_dim; d += 32) qs[d] = to_f32(q[d]);
  __syncwarp();
  // the document of the row: binary search
  int lo = -1, hi = a.docs;
  if (!a.cu_q) lo = 0;
  else if (t >= a.cu_q[0]) {
    lo = 0;
    hi = a.docs + 1;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu_q[mid] <= t) lo = mid;
      else hi = mid;
    }
  }
  const Doc doc = get_doc(a, lo);
  const int p = (int)(t - doc.q0) + doc.shift;
  const Sight see = sight_of(a, doc, p);
  const T* k = static_cast<const T*>(a.k) + doc.k0 * a.k_tok_stride + hk * a.k_head_stride;
  const T* v = static_cast<const T*>(a.v) + doc.k0 * a.v_tok_stride + hk * a.v_head_stride;
  T* out = static_cast<T*>(a.out) + t * a.out_tok_stride + h * a.out_head_stride;
  const float lse = attend_row<T, DMAX, WIDE, false>(
      qs, a.head_dim, RowScore{a.scale, a.softcap, a.slopes ? -a.slopes[h] : 0.f}, 1.f, 0, doc.n,
      [&](int j) { return !(j < doc.prefix || (j >= see.lo && j < see.hi)); },
      [&](int j) { return k + j * a.k_tok_stride; }, [&](int j) { return v + j * a.v_tok_stride; },
      [&](int j) { return fabsf((float)(p - j)); }, [&](int d, float x) { out[d] = from_f32<T>(x); });
  if (a.lse && lane == 0) a.lse[t * a.lse_tok_stride + h] = lse;
}

template <typename T>
int launch_rows(const oc_prompt_args& a, void* stream) {
  auto wide = [&](const void* p, int64_t tok, int64_t head) {
    return aligned_to(p, 16) && tok * sizeof(T) % 16 == 0 && head * sizeof(T) % 16 == 0;
  };
  const bool w = a.head_dim * sizeof(T) % 16 == 0 && wide(a.k, a.k_tok_stride, a.k_head_stride);
  auto kernel = a.head_dim > 128 ? prompt_row_kernel<T, 256, false>
                : w              ? prompt_row_kernel<T, 128, true>
                                 : prompt_row_kernel<T, 128, false>;
  return launch_pdl(kernel, dim3((unsigned)a.tokens, (unsigned)(a.kv_heads * a.group)), 32, 0, stream, a);
}

// ------------------------------------------------------------------ host side
PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

// A (rows, heads, head_dim) tensor of 16-bit elements as boxes of 128 rows of 64 columns of one head.
bool encode(CUtensorMap* map, int& swap, const void* base, int dtype, int head_dim, int64_t rows, int heads,
            int64_t tok_stride, int64_t head_stride) {
  const auto enc = map_encoder();
  if (!enc || !aligned_to(base, 16) || rows < 1) return false;
  const int64_t row_bytes = (int64_t)head_dim * 2;
  int64_t size[2] = {heads, rows}, stride[2] = {head_stride * 2, tok_stride * 2};
  // dimensions by increasing stride; the stride of a single entry is free
  swap = size[0] == 1 || (size[1] > 1 && stride[1] < stride[0]);
  cuuint64_t dim[3] = {(cuuint64_t)head_dim}, bytes[2];
  cuuint32_t box[3] = {64}, step[3] = {1, 1, 1};
  int64_t nest = (row_bytes + 15) / 16 * 16;
  for (int i = 0; i < 2; ++i) {
    const int r = swap ? 1 - i : i;
    int64_t b = stride[r];
    if (size[r] == 1) b = nest;
    if (b < nest || b % 16) return false;
    dim[i + 1] = (cuuint64_t)size[r];
    bytes[i] = (cuuint64_t)b;
    box[i + 1] = r == 1 ? kBN : 1;
    nest = size[r] == 1 ? nest : b;
  }
  return enc(map, dtype == OC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
             const_cast<void*>(base), dim, bytes, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP, int TILES, bool GENERAL, bool LSE>
int launch_tiled(const oc_prompt_args& a, const Maps& maps, unsigned tiles, void* stream) {
  using L = Tile<DP, TILES>;
  auto kernel = prompt_kernel<T, DP, TILES, GENERAL, LSE>;
  static std::atomic<uint64_t> ready;
  if (!allow_smem(reinterpret_cast<const void*>(kernel), ready, L::SMEM)) return OC_ERR_CUDA;
  return launch_pdl(kernel, dim3((unsigned)(a.kv_heads * a.group), tiles), dim3(L::THREADS), L::SMEM, stream, a, maps);
}

template <typename T>
int launch(const oc_prompt_args& a, void* stream) {
  Maps maps;
  const int es_ok = a.head_dim % 8 == 0 && a.head_dim <= 128 && aligned_to(a.out, 16) && a.out_tok_stride % 8 == 0 &&
                    a.out_head_stride % 8 == 0;
  if (!es_ok ||
      !encode(&maps.q, maps.q_swap, a.q, a.dtype, a.head_dim, a.tokens, a.kv_heads * a.group, a.q_tok_stride,
              a.q_head_stride) ||
      !encode(&maps.k, maps.k_swap, a.k, a.dtype, a.head_dim, a.key_tokens, a.kv_heads, a.k_tok_stride,
              a.k_head_stride) ||
      !encode(&maps.v, maps.v_swap, a.v, a.dtype, a.head_dim, a.key_tokens, a.kv_heads, a.v_tok_stride,
              a.v_head_stride))
    return launch_rows<T>(a, stream);
  // Two query tiles a CTA share every copy of K and V; one a CTA, two CTAs an SM, begin and end apart and waste less at
  // the edges of documents and windows.  Up to 64 columns the second have room, and a document of some 4096 tokens, or
  // a window, is where they meet (32 heads of 64: a window of 512 in 8192 tokens 100 us by two, 88 by one; 16 heads,
  // 2048 tokens capped 49 and 45; 3001 tokens 61.4 and 60.3; 32 heads, 8192 tokens 380 and 390).
  const int64_t reach = a.cu_q && a.docs > 0 ? a.key_tokens / a.docs : a.key_tokens;
  const int per_cta = a.head_dim <= 64 && (reach <= 4096 || (a.window > 0 && a.window <= 4096)) ? 1 : 2;
  // groups of query tiles: the documents' lengths are on the device, so an upper bound; the rest leave at once
  const int64_t tiles = a.tokens / (per_cta * kBM) + (a.cu_q ? a.docs + 2 : 1);
  if (tiles > 65535) return OC_ERR_TOO_LARGE;
  // A few tokens: a warp per row is through sooner than a tile is set up, and many short documents would each take a
  // CTA for a part of its rows (31 tokens in 12 documents, 32 heads: 24 us by tiles, 5.5 by rows; 152 in 8: 15.5 and 41;
  // one prompt of 77: 6.3 by tiles).
  const int64_t heads = (int64_t)a.kv_heads * a.group;
  if (a.key_tokens <= 32 || (a.key_tokens <= 64 && tiles * heads > a.num_sms)) return launch_rows<T>(a, stream);
  const bool general = a.softcap > 0.f || a.slopes || !(a.scale > 0.f);
  auto by_lse = [&](auto dp, auto n, auto gen) {
    return a.lse ? launch_tiled<T, dp(), n(), gen(), true>(a, maps, (unsigned)tiles, stream)
                 : launch_tiled<T, dp(), n(), gen(), false>(a, maps, (unsigned)tiles, stream);
  };
  auto by_scores = [&](auto dp, auto n) {
    return general ? by_lse(dp, n, std::true_type()) : by_lse(dp, n, std::false_type());
  };
  using std::integral_constant;
  if (a.head_dim > 64) return by_scores(integral_constant<int, 128>(), integral_constant<int, 2>());
  return per_cta == 2 ? by_scores(integral_constant<int, 64>(), integral_constant<int, 2>())
                      : by_scores(integral_constant<int, 64>(), integral_constant<int, 1>());
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
  if (a.tokens > 0x7fffff00 || a.key_tokens > 0x7fffff00) return OC_ERR_TOO_LARGE;
  if (a.head_dim > kRowMaxDim) return OC_ERR_UNSUPPORTED;
  switch (a.dtype) {
    case OC_F32: return launch_rows<float>(a, stream);
    case OC_F16: return launch<__half>(a, stream);
    case OC_BF16: return launch<__nv_bfloat16>(a, stream);
    default: return OC_ERR_UNSUPPORTED;
  }
}
