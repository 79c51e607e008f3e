// One query row of attention by one warp, from the definition: a lane per key
// for the scores, a lane per column for the values, the running maximum and
// sum of the softmax in float32.  A key that the mask hides is never read, so
// whatever its slot holds has no effect.  Used for float32 inputs, for
// alignments that the copy engine does not take, for prompts of a few tokens,
// and for the rows whose result in the tiled kernels is not finite.
#pragma once

#include "oc_ops.cuh"

namespace oc {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kRowMaxDim = 256;

struct RowScore {
  float scale, softcap, slope;  // slope: of the distance bias
};

// q_row: head_dim floats (shared memory); keys [first, last); hidden(j): the
// mask within that range; key(j) / value(j): the row's address (null: not
// readable, counts as zeros); bias_of(j): what slope multiplies.  out(d, x)
// takes the normalised columns.  DMAX: head_dim at most; WIDE: rows of whole,
// aligned 16-byte vectors.  Returns the natural-log sum (-inf if empty).  A row
// without a visible key is 0, one whose visible scores are all -inf is NaN
// (0 / 0); with PART, for one stretch of a row's keys, both are the sum itself.
template <typename T, int DMAX, bool WIDE, bool PART, typename Hidden, typename Key, typename Value, typename Bias, typename Out>
__device__ float attend_row(const float* q_row, int head_dim, RowScore sc, float v_scale, int first, int last,
                            Hidden hidden, Key key, Value value, Bias bias_of, Out out) {
  constexpr int C = DMAX / 32;         // columns of a lane
  constexpr int U = DMAX > 128 ? 4 : 8;  // value rows on their way at once
  const int lane = threadIdx.x & 31;
  float acc[C];
#pragma unroll
  for (int i = 0; i < C; ++i) acc[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  bool some = false;  // a visible key
  for (int j0 = first; j0 < last; j0 += 32) {
    const int j = j0 + lane;
    const bool visible = j < last && !hidden(j);
    const unsigned seen = __ballot_sync(0xffffffffu, visible);
    if (!seen) continue;
    some = true;
    float s = -INFINITY;
    if (visible) {
      const T* k = key(j);
      float x = 0.f;
      if (k) {
        if constexpr (WIDE) {
          constexpr int N = 16 / sizeof(T);
#pragma unroll 4
          for (int d = 0; d < head_dim; d += N) {
            const Vec<T, N> v = *reinterpret_cast<const Vec<T, N>*>(k + d);
#pragma unroll
            for (int e = 0; e < N; ++e) x = fmaf(q_row[d + e], to_f32(v.e[e]), x);
          }
        } else {
          for (int d = 0; d < head_dim; ++d) x = fmaf(q_row[d], to_f32(k[d]), x);
        }
      }
      x *= sc.scale;
      if (sc.softcap > 0.f) x = sc.softcap * tanhf(x / sc.softcap);
      s = x + (sc.slope != 0.f ? sc.slope * bias_of(j) : 0.f);
    }
    float top = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float m_new = fmaxf(m, top);
    // fmaxf passes NaN over: a NaN score makes p, and through it the row, NaN
    const float shift = m_new == -INFINITY ? 0.f : m_new;
    const float p = s == -INFINITY ? 0.f : exp2f((s - shift) * kLog2e);
    const float back = m == -INFINITY ? 0.f : exp2f((m - shift) * kLog2e);
    float sum = p;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = l * back + sum;
    m = m_new;
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] *= back;
    for (int k0 = 0; k0 < 32; k0 += U) {
      if (!(seen >> k0 & ((1u << U) - 1))) continue;
      float v[U][C];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const T* row = seen >> (k0 + u) & 1 ? value(j0 + k0 + u) : nullptr;
#pragma unroll
        for (int i = 0; i < C; ++i) v[u][i] = row && lane + 32 * i < head_dim ? to_f32(row[lane + 32 * i]) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float pk = __shfl_sync(0xffffffffu, p, k0 + u);
#pragma unroll
        for (int i = 0; i < C; ++i)
          if (seen >> (k0 + u) & 1) acc[i] = fmaf(pk, v[u][i], acc[i]);
      }
    }
  }
  const float inv = l == 0.f ? (some && !PART ? NAN : 0.f) : v_scale / l;
#pragma unroll
  for (int i = 0; i < C; ++i)
    if (lane + 32 * i < head_dim) out(lane + 32 * i, acc[i] * inv);
  return l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) + kLn2 * log2f(l);
}

}  // namespace oc
