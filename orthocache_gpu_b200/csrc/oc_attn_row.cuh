// One query row of attention by one warp, from the definition: a lane per key
// for the scores, a lane per column for the values, the running maximum and
// sum of the softmax in float32.  A key that the mask hides is never read, so
// whatever its slot holds has no effect.  Used for float32 inputs and for the
// rows whose result in the tiled kernels is not finite.
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
// takes the normalised columns.  Returns the natural-log sum (-inf if empty).
template <typename T, typename Hidden, typename Key, typename Value, typename Bias, typename Out>
__device__ float attend_row(const float* q_row, int head_dim, RowScore sc, float v_scale, int first, int last,
                            Hidden hidden, Key key, Value value, Bias bias_of, Out out) {
  const int lane = threadIdx.x & 31;
  float acc[kRowMaxDim / 32];
#pragma unroll
  for (int i = 0; i < kRowMaxDim / 32; ++i) acc[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int j0 = first; j0 < last; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j < last && !hidden(j)) {
      const T* k = key(j);
      float x = 0.f;
      if (k)
        for (int d = 0; d < head_dim; ++d) x = fmaf(q_row[d], to_f32(k[d]), x);
      x *= sc.scale;
      if (sc.softcap > 0.f) x = sc.softcap * tanhf(x / sc.softcap);
      s = x + (sc.slope != 0.f ? sc.slope * bias_of(j) : 0.f);
    }
    float top = s;
    bool nan = s != s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float m_new = fmaxf(m, top);
    nan = __any_sync(0xffffffffu, nan);
    if (m_new == -INFINITY && !nan) continue;  // nothing visible yet (or scores of -inf, which weigh nothing)
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
    for (int i = 0; i < kRowMaxDim / 32; ++i) acc[i] *= back;
    for (int k = 0; k < 32; ++k) {
      const float pk = __shfl_sync(0xffffffffu, p, k);
      const float seen = __shfl_sync(0xffffffffu, s, k);
      if (seen == -INFINITY) continue;
      const T* v = value(j0 + k);
      if (!v) continue;
#pragma unroll
      for (int i = 0; i < kRowMaxDim / 32; ++i)
        if (lane + 32 * i < head_dim) acc[i] = fmaf(pk, to_f32(v[lane + 32 * i]), acc[i]);
    }
  }
  const float inv = l == 0.f ? 0.f : v_scale / l;
#pragma unroll
  for (int i = 0; i < kRowMaxDim / 32; ++i)
    if (lane + 32 * i < head_dim) out(lane + 32 * i, acc[i] * inv);
  return l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) + kLn2 * log2f(l);
}

}  // namespace oc
