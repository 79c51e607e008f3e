// Exact attention of one new token per sequence over its pages.
//
//   s_j = cap(scale q.k_j) + slope (j - (n - 1)),  o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m)
//
// Each key and value is read once and used for the query heads of its group
// only, so the kernel is bound by HBM; the tensor cores (mma.sync m16n8k16)
// keep the arithmetic out of the way at any group size.  Keys are the rows of
// the products: S^T = K Q^T (16 keys x 8 heads) and O^T = V^T P^T (16 columns
// x 8 heads), so a group of up to 8 heads fills a tile and P moves from the
// first product to the second in registers (one 8x8 transpose per 8 keys).
//
// Work is cut into tiles of 4 warps x KW keys.  All tiles of the batch form
// one sequence of which every CTA of one resident wave takes an equal run
// (lengths are read on the device, so ragged batches balance without the
// host); a unit (sequence, kv head, 16 heads) that is split over CTAs leaves
// partial states in the workspace, which a small dependent launch joins in a
// fixed order.  Each warp streams its own keys and values through a private
// ring of three 4 KB buffers (K, V, K, ...) that tiled TMA copies fill, a
// 128-byte-swizzled box per page and 128 bytes of columns, the page id looked
// up two tiles ahead: no CTA barrier until a unit ends, and 16 warps per SM to
// cover the latency of one another's products.  Values in slots that are not
// visible are zeroed in shared memory before use and their scores masked, so
// their contents have no effect.
//
// The weights are rounded to the products' 16 bits, since a matrix instruction
// takes both operands in one type; sums stay in float32, and the sum that
// normalises is that of the rounded weights.  Against 64 bits an output is then
// off by 0.0021 (bfloat16, 32768 tokens) where one rounding alone gives 0.0016.
//
// Measured on one B200, in a graph: 16 ragged sequences of up to 8191 tokens,
// 32 heads of 64 in float16, 98 us for 593 MB (6.0 TB/s, 0.92 of a copy); 64
// sequences of up to 8192, 8 heads of 128 in 8 bits, 99 us for 537 MB (5.4
// TB/s; conversions to 16 bits keep the issue slots 56% busy); one sequence of
// 32768 tokens, 8 heads of 128 in bfloat16, 32 us for 134 MB: 21 us of data at
// 6.4 TB/s, the rest is the chain length, page, first copy, and the join.  300
// tokens of one sequence: 6.1 us, that chain alone.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>
#include <utility>

#include "oc_attn_row.cuh"
#include "oc_ptx.cuh"

namespace {

using namespace oc;

constexpr int kWarps = 4;
constexpr int kBufs = 3;         // buffers of a warp's ring
constexpr int kMinShare = 2;     // tiles that a CTA takes at least before a unit is split
constexpr int kLongRun = 24;     // places per CTA from which runs have a finer tail
constexpr int kTailPart = 4;     // which is one kTailPart-th of all places
constexpr int kUnitCost = 3;     // what beginning and ending a unit costs, in tiles, when shares are equalised
constexpr int kDirectTiles = 8;  // units of at most so many tiles get a CTA each and no joining launch

// ------------------------------------------------------------------ tile shape
template <int ES, int DP, int NT>
struct Shape {
  static constexpr int ROW = DP * ES;                       // bytes of a row
  // 16-key groups of a warp tile: 4 KB of keys or more, and room for 8 heads' output
  static constexpr int KT = 16 * ROW < 4096 ? 4096 / (16 * ROW) : ES == 1 ? 2 : 1;
  static constexpr int KW = 16 * KT;                        // keys of a warp tile
  static constexpr int CT = kWarps * KW;                    // keys of a CTA tile
  static constexpr int BUF = KW * ROW;                      // bytes of a K (or V) tile, and of 8 heads' output at most
  static constexpr int PANEL = ROW < 128 ? ROW : 128;       // bytes of columns that one box brings
  static constexpr int PANELS = ROW / PANEL;
  static_assert(PANEL == 128 || PANEL == 64, "one of the copy engine's swizzles");
  static constexpr int SMEM = kWarps * kBufs * BUF + 1024;  // + alignment of the swizzle pattern
  static constexpr int PER_SM = DP == 256 || NT == 2 ? 2 : 4;  // resident CTAs, by registers (and shared memory)
  static_assert(BUF >= 8 * DP * 4, "a buffer holds 8 heads' partial output");
  // Byte offset of 16-byte chunk ch of row r: panels of KW rows.  The swizzle is as wide as a panel: with a
  // wider one the copy engine pads every row to the swizzle's width.
  static __device__ __forceinline__ uint32_t at(int r, int ch) {
    constexpr int PC = PANEL / 16;
    const uint32_t lin = (uint32_t)(r * PANEL + (ch % PC) * 16);
    return (uint32_t)(ch / PC) * (KW * PANEL) + (lin ^ ((lin >> 3) & (PANEL == 128 ? 0x70 : 0x30)));
  }
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 - 2 / (1 + e^2x): absolute error some 1e-7
__device__ __forceinline__ float tanh_of(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + ex2(x * (2.f * kLog2e))));
  return fmaf(-2.f, y, 1.f);
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
// Two 8-bit values (the low half of `two`) as two float16.
__device__ __forceinline__ uint32_t fp8x2_to_half2(uint32_t two) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(h) : "r"(two));
  return h;
}
__device__ __forceinline__ uint32_t fp8x2_to_half2_hi(uint32_t two) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(h) : "r"(two));
  return h;
}

// Visible keys [lo, n) of a sequence; its tiles start at base, a multiple of KW.
struct Span {
  int lo, n;
};
__device__ __forceinline__ Span span_of(const oc_paged_decode_args& a, int seq) {
  int n = a.seq_lens[seq];
  const int64_t room = (int64_t)a.max_blocks * a.block_size;
  if (n < 0 || n > room) {
    raise_status(a.status, OC_STATUS_POSITION);
    n = n < 0 ? 0 : (int)room;
  }
  return Span{a.window > 0 && n > a.window ? n - a.window : 0, n};
}
template <typename S>
__device__ __forceinline__ int tiles_of(Span s) {
  const int t = (s.n - (s.lo & -S::KW) + S::CT - 1) / S::CT;
  return t < 1 ? 1 : t;  // an empty sequence still has an output to write
}

// Exclusive prefix sum over the CTA's kWarps * 32 threads.
__device__ __forceinline__ int scan128(int v, int& total, int* part) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) part[w] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    before += i < w ? part[i] : 0;
    total += part[i];
  }
  return before + x - v;
}

// Walks the tiles of the batch in order: sequence, then unit, then tile.  `at`
// is the tile's place when each unit takes its tiles and kUnitCost.
template <typename S>
struct Walk {
  int seq, sub, tile, tiles, at;
  Span span;
  __device__ __forceinline__ void enter(const oc_paged_decode_args& a) {
    span = span_of(a, seq);
    tiles = tiles_of<S>(span);
  }
  __device__ __forceinline__ void next_unit(const oc_paged_decode_args& a, int subs) {
    tile = 0;
    if (++sub < subs) return;
    sub = 0;
    if (++seq < a.num_seqs) enter(a);
  }
  __device__ __forceinline__ void next(const oc_paged_decode_args& a, int subs) {
    ++at;
    if (++tile < tiles) return;
    at += kUnitCost;
    next_unit(a, subs);
  }
};

// How the places [0, total) are cut into runs, one per CTA.  The first `wave`
// CTAs, those that are resident from the start, take equal runs.  SMs do not
// stream equally fast (on this part some take 15% longer than the mean), so
// where runs are long the last quarter of all places is cut finer and left to
// `late` CTAs that start as others leave (16 ragged sequences of fp16: 110 to
// 99 us).  Not with 8-bit caches, whose tiles are bound by their conversion,
// the same on every SM (64 x 8192: 98 us without, 103 with).
struct Runs {
  int wave, big, small;
  __device__ __forceinline__ Runs(int total, int wave, int late) : wave(wave) {
    const bool tail = late > 0 && total >= kLongRun * wave;
    big = tail ? (total - total / kTailPart) / wave : (total + wave - 1) / wave;
    big = big < kMinShare ? kMinShare : big;
    small = tail ? (total - big * wave + late - 1) / late : 1;
  }
  __device__ __forceinline__ int64_t start(int c) const {
    return c < wave ? (int64_t)c * big : (int64_t)wave * big + (int64_t)(c - wave) * small;
  }
  __device__ __forceinline__ int owner(int place) const {
    const int64_t first = (int64_t)wave * big;
    return place < first ? place / big : wave + (int)(place - first) / small;
  }
};

// Workspace: header (the place before each sequence, and after all), then per CTA two states of 8 NT heads.
struct Space {
  int32_t* before;  // num_seqs + 1
  float* states;
  __host__ __device__ static size_t header(int num_seqs) { return (((size_t)num_seqs + 1) * 4 + 15) / 16 * 16; }
  __host__ __device__ Space(void* p, int num_seqs)
      : before(static_cast<int32_t*>(p)), states(reinterpret_cast<float*>(static_cast<char*>(p) + header(num_seqs))) {}
};
// acc, then of each head the maximum, the sum of the rounded weights, the sum of the weights
__host__ __device__ constexpr int state_floats(int heads, int dp) { return heads * (dp + 4); }

// A cache as the copy engine sees it: dimension 0 is a row's columns, the
// others (slot, kv head, page) are ordered by their strides; role[i] says
// which of them (0, 1, 2) dimension i + 1 is.
struct Maps {
  CUtensorMap k, v;
  int k_role[3], v_role[3];
};

template <typename T, typename C, int DP, int NT, bool DIRECT>
__global__ void __launch_bounds__(kWarps * 32, Shape<sizeof(C), DP, NT>::PER_SM)
    decode_kernel(const __grid_constant__ oc_paged_decode_args a, const __grid_constant__ Maps maps, int late_ctas) {
  using S = Shape<sizeof(C), DP, NT>;
  constexpr bool F8 = sizeof(C) == 1;
  constexpr bool BF16 = !F8 && std::is_same<T, __nv_bfloat16>::value;  // 8-bit caches multiply in float16
  constexpr int HT = 8 * NT;
  constexpr int KS = DP / 16;  // steps of 16 columns
  extern __shared__ char raw[];
  __shared__ __align__(8) uint64_t bars[kWarps][kBufs];
  __shared__ int part[kWarps];
  __shared__ int found[3];  // sequence, unit, tile
  __shared__ float stat[kWarps][8][3];
  char* const ring = raw + (-smem_u32(raw) & 1023u);

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int gtiles = (a.group + HT - 1) / HT, subs = a.kv_heads * gtiles;
  const uint32_t my_ring = smem_u32(ring) + warp * kBufs * S::BUF, my_bar = smem_u32(bars[warp]);
  if (lane == 0) {
    for (int i = 0; i < kBufs; ++i) mbar_init(my_bar + 8 * i, 1);
    mbar_init_fence();
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
  }
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait();

  // ---------------------------------------------------------------- this CTA's run of tiles
  Walk<S> cs;
  int end;  // the run goes up to this place
  if constexpr (DIRECT) {
    cs.seq = blockIdx.x / subs;
    cs.sub = blockIdx.x - cs.seq * subs;
    cs.tile = 0;
    cs.at = 0;
    cs.enter(a);
    end = cs.tiles;
  } else {
    const Space ws(a.workspace, a.num_seqs);
    const int wave = (int)gridDim.x - late_ctas;
    if (a.num_seqs <= 32) {  // each warp for itself, without a barrier
      const Span sp = lane < a.num_seqs ? span_of(a, lane) : Span{0, 0};
      const int n = lane < a.num_seqs ? (tiles_of<S>(sp) + kUnitCost) * subs : 0;
      int up = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += y;
      }
      const int total = __shfl_sync(0xffffffffu, up, 31), at = up - n;
      const Runs runs(total, wave, late_ctas);
      const int64_t start = runs.start(blockIdx.x);
      if (blockIdx.x == 0 && warp == 0) {  // for the joining launch
        if (lane < a.num_seqs) ws.before[lane] = at;
        if (lane == 0) ws.before[a.num_seqs] = total;
      }
      if (start >= total) return;
      end = (int)min(runs.start(blockIdx.x + 1), (int64_t)total);
      const int who = __ffs(__ballot_sync(0xffffffffu, start >= at && start < up)) - 1;
      const int unit = __shfl_sync(0xffffffffu, n, who) / subs, off = (int)start - __shfl_sync(0xffffffffu, at, who);
      cs.seq = who;
      cs.sub = off / unit;
      cs.tile = off % unit;
      cs.at = (int)start;
      cs.span.lo = __shfl_sync(0xffffffffu, sp.lo, who);
      cs.span.n = __shfl_sync(0xffffffffu, sp.n, who);
      cs.tiles = unit - kUnitCost;
    } else {
      int mine = 0, own = 0;  // own: of sequence threadIdx.x
      for (int s = threadIdx.x; s < a.num_seqs; s += kWarps * 32) {
        const int n = (tiles_of<S>(span_of(a, s)) + kUnitCost) * subs;
        if (s == (int)threadIdx.x) own = n;
        mine += n;
      }
      int total;
      scan128(mine, total, part);
      const Runs runs(total, wave, late_ctas);
      const int64_t start = runs.start(blockIdx.x);
      if (start >= total && blockIdx.x != 0) return;
      end = (int)min(runs.start(blockIdx.x + 1), (int64_t)total);
      // the sequence that holds `start` (CTA 0 also leaves the prefix sums for the joining launch)
      int base = 0;
      for (int s0 = 0; s0 < a.num_seqs; s0 += kWarps * 32) {
        const int s = s0 + threadIdx.x;
        const int n = s >= a.num_seqs ? 0 : s0 == 0 ? own : (tiles_of<S>(span_of(a, s)) + kUnitCost) * subs;
        int sum;
        const int at = base + scan128(n, sum, part);
        if (s < a.num_seqs && start >= at && start < at + n) {
          const int unit = n / subs, off = (int)(start - at);
          found[0] = s;
          found[1] = off / unit;
          found[2] = off % unit;
        }
        if (blockIdx.x == 0 && s < a.num_seqs) ws.before[s] = at;
        base += sum;
        if (blockIdx.x != 0 && start < base) break;
      }
      if (blockIdx.x == 0 && threadIdx.x == 0) ws.before[a.num_seqs] = total;
      __syncthreads();
      cs.seq = found[0];
      cs.sub = found[1];
      cs.tile = found[2];
      cs.at = (int)start;
      cs.enter(a);
    }
    if (cs.tile >= cs.tiles) {  // in the cost of a unit that others have done
      cs.at += cs.tiles + kUnitCost - cs.tile;
      cs.next_unit(a, subs);
      if (cs.at >= end) return;
    }
  }

  // ---------------------------------------------------------------- the copy stream of this warp
  // A run is the part of a warp tile that lies in one page: KW keys, or a whole
  // page where pages are smaller.  Lane r copies run r.
  const int block_shift = __ffs(a.block_size) - 1;
  const int run_rows = a.block_size < S::KW ? a.block_size : S::KW, runs = S::KW / run_rows;
  Walk<S> ld = cs;
  static_assert(S::KW <= 32 || (S::KW == 64 && S::ROW == 64), "a lane per run: pages of one 64-byte row are not tiled");
  struct Source {
    bool on, run;        // there is such a tile; it has a run `lane` with visible keys
    int page, slot, hk;  // of that run
  };
  // the pages of the next tile, as the table has them: nothing waits for them here
  auto look = [&]() {
    Source p = {ld.at < end, false, 0, 0, 0};
    if (!p.on) return p;
    const int key0 = (ld.span.lo & -S::KW) + ld.tile * S::CT + warp * S::KW;
    p.hk = ld.sub / gtiles;
    const int32_t* table = a.block_tables + (int64_t)ld.seq * a.block_table_stride;
    const int j = key0 + lane * run_rows;
    p.slot = key0 & (a.block_size - 1);  // 0 where a tile has several runs
    p.run = lane < runs && j < ld.span.n && j + run_rows > ld.span.lo;
    if (p.run) p.page = table[j >> block_shift];
    ld.next(a, subs);
    return p;
  };
  const uint64_t policy = policy_evict_first();
  auto copy_run = [&](const CUtensorMap* map, const int* role, const Source& p, int page, uint32_t buf, uint32_t bar) {
    auto coord = [&](int i) { return role[i] == 0 ? p.slot : role[i] == 1 ? p.hk : page; };
    const int c1 = coord(0), c2 = coord(1), c3 = coord(2);
    for (int x = 0; x < S::PANELS; ++x)  // columns from head_dim on arrive as zeros
      tma_load_4d(buf + x * (S::KW * S::PANEL) + lane * run_rows * S::PANEL, map, x * (S::PANEL / (int)sizeof(C)), c1, c2,
                  c3, bar, policy);
  };
  // fills buffer b with K (or V) of a tile
  auto issue = [&](const CUtensorMap* map, const int* role, const Source& p, int b) {
    const uint32_t buf = my_ring + b * S::BUF, bar = my_bar + 8 * b;
    const int n = __popc(__ballot_sync(0xffffffffu, p.run));
    if (lane == 0) mbar_arrive_expect_tx(bar, n * S::PANELS * run_rows * S::PANEL);
    __syncwarp();
    if (p.run) {
      int page = p.page;
      if (page < 0 || page >= a.num_blocks) {  // a coordinate outside the cache: the copy engine delivers zeros
        raise_status(a.status, OC_STATUS_BAD_PAGE);
        page = -1;
      }
      copy_run(map, role, p, page, buf, bar);
    }
  };
  // The unit's queries: head g, the columns of this lane's operand (8-bit keys come out of their conversion in
  // another order: 4t, 4t + 1 | 4t + 2, 4t + 3).  Loads without branches, of a head and column that exist, so that
  // all are on their way at once.
  Vec<T, 4> query[NT][KS];
  auto column = [&](int k, int e) { return k * 16 + (F8 ? 4 * t + e : 2 * t + (e & 1) + (e >> 1) * 8); };
  auto load_query = [&]() {
    const int first = (cs.sub % gtiles) * HT, heads = min(HT, a.group - first);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int hr = n * 8 + g;
      const T* q = static_cast<const T*>(a.q) + (int64_t)cs.seq * a.q_seq_stride +
                   (int64_t)(cs.sub / gtiles * a.group + first + (hr < heads ? hr : 0)) * a.q_head_stride;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) query[n][k].e[e] = q[column(k, e) < a.head_dim ? column(k, e) : 0];
    }
  };
  load_query();
  Source for_v, for_k;  // the tile whose values, and the one whose keys, are copied next
  {
    const Source s0 = look(), s1 = look();
    for_k = look();
    issue(&maps.k, maps.k_role, s0, 0);
    issue(&maps.v, maps.v_role, s0, 1);
    if (s1.on) issue(&maps.k, maps.k_role, s1, 2);
    for_v = s1;
  }
  uint32_t parity = 0;  // bit b: the phase of buffer b that completes next
  auto arrived = [&](int b) {  // the same answer for the whole warp
    const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(my_bar + 8 * b, parity >> b & 1, kPolls));
    parity ^= ok ? 1u << b : 0u;
    return ok;
  };

  // ---------------------------------------------------------------- the unit's state
  uint32_t qf[KS][NT][2];
  float acc[KS][NT][4], m[NT][2], sc[NT][2], slope[NT][2];
  // sums of the weights, by the products' own unit (a row of ones times P): of the weights as they were rounded, so
  // that a row with one large weight loses nothing; [0] and [1] are this lane's heads, summed over all keys of the warp
  float l[NT][4];
  float le[NT][2];  // and of the weights before rounding, over this lane's keys: what the logarithm is taken of
  const bool capped = a.softcap > 0.f, biased = a.slopes != nullptr;
  const float cap2 = a.softcap * kLog2e;

  auto begin_unit = [&]() {
    const int hk = cs.sub / gtiles, h0 = hk * a.group + (cs.sub % gtiles) * HT;
    const int heads = min(HT, a.group - (cs.sub % gtiles) * HT);
    float qscale[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int hr = n * 8 + g;
      float x[KS][4];
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[k][e] = hr < heads && column(k, e) < a.head_dim ? to_f32(query[n][k].e[e]) : 0.f;
      qscale[n] = 1.f;
      if constexpr (F8 && std::is_same<T, __nv_bfloat16>::value) {
        // bfloat16 queries go through float16 times a power of two that puts their largest below 2^8
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[k][e]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (top > 0.f && top < INFINITY) {
          int e = 7 - ilogbf(top);
          e = e > 120 ? 120 : e;
          qscale[n] = exp2f((float)e);
        }
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        qf[k][n][0] = pack16<BF16>(x[k][0] * qscale[n], x[k][1] * qscale[n]);
        qf[k][n][1] = pack16<BF16>(x[k][2] * qscale[n], x[k][3] * qscale[n]);
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int hr = n * 8 + 2 * t + c;
        const float qs = __shfl_sync(0xffffffffu, qscale[n], (2 * t + c) * 4);
        sc[n][c] = a.scale * a.k_scale / qs * (capped ? 1.f / a.softcap : kLog2e);
        slope[n][c] = biased && hr < heads ? a.slopes[h0 + hr] * kLog2e : 0.f;
        m[n][c] = -INFINITY;
        l[n][c] = l[n][c + 2] = le[n][c] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) acc[k][n][c] = acc[k][n][c + 2] = 0.f;
      }
  };

  // ---------------------------------------------------------------- one warp tile
  float s[S::KT][NT][4];
  // scores in log2 units, the mask, and the running maximum
  auto scores = [&](int b) {
    const uint32_t kd = my_ring + b * S::BUF;
    const int key0 = (cs.span.lo & -S::KW) + cs.tile * S::CT + warp * S::KW;
#pragma unroll
    for (int kt = 0; kt < S::KT; ++kt) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[kt][n][c] = 0.f;
      const int row = kt * 16 + (lane & 15);
      if constexpr (F8) {
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          uint32_t r[4];
          ldsm_x4(kd + S::at(row, k + (lane >> 4)), r);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t f[4] = {fp8x2_to_half2(r[2 * u]), fp8x2_to_half2(r[2 * u + 1]), fp8x2_to_half2_hi(r[2 * u]),
                                   fp8x2_to_half2_hi(r[2 * u + 1])};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<BF16>(s[kt][n], f, qf[k + u][n][0], qf[k + u][n][1]);
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t r[4];
          ldsm_x4(kd + S::at(row, 2 * k + (lane >> 4)), r);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<BF16>(s[kt][n], r, qf[k][n][0], qf[k][n][1]);
        }
      }
    }
#pragma unroll
    for (int kt = 0; kt < S::KT; ++kt)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[kt][n][c] *= sc[n][c & 1];
    if (capped) {
#pragma unroll
      for (int kt = 0; kt < S::KT; ++kt)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[kt][n][c] = cap2 * tanh_of(s[kt][n][c]);
    }
    if (biased) {
#pragma unroll
      for (int kt = 0; kt < S::KT; ++kt)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            s[kt][n][c] = fmaf(slope[n][c & 1], (float)(key0 + kt * 16 + g + (c >> 1) * 8 - (cs.span.n - 1)), s[kt][n][c]);
    }
    if (key0 < cs.span.lo || key0 + S::KW > cs.span.n) {
#pragma unroll
      for (int kt = 0; kt < S::KT; ++kt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int j = key0 + kt * 16 + g + (c >> 1) * 8;
          if (j < cs.span.lo || j >= cs.span.n)
#pragma unroll
            for (int n = 0; n < NT; ++n) s[kt][n][c] = -INFINITY;
        }
    }
    // The maximum moves only when a score exceeds it by 2^8 (sums stay in float32, p below 2^8 in 16
    // bits loses nothing): most tiles skip the reduction and the rescaling.
    bool grow = false;
    float top[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[n][c] = fmaxf(s[0][n][c], s[0][n][c + 2]);
#pragma unroll
        for (int kt = 1; kt < S::KT; ++kt) top[n][c] = fmaxf(top[n][c], fmaxf(s[kt][n][c], s[kt][n][c + 2]));
        grow |= top[n][c] > m[n][c] + 8.f;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = fmaxf(m[n][c], top[n][c]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
          const float back = m[n][c] == -INFINITY ? 0.f : exp2f(m[n][c] - x);
          m[n][c] = x;
          l[n][c] *= back;
          l[n][c + 2] *= back;
          le[n][c] *= back;
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            acc[k][n][c] *= back;
            acc[k][n][c + 2] *= back;
          }
        }
    }
  };
  // values that the mask hides become zeros: 0 times what a free slot holds need not be 0
  auto clear_hidden = [&](int b) {
    const int key0 = (cs.span.lo & -S::KW) + cs.tile * S::CT + warp * S::KW;
    if (key0 >= cs.span.lo && key0 + S::KW <= cs.span.n) return;
    char* vb = ring + (warp * kBufs + b) * S::BUF;
    for (int i = lane; i < S::KW * (S::ROW / 16); i += 32) {
      const int r = i / (S::ROW / 16), j = key0 + r;
      if (j < cs.span.lo || j >= cs.span.n) *reinterpret_cast<uint4*>(vb + S::at(r, i % (S::ROW / 16))) = uint4{0, 0, 0, 0};
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy into the buffer
    __syncwarp();
  };
  auto values = [&](int b) {
    const uint32_t vd = my_ring + b * S::BUF;
#pragma unroll
    for (int kt = 0; kt < S::KT; ++kt) {
      uint32_t p[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float e[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float mc = m[n][c & 1];
          e[c] = ex2(s[kt][n][c] - (mc == -INFINITY ? 0.f : mc));
          le[n][c & 1] += e[c];
        }
        p[n][0] = transpose8x8(pack16<BF16>(e[0], e[1]));
        p[n][1] = transpose8x8(pack16<BF16>(e[2], e[3]));
        constexpr uint32_t one = BF16 ? 0x3f803f80u : 0x3c003c00u;
        const uint32_t ones[4] = {one, one, one, one};
        mma16816<BF16>(l[n], ones, p[n][0], p[n][1]);
      }
      if constexpr (F8) {
        // matrices: keys 0-7 and 8-15 of one 16-column chunk, then of the next
        const int row = kt * 16 + (lane & 15);
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          uint32_t r[4];
          ldsm_x4_t(vd + S::at(row, k + (lane >> 4)), r);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            // bytes (key 2t: d, d + 1; key 2t + 1: d, d + 1) to (d: both keys; d + 1: both keys)
            const uint32_t r0 = __byte_perm(r[2 * u], 0, 0x3120), r1 = __byte_perm(r[2 * u + 1], 0, 0x3120);
            const uint32_t f[4] = {fp8x2_to_half2(r0), fp8x2_to_half2_hi(r0), fp8x2_to_half2(r1), fp8x2_to_half2_hi(r1)};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<BF16>(acc[k + u][n], f, p[n][0], p[n][1]);
          }
        }
      } else {
        const int row = kt * 16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t r[4];
          ldsm_x4_t(vd + S::at(row, 2 * k + ((lane >> 3) & 1)), r);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<BF16>(acc[k][n], r, p[n][0], p[n][1]);
        }
      }
    }
  };

  // ---------------------------------------------------------------- end of a unit (or of the CTA's part of it)
  // The warps' states meet in the buffers that each has just consumed, 8 heads at a time.
  auto end_unit = [&](int b, bool complete, int slot) {
    float* mine = reinterpret_cast<float*>(ring + (warp * kBufs + b) * S::BUF);
    const int hk = cs.sub / gtiles, h0 = hk * a.group + (cs.sub % gtiles) * HT;
    const int heads = min(HT, a.group - (cs.sub % gtiles) * HT);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (n * 8 >= heads) break;
      __syncthreads();  // every warp has left its buffer (and the round before) behind
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float exact = le[n][c];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) exact += __shfl_xor_sync(0xffffffffu, exact, o);
        const int hr = 2 * t + c;
        if (g == 0) {
          stat[warp][hr][0] = m[n][c];
          stat[warp][hr][1] = l[n][c];
          stat[warp][hr][2] = exact;
        }
#pragma unroll
        for (int k = 0; k < KS; ++k) {  // columns are XORed by the head so that the four lanes of a row spread over banks
          const int d0 = F8 ? k * 16 + 2 * g : k * 16 + g, d1 = F8 ? d0 + 1 : d0 + 8;
          mine[hr * DP + (d0 ^ (t << 3))] = acc[k][n][c];
          mine[hr * DP + (d1 ^ (t << 3))] = acc[k][n][c + 2];
        }
      }
      __syncthreads();
      // a warp per head
      for (int hr = warp; hr < min(8, heads - n * 8); hr += kWarps) {
        float top = -INFINITY, sum = 0.f, exact = 0.f, f[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stat[w][hr][0]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          // a maximum of -inf with a sum that is not 0 is a NaN score: it stays
          f[w] = stat[w][hr][0] == -INFINITY ? (stat[w][hr][1] == 0.f ? 0.f : 1.f) : exp2f(stat[w][hr][0] - top);
          sum = fmaf(stat[w][hr][1], f[w], sum);
          exact = fmaf(stat[w][hr][2], f[w], exact);
        }
        const int swz = ((hr >> 1) & 3) << 3, head = h0 + n * 8 + hr;
        // no weight at all: 0 where nothing is visible, NaN (0 / 0) where every visible score is -inf
        const float inv = sum == 0.f ? (cs.span.n > cs.span.lo ? NAN : 0.f) : a.v_scale / sum;
        float* state = nullptr;
        if constexpr (!DIRECT)
          state = Space(a.workspace, a.num_seqs).states + (int64_t)(2 * blockIdx.x + slot) * state_floats(HT, DP);
        T* out = static_cast<T*>(a.out) + (int64_t)cs.seq * a.out_seq_stride + (int64_t)head * a.out_head_stride;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          const int d = lane + 32 * i;
          float x = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w)
            x = fmaf(reinterpret_cast<const float*>(ring + (w * kBufs + b) * S::BUF)[hr * DP + (d ^ swz)], f[w], x);
          if (DIRECT || complete) {
            if (d < a.head_dim) out[d] = from_f32<T>(x * inv);
          } else {
            state[(n * 8 + hr) * DP + d] = x;
          }
        }
        if (lane == 0) {
          if (DIRECT || complete) {
            if (a.lse)
              a.lse[(int64_t)cs.seq * a.kv_heads * a.group + head] =
                  sum == 0.f ? -INFINITY : ((top == -INFINITY ? 0.f : top) + log2f(exact)) * kLn2;
          } else {
            float* totals = state + HT * DP + 4 * (n * 8 + hr);
            totals[0] = top;
            totals[1] = sum;
            totals[2] = exact;
          }
        }
      }
    }
    __syncthreads();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy into the buffer
    __syncwarp();
  };

  // ---------------------------------------------------------------- main loop
  begin_unit();
  bool from_start = cs.tile == 0;  // this CTA has the unit from its first tile
  int kb = 0;                      // buffer of the tile's keys; its values are in the next one
  unsigned owed = 0;               // a copy did not arrive within the bound: the buffers that copies are on their way to
  for (;;) {
    const int vb = kb + 1 == kBufs ? 0 : kb + 1;
    if (!arrived(kb)) {  // this tile's two, and the next tile's keys
      owed = for_v.on ? (1u << kBufs) - 1 : 1u << kb | 1u << vb;
      break;
    }
    scores(kb);
    __syncwarp();
    const bool more = for_v.on;
    if (more) issue(&maps.v, maps.v_role, for_v, kb);
    if (!arrived(vb)) {  // this tile's values, and the next tile's two
      owed = more ? (1u << kBufs) - 1 : 1u << vb;
      break;
    }
    clear_hidden(vb);
    values(vb);
    __syncwarp();
    const bool last_tile = cs.tile + 1 == cs.tiles;
    // a CTA leaves at most two partial states: of a unit begun by others, and of one that it began
    if (last_tile || !more) end_unit(vb, from_start && last_tile, from_start ? 1 : 0);
    if (!more) break;
    if (for_k.on) issue(&maps.k, maps.k_role, for_k, vb);
    for_v = for_k;
    for_k = look();
    kb = vb + 1 == kBufs ? 0 : vb + 1;
    cs.next(a, subs);
    if (cs.tile == 0) {
      load_query();
      begin_unit();
      from_start = true;
    }
  }
  if (owed) {  // report it, and let this warp's copies land before the CTA's memory is reused
    raise_status(a.status, OC_STATUS_TIMEOUT);
#pragma unroll 1
    for (int b = 0; b < kBufs; ++b)
      if (owed >> b & 1) mbar_wait_bounded(my_bar + 8 * b, parity >> b & 1, kLandPolls);
  }
}

// Joins the partial states of the units that were split: one CTA per
// (sequence, head); its warps take the parts in turn, and their states are
// joined in a fixed order.
template <typename T, int DP, int NT>
__global__ void __launch_bounds__(512) join_kernel(const __grid_constant__ oc_paged_decode_args a, int wave, int late_ctas) {
  constexpr int HT = 8 * NT, MOST = 16;
  const int W = blockDim.x >> 5;
  __shared__ float sm[MOST][3];
  __shared__ float so[MOST][DP];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gtiles = (a.group + HT - 1) / HT, subs = a.kv_heads * gtiles;
  const int h = blockIdx.x, seq = blockIdx.y, hk = h / a.group, hg = h - hk * a.group;
  const int sub = hk * gtiles + hg / HT, hr = hg % HT;
  const Space ws(a.workspace, a.num_seqs);
  const int before = ws.before[seq], tiles = (ws.before[seq + 1] - before) / subs - kUnitCost;
  const Runs runs(ws.before[a.num_seqs], wave, late_ctas);
  const int t0 = before + sub * (tiles + kUnitCost), c0 = runs.owner(t0), c1 = runs.owner(t0 + tiles - 1);
  if (c0 == c1) return;  // one CTA had it all and wrote the output
  auto state = [&](int c) {
    // the unit is the CTA's first unless it starts inside the CTA's run
    const int slot = t0 >= runs.start(c) ? 1 : 0;
    return ws.states + (int64_t)(2 * c + slot) * state_floats(HT, DP);
  };
  // each warp joins every W-th part by itself, then the warps' states are joined
  float top = -INFINITY, sum = 0.f, exact = 0.f, x[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) x[i] = 0.f;
  constexpr int U = 5;  // parts whose loads go out together
  for (int c = c0 + warp; c <= c1; c += U * W) {
    float mc[U], lc[U], le[U], v[U][DP / 32];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool on = c + u * W <= c1;
      const float* s = state(on ? c + u * W : c);
      mc[u] = s[HT * DP + 4 * hr];
      lc[u] = s[HT * DP + 4 * hr + 1];
      le[u] = s[HT * DP + 4 * hr + 2];
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) v[u][i] = s[hr * DP + lane + 32 * i];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c + u * W > c1) continue;
      // a maximum of -inf with a sum that is not 0 is a NaN score: it stays; and 0 times an infinite value is NaN
      const float m = fmaxf(top, mc[u]);
      const float back = top == -INFINITY ? 1.f : exp2f(top - m);
      const float f = mc[u] == -INFINITY ? (lc[u] == 0.f ? 0.f : 1.f) : exp2f(mc[u] - m);
      top = m;
      sum = fmaf(lc[u], f, sum * back);
      exact = fmaf(le[u], f, exact * back);
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) x[i] = fmaf(v[u][i], f, x[i] * back);
    }
  }
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) so[warp][lane + 32 * i] = x[i];
  if (lane == 0) {
    sm[warp][0] = top;
    sm[warp][1] = sum;
    sm[warp][2] = exact;
  }
  __syncthreads();
  top = -INFINITY;
  for (int w = 0; w < W; ++w) top = fmaxf(top, sm[w][0]);
  float all = 0.f, all_exact = 0.f, f[MOST];
#pragma unroll
  for (int w = 0; w < MOST; ++w) {
    f[w] = w >= W ? 0.f : sm[w][0] == -INFINITY ? (sm[w][1] == 0.f ? 0.f : 1.f) : exp2f(sm[w][0] - top);
    if (w < W) {
      all = fmaf(sm[w][1], f[w], all);
      all_exact = fmaf(sm[w][2], f[w], all_exact);
    }
  }
  const float inv = all == 0.f ? NAN : a.v_scale / all;  // a unit that is split sees some keys
  T* out = static_cast<T*>(a.out) + (int64_t)seq * a.out_seq_stride + (int64_t)h * a.out_head_stride;
  for (int d = threadIdx.x; d < a.head_dim; d += blockDim.x) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < MOST; ++w)
      if (w < W) y = fmaf(so[w][d], f[w], y);
    out[d] = from_f32<T>(y * inv);
  }
  if (a.lse && threadIdx.x == 0)
    a.lse[(int64_t)seq * a.kv_heads * a.group + h] =
        all == 0.f ? -INFINITY : ((top == -INFINITY ? 0.f : top) + log2f(all_exact)) * kLn2;
}

// ------------------------------------------------------------------ any type, any alignment
// One CTA per (sequence, query head): each warp attends to a stretch of the
// keys, and the warps' results are weighted by their sums.  Not split over CTAs,
// and every head reads its keys for itself: 16 ragged sequences of up to 8191
// tokens, 32 heads of 64 in float32 take 1.15 ms (0.18 are the bytes'), one of
// 32768 tokens, 32 / 8 heads of 128, 2.8 ms (0.04).
constexpr int kRowWarps = 8;

template <typename T, typename C>
__global__ void __launch_bounds__(kRowWarps * 32) decode_row_kernel(const __grid_constant__ oc_paged_decode_args a) {
  __shared__ float qs[kRowMaxDim];
  __shared__ float part[kRowWarps][kRowMaxDim];
  __shared__ float sums[kRowWarps];
  pdl_launch_dependents();
  pdl_wait();
  const int seq = blockIdx.y, h = blockIdx.x, hk = h / a.group, warp = threadIdx.x >> 5;
  const T* q = static_cast<const T*>(a.q) + seq * a.q_seq_stride + h * a.q_head_stride;
  for (int d = threadIdx.x; d < a.head_dim; d += blockDim.x) qs[d] = to_f32(q[d]);
  __syncthreads();
  const Span span = span_of(a, seq);
  const int32_t* table = a.block_tables + seq * a.block_table_stride;
  auto row = [&](const void* cache, int64_t bs, int64_t hs, int64_t ts, int j) -> const C* {
    const int64_t page = table[j / a.block_size];
    if (page < 0 || page >= a.num_blocks) {
      raise_status(a.status, OC_STATUS_BAD_PAGE);
      return nullptr;
    }
    return static_cast<const C*>(cache) + page * bs + hk * hs + (j % a.block_size) * ts;
  };
  const int each = ((span.n - span.lo + kRowWarps - 1) / kRowWarps + 31) & ~31;  // keys of a warp
  const int first = min(span.n, span.lo + warp * each), last = min(span.n, first + each);
  const float lse = attend_row<C, kRowMaxDim, false, true>(
      qs, a.head_dim, RowScore{a.scale * a.k_scale, a.softcap, a.slopes ? a.slopes[h] : 0.f}, a.v_scale, first, last,
      [](int) { return false; },
      [&](int j) { return row(a.k_cache, a.kc_block_stride, a.kc_head_stride, a.kc_tok_stride, j); },
      [&](int j) { return row(a.v_cache, a.vc_block_stride, a.vc_head_stride, a.vc_tok_stride, j); },
      [&](int j) { return (float)(j - (span.n - 1)); }, [&](int d, float x) { part[warp][d] = x; });
  if ((threadIdx.x & 31) == 0) sums[warp] = lse;
  __syncthreads();
  float top = -INFINITY, all = 0.f, f[kRowWarps];
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, sums[w]);
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) {
    f[w] = sums[w] == -INFINITY ? 0.f : exp2f((sums[w] - (top == -INFINITY ? 0.f : top)) * kLog2e);  // NaN stays
    all += f[w];
  }
  const float inv = all == 0.f ? (span.n > span.lo ? NAN : 0.f) : 1.f / all;
  T* out = static_cast<T*>(a.out) + seq * a.out_seq_stride + h * a.out_head_stride;
  for (int d = threadIdx.x; d < a.head_dim; d += blockDim.x) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) x = fmaf(part[w][d], f[w], x);
    out[d] = from_f32<T>(x * inv);
  }
  if (a.lse && threadIdx.x == 0)
    a.lse[(int64_t)seq * a.kv_heads * a.group + h] =
        all == 0.f ? -INFINITY : (top == -INFINITY ? 0.f : top) + log2f(all) * kLn2;
}

template <typename T, typename C>
int launch_rows(const oc_paged_decode_args& a, void* stream) {
  return launch_pdl(decode_row_kernel<T, C>, dim3((unsigned)(a.kv_heads * a.group), (unsigned)a.num_seqs),
                    kRowWarps * 32, 0, stream, a);
}

// ------------------------------------------------------------------ host side
int padded(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// Tiles by 16-byte copies: 16-bit inputs, rows and pages at multiples of 16 bytes.
bool tiled(const oc_paged_decode_args& a) {
  if (a.dtype == OC_F32 || a.max_blocks == 0) return false;
  const int es = type_bytes(a.cache_dtype);
  auto ok = [&](int64_t s) { return (s * es) % 16 == 0; };
  // a box of the copy engine lands on a multiple of 128 bytes
  if (padded(a.head_dim) * es * a.block_size < 128) return false;
  return a.head_dim * es % 16 == 0 && a.head_dim >= 16 && aligned_to(a.k_cache, 16) && aligned_to(a.v_cache, 16) &&
         ok(a.kc_block_stride) && ok(a.kc_head_stride) && ok(a.kc_tok_stride) && ok(a.vc_block_stride) &&
         ok(a.vc_head_stride) && ok(a.vc_tok_stride);
}

struct Plan {
  bool direct;
  int64_t grid, late;  // CTAs, and those of them that wait for others to leave
  int64_t places;      // of all units at their longest, where they are split: kernels count them in 32 bits
  int nt;
};

template <int ES, int DP, int NT>
void plan_nt(const oc_paged_decode_args& a, Plan& p) {
  using S = Shape<ES, DP, NT>;
  const int64_t gt = (a.group + 8 * NT - 1) / (8 * NT), units = a.num_seqs * (int64_t)a.kv_heads * gt;
  int64_t most = (int64_t)a.max_blocks * a.block_size;
  if (a.window > 0 && (int64_t)a.window + S::KW < most) most = (int64_t)a.window + S::KW;
  const int64_t tiles = (most + S::CT - 1) / S::CT, wave = (int64_t)a.num_sms * S::PER_SM;
  const int64_t useful = (units * (tiles + kUnitCost) + kMinShare - 1) / kMinShare;
  p.nt = NT;
  p.direct = tiles <= kDirectTiles;
  p.places = p.direct ? 0 : units * (tiles + kUnitCost);
  p.late = ES > 1 && !p.direct && units * (tiles + kUnitCost) >= kLongRun * wave ? wave : 0;
  p.grid = p.direct ? units : useful < wave ? useful : wave + p.late;
}
template <int ES, int DP>
Plan plan_of(const oc_paged_decode_args& a) {
  Plan p;
  // groups above 8 take two tiles of 8 heads at once, where the state fits the registers
  if constexpr (DP < 256) {
    if (a.group > 8) {
      plan_nt<ES, DP, 2>(a, p);
      return p;
    }
  }
  plan_nt<ES, DP, 1>(a, p);
  return p;
}

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

bool encode(CUtensorMap* map, int (&role)[3], const void* base, const oc_paged_decode_args& a, int64_t tok_stride,
            int64_t head_stride, int64_t block_stride, int panel_bytes, int rows) {
  const auto enc = map_encoder();
  if (!enc) return false;
  const int es = type_bytes(a.cache_dtype);
  const int64_t size[3] = {a.block_size, a.kv_heads, a.num_blocks}, stride[3] = {tok_stride, head_stride, block_stride};
  auto key = [&](int r) { return size[r] == 1 ? INT64_MAX : stride[r]; };  // the stride of a single entry is free
  for (int i = 0; i < 3; ++i) role[i] = i;
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (key(role[j]) < key(role[i])) std::swap(role[i], role[j]);
  cuuint64_t dim[4] = {(cuuint64_t)a.head_dim}, bytes[3];
  cuuint32_t box[4] = {(cuuint32_t)(panel_bytes / es)}, step[4] = {1, 1, 1, 1};
  int64_t nest = ((int64_t)a.head_dim * es + 15) / 16 * 16;
  for (int i = 0; i < 3; ++i) {
    const int64_t b = size[role[i]] == 1 ? nest : stride[role[i]] * es;
    if (b < nest && size[role[i]] > 1) return false;  // rows that overlap (broadcast caches)
    dim[i + 1] = (cuuint64_t)size[role[i]];
    bytes[i] = (cuuint64_t)b;
    box[i + 1] = role[i] == 0 ? rows : 1;
    nest = b;
  }
  const CUtensorMapDataType type = a.cache_dtype == OC_F8E4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : a.cache_dtype == OC_F16  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                              : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return enc(map, type, 4, const_cast<void*>(base), dim, bytes, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
             panel_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename F>
auto by_shape(const oc_paged_decode_args& a, F f) {
  const int dp = padded(a.head_dim);
  if (a.cache_dtype == OC_F8E4M3) {
    if (dp == 64) return f(std::integral_constant<int, 1>(), std::integral_constant<int, 64>());
    if (dp == 128) return f(std::integral_constant<int, 1>(), std::integral_constant<int, 128>());
    return f(std::integral_constant<int, 1>(), std::integral_constant<int, 256>());
  }
  if (dp == 64) return f(std::integral_constant<int, 2>(), std::integral_constant<int, 64>());
  if (dp == 128) return f(std::integral_constant<int, 2>(), std::integral_constant<int, 128>());
  return f(std::integral_constant<int, 2>(), std::integral_constant<int, 256>());
}

template <typename T, typename C, int DP, int NT>
int launch_tiled(const oc_paged_decode_args& a, const Plan& p, void* stream) {
  using S = Shape<sizeof(C), DP, NT>;
  Maps maps;
  const int rows = a.block_size < S::KW ? a.block_size : S::KW;
  if (!encode(&maps.k, maps.k_role, a.k_cache, a, a.kc_tok_stride, a.kc_head_stride, a.kc_block_stride, S::PANEL, rows) ||
      !encode(&maps.v, maps.v_role, a.v_cache, a, a.vc_tok_stride, a.vc_head_stride, a.vc_block_stride, S::PANEL, rows))
    return launch_rows<T, C>(a, stream);
  auto kernel = p.direct ? decode_kernel<T, C, DP, NT, true> : decode_kernel<T, C, DP, NT, false>;
  static std::atomic<uint64_t> ready[2];
  if (!allow_smem(reinterpret_cast<const void*>(kernel), ready[p.direct], S::SMEM)) return OC_ERR_CUDA;
  int rc = launch_pdl(kernel, dim3((unsigned)p.grid), dim3(kWarps * 32), S::SMEM, stream, a, maps, (int)p.late);
  if (rc != OC_OK || p.direct) return rc;
  // few outputs have many parts each, many outputs two or three
  const int64_t outputs = (int64_t)a.num_seqs * a.kv_heads * a.group;
  return launch_pdl(join_kernel<T, DP, NT>, dim3((unsigned)(a.kv_heads * a.group), (unsigned)a.num_seqs),
                    dim3(outputs <= a.num_sms ? 512 : 128), 0, stream, a, (int)(p.grid - p.late), (int)p.late);
}

template <typename T, typename C, int DP>
int launch_nt(const oc_paged_decode_args& a, void* stream) {
  const Plan p = plan_of<sizeof(C), DP>(a);
  if (p.grid > 0x7fffffff || p.places > 0x7fffffff) return OC_ERR_TOO_LARGE;
  if constexpr (DP < 256) {
    if (p.nt == 2) return launch_tiled<T, C, DP, 2>(a, p, stream);
  }
  return launch_tiled<T, C, DP, 1>(a, p, stream);
}

template <typename T, typename C>
int launch_type(const oc_paged_decode_args& a, void* stream) {
  switch (padded(a.head_dim)) {
    case 64: return launch_nt<T, C, 64>(a, stream);
    case 128: return launch_nt<T, C, 128>(a, stream);
    default: return launch_nt<T, C, 256>(a, stream);
  }
}

int invalid(const oc_paged_decode_args& a) {
  if (a.num_seqs < 0 || a.kv_heads < 1 || a.group < 1 || a.head_dim < 1 || a.block_size < 1 ||
      (a.block_size & (a.block_size - 1)) || a.max_blocks < 0 || a.window < 0 || a.num_sms < 1 || a.num_blocks < 0 ||
      !(a.softcap >= 0.f))
    return OC_ERR_INVALID;
  if (a.head_dim > kRowMaxDim) return OC_ERR_UNSUPPORTED;
  if (a.cache_dtype != a.dtype && a.cache_dtype != OC_F8E4M3) return OC_ERR_UNSUPPORTED;
  if (a.dtype != OC_F32 && a.dtype != OC_F16 && a.dtype != OC_BF16) return OC_ERR_UNSUPPORTED;
  if (a.num_seqs > 65535 || (int64_t)a.max_blocks * a.block_size > 0x7fffff00) return OC_ERR_TOO_LARGE;
  return OC_OK;
}

}  // namespace

extern "C" size_t oc_paged_decode_workspace_bytes(const oc_paged_decode_args* a) {
  if (!a || invalid(*a) != OC_OK || a->num_seqs == 0 || !tiled(*a)) return 0;
  return by_shape(*a, [&](auto es, auto dp) -> size_t {
    const Plan p = plan_of<es(), dp()>(*a);
    if (p.direct) return 0;
    return Space::header(a->num_seqs) + (size_t)p.grid * 2 * state_floats(8 * p.nt, dp()) * sizeof(float);
  });
}

extern "C" int oc_paged_decode_attention(const oc_paged_decode_args* args, void* stream) {
  if (!args) return OC_ERR_INVALID;
  const oc_paged_decode_args& a = *args;
  const int bad = invalid(a);
  if (bad != OC_OK) return bad;
  if (a.num_seqs == 0) return OC_OK;
  if (!a.q || !a.out || !a.seq_lens || (a.max_blocks && (!a.block_tables || !a.k_cache || !a.v_cache)))
    return OC_ERR_INVALID;
  const bool f8 = a.cache_dtype == OC_F8E4M3;
  if (tiled(a)) {
    const size_t need = oc_paged_decode_workspace_bytes(&a);
    if (need && (!a.workspace || !aligned_to(a.workspace, 16) || a.workspace_bytes < need)) return OC_ERR_WORKSPACE;
    if (a.dtype == OC_F16) return f8 ? launch_type<__half, fp8_t>(a, stream) : launch_type<__half, __half>(a, stream);
    return f8 ? launch_type<__nv_bfloat16, fp8_t>(a, stream) : launch_type<__nv_bfloat16, __nv_bfloat16>(a, stream);
  }
  switch (a.dtype) {
    case OC_F32: return f8 ? launch_rows<float, fp8_t>(a, stream) : launch_rows<float, float>(a, stream);
    case OC_F16: return f8 ? launch_rows<__half, fp8_t>(a, stream) : launch_rows<__half, __half>(a, stream);
    default:
      return f8 ? launch_rows<__nv_bfloat16, fp8_t>(a, stream) : launch_rows<__nv_bfloat16, __nv_bfloat16>(a, stream);
  }
}
