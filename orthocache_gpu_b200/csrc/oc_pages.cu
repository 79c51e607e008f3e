// Page bookkeeping of the paged cache, all on the device and without a host
// synchronisation: fork / free sequences, reserve (copy-on-write and growth),
// compact, and the copy of pages across the caches of every layer.
//
// The bookkeeping is integer work on a few tens of KB and bound by latency:
// one CTA (a cluster of CTAs for the fork, whose tables are larger) whose
// phases are separated by barriers, instead of a chain of launches.  Which
// page is handed out never depends on timing: the k-th request, by row and
// column, gets the k-th lowest free page, both by prefix sums.  Copies run in
// a dependent launch over all caches; they are bound by memory bandwidth.
//
// Measured on one B200, in a graph: 64 sequences of up to 900 tokens over 4096
// pages of 16, fork 3.5 us, reserve 3.2 us without a request; fork, reserve
// and the copies of 32 pages in each of 44 caches together 11.4 us, three
// launches that each wait for the one before.  Compaction of the same after
// half of the sequences have ended, over 44 caches of 8 KB pages: 101 us, of
// which the copies take 89 (6.2 TB/s, read and write).
#include <cooperative_groups.h>

#include "oc_ops.cuh"
#include "oc_ptx.cuh"

namespace {

using namespace oc;

constexpr int kMaxCaches = 128;  // pointers that travel in one launch's parameters
constexpr int kThreads = 1024;
constexpr int kShortList = 2048;  // pages handed out by a reserve call whose list stays in shared memory

struct Caches {
  char* base[kMaxCaches];
  int64_t stride[kMaxCaches];  // bytes from page to page
};

// ------------------------------------------------------------------ block scan
struct Two {
  int a, b;
};
// Exclusive prefix sums of two counts over the CTA; total returns their sums.
__device__ __forceinline__ Two block_scan(Two v, Two& total) {
  __shared__ long long part[33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long own = (long long)v.a << 32 | (unsigned)v.b;  // no sum reaches 2^31
  long long x = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // part may still be read by an earlier call
  if (lane == 31) part[w] = x;
  __syncthreads();
  if (w == 0) {
    const long long mine = lane < (int)(blockDim.x >> 5) ? part[lane] : 0;
    long long p = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, p, o);
      if (lane >= o) p += y;
    }
    part[lane] = p - mine;
    if (lane == 31) part[32] = p;
  }
  __syncthreads();
  total = Two{(int)(part[32] >> 32), (int)(part[32] & 0xffffffff)};
  const long long before = part[w] + x - own;
  return Two{(int)(before >> 32), (int)(before & 0xffffffff)};
}

__device__ __forceinline__ int pages_for(int tokens, int block_size) {  // 32-bit arithmetic, for any tokens >= 0
  return (int)(((unsigned)tokens + (unsigned)block_size - 1u) / (unsigned)block_size);
}

// Four counts from index i on; beyond n: `fill`.
__device__ __forceinline__ int4 four_at(const int32_t* p, int64_t i, int64_t n, int fill) {
  if (i + 4 <= n && (reinterpret_cast<uintptr_t>(p + i) & 15) == 0) return *reinterpret_cast<const int4*>(p + i);
  return int4{i < n ? p[i] : fill, i + 1 < n ? p[i + 1] : fill, i + 2 < n ? p[i + 2] : fill, i + 3 < n ? p[i + 3] : fill};
}

// ------------------------------------------------------------------ page copies
// The table of a compaction, renumbered by the launch that moves its pages.
struct Renumber {
  const int32_t *in, *to;
  int32_t* out;
  int64_t in_stride, out_stride, num_seqs, max_blocks;
};

__device__ __forceinline__ void renumber(const Renumber& table, int64_t num_pages, uint32_t* status) {
  const int64_t entries = table.num_seqs * table.max_blocks;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < entries; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = e / table.max_blocks, c = e - r * table.max_blocks;
    const int32_t p = table.in[r * table.in_stride + c];
    if (p >= num_pages) raise_status(status, OC_STATUS_BAD_PAGE);
    table.out[r * table.out_stride + c] = p < 0 || p >= num_pages ? -1 : table.to[p];
  }
}

// The copies of one launch: pairs come from arrays of n entries, or of *n_dev
// entries on the device.
struct Copies {
  const int32_t *src, *dst, *n_dev;
  int64_t n, page_bytes, num_pages;
  int num_caches;
};

// Pages through shared memory, by bulk copies in both directions: one lane of
// each warp keeps kStages pieces of up to 8 KB on their way, 192 KB an SM, and
// spends no registers on them.  A warp takes an equal run of the pieces.
constexpr int kCopyWarps = 6, kStages = 4, kPiece = 8192;

__global__ void __launch_bounds__(kCopyWarps * 32)
    copy_bulk_kernel(const __grid_constant__ Caches caches, const __grid_constant__ Copies job, Renumber table,
                     uint32_t* status) {
  extern __shared__ __align__(128) char ring[];
  __shared__ __align__(8) uint64_t bars[kCopyWarps][kStages];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t bar = smem_u32(bars[warp]), mine = smem_u32(ring) + warp * kStages * kPiece;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(bar + 8 * i, 1);
    mbar_init_fence();
  }
  pdl_launch_dependents();
  pdl_wait();
  if (table.out) renumber(table, job.num_pages, status);
  if (lane != 0) return;
  const int64_t n = job.n_dev ? *job.n_dev : job.n, per_page = (job.page_bytes + kPiece - 1) / kPiece;
  const int64_t total = n * job.num_caches * per_page, warps = (int64_t)gridDim.x * kCopyWarps;
  const int64_t me = (int64_t)blockIdx.x * kCopyWarps + warp;
  const int64_t begin = total * me / warps, end = total * (me + 1) / warps;
  if (begin >= end) return;
  // walks over (pair, cache, piece of the page)
  struct Walk {
    int64_t pair, piece, from, to;
    int cache;
  };
  auto enter = [&](Walk& w) {  // from -1: the pair is skipped
    w.from = job.src[w.pair];
    w.to = job.dst[w.pair];
    if (w.from >= job.num_pages || w.to >= job.num_pages) {
      raise_status(status, OC_STATUS_BAD_PAGE);
      w.from = -1;
    }
    if (w.to < 0) w.from = -1;
  };
  auto next = [&](Walk& w, int64_t at) {  // to piece `at` of all
    if (++w.piece < per_page) return;
    w.piece = 0;
    if (++w.cache < job.num_caches) return;
    w.cache = 0;
    ++w.pair;
    if (at < end) enter(w);
  };
  Walk ld;
  ld.pair = begin / (per_page * job.num_caches);
  const int64_t rest = begin - ld.pair * per_page * job.num_caches;
  ld.cache = (int)(rest / per_page);
  ld.piece = rest - ld.cache * per_page;
  enter(ld);
  Walk st = ld;
  auto bytes_of = [&](const Walk& w) { return (uint32_t)min((int64_t)kPiece, job.page_bytes - w.piece * kPiece); };
  auto load = [&](int64_t at) {
    if (at >= end) return;
    const int s = (int)((at - begin) % kStages);
    if (ld.from >= 0) {
      mbar_arrive_expect_tx(bar + 8 * s, bytes_of(ld));
      bulk_load(mine + s * kPiece, caches.base[ld.cache] + ld.from * caches.stride[ld.cache] + ld.piece * kPiece,
                bytes_of(ld), bar + 8 * s);
    } else {
      mbar_arrive_expect_tx(bar + 8 * s, 0);
    }
    next(ld, at + 1);
  };
  for (int i = 0; i < kStages - 1; ++i) load(begin + i);
  bool late = false;
  int64_t at = begin;
  for (; at < end; ++at) {
    const int s = (int)((at - begin) % kStages);
    late = !mbar_wait_bounded(bar + 8 * s, (uint32_t)((at - begin) / kStages) & 1, kPolls);
    if (late) break;
    if (st.from >= 0)
      bulk_store(caches.base[st.cache] + st.to * caches.stride[st.cache] + st.piece * kPiece, mine + s * kPiece,
                 bytes_of(st));
    bulk_commit();
    bulk_wait_read<1>();  // the piece before this one has left its buffer
    load(at + kStages - 1);
    next(st, at + 1);
  }
  if (late) {  // report it, and let the other copies land before the CTA's memory is reused
    raise_status(status, OC_STATUS_TIMEOUT);
    for (int64_t i = at; i < end && i < at + kStages - 1; ++i)
      mbar_wait_bounded(bar + 8 * (uint32_t)((i - begin) % kStages), (uint32_t)((i - begin) / kStages) & 1, kLandPolls);
  }
  bulk_wait<0>();
}

// Any size and alignment: a warp moves 128 bytes of one page at a time.
__global__ void __launch_bounds__(256)
    copy_bytes_kernel(const __grid_constant__ Caches caches, const __grid_constant__ Copies job, Renumber table,
                      uint32_t* status) {
  pdl_launch_dependents();
  pdl_wait();
  if (table.out) renumber(table, job.num_pages, status);
  const int lane = threadIdx.x & 31;
  const int64_t n = job.n_dev ? *job.n_dev : job.n, per_page = (job.page_bytes + 127) / 128;
  const int64_t units = n * job.num_caches * per_page;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (int64_t)gridDim.x * 8) {
    const int64_t pc = u / per_page, pair = pc / job.num_caches;
    const int c = (int)(pc - pair * job.num_caches);
    const int64_t s = job.src[pair], d = job.dst[pair];
    if (s < 0 || d < 0) continue;
    if (s >= job.num_pages || d >= job.num_pages) {
      if (lane == 0) raise_status(status, OC_STATUS_BAD_PAGE);
      continue;
    }
    for (int64_t i = (u - pc * per_page) * 128 + lane; i < min((u - pc * per_page + 1) * 128, job.page_bytes); i += 32)
      caches.base[c][d * caches.stride[c] + i] = caches.base[c][s * caches.stride[c] + i];
  }
}

// Copies over every cache; at most `most` pairs.
int copy_all(void* const* caches, const int64_t* strides, int num_caches, int64_t page_bytes, int64_t num_pages,
             const int32_t* src, const int32_t* dst, int64_t most, const int32_t* n_dev, Renumber table,
             uint32_t* status, int num_sms, void* stream) {
  for (int first = 0; first < num_caches || table.out; first += kMaxCaches) {
    const int m = num_caches - first < kMaxCaches ? num_caches - first : kMaxCaches;
    Caches c;
    bool vec = page_bytes % 16 == 0;
    for (int i = 0; i < m; ++i) {
      c.base[i] = static_cast<char*>(caches[first + i]);
      c.stride[i] = strides[first + i];
      vec = vec && aligned_to(c.base[i], 16) && c.stride[i] % 16 == 0;
    }
    const Copies job = {src, dst, n_dev, most, page_bytes, num_pages, m};
    constexpr int smem = kCopyWarps * kStages * kPiece;
    int rc;
    if (vec) {
      const int64_t pieces = most * m * ((page_bytes + kPiece - 1) / kPiece), entries = table.num_seqs * table.max_blocks;
      int64_t ctas = (pieces + kCopyWarps - 1) / kCopyWarps;
      if (table.out && ctas < entries / (kCopyWarps * 32) + 1) ctas = entries / (kCopyWarps * 32) + 1;
      ctas = ctas < 1 ? 1 : ctas < num_sms ? ctas : num_sms;
      static std::atomic<uint64_t> ready;
      if (!allow_smem(reinterpret_cast<const void*>(copy_bulk_kernel), ready, smem)) return OC_ERR_CUDA;
      rc = launch_pdl(copy_bulk_kernel, (unsigned)ctas, kCopyWarps * 32, smem, stream, c, job, table, status);
    } else {
      rc = launch_pdl(copy_bytes_kernel, (unsigned)num_sms * 8, 256, 0, stream, c, job, table, status);
    }
    if (rc != OC_OK) return rc;
    table.out = nullptr;
  }
  return OC_OK;
}

// ------------------------------------------------------------------ fork
// One cluster.  The counts are copied and the first entries of both tables
// read; after the cluster's barrier, what came and went is added (integer
// atomics: any order gives the same counts).
__global__ void __launch_bounds__(kThreads) fork_kernel(const int32_t* table_in, int64_t in_stride, int32_t* table_out,
                                                        int64_t out_stride, const int32_t* lens_in, int32_t* lens_out,
                                                        const int32_t* refs_in, int32_t* refs_out,
                                                        const int32_t* source, int num_seqs, int max_blocks,
                                                        int64_t num_pages, int block_size, uint32_t* status) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kEntries = 4;  // of a thread at a time
  const unsigned me = blockIdx.x * blockDim.x + threadIdx.x, all = gridDim.x * blockDim.x;
  const unsigned entries = (unsigned)num_seqs * (unsigned)max_blocks;
  auto source_of = [&](int row) {
    const int from = source[row];
    if (from < num_seqs) return from;
    raise_status(status, OC_STATUS_POSITION);
    return row;
  };
  for (int64_t i = me; i < num_pages; i += all) refs_out[i] = refs_in[i];
  for (unsigned r = me; r < (unsigned)num_seqs; r += all) {
    const int from = source_of((int)r);
    lens_out[r] = from >= 0 ? lens_in[from] : 0;
  }
  for (unsigned base = 0; base < entries; base += all * kEntries) {
    int old[kEntries], now[kEntries];
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      const unsigned e = base + i * all + me;
      old[i] = now[i] = -1;
      if (e >= entries) continue;
      const int row = (int)(e / (unsigned)max_blocks), c = (int)(e - (unsigned)row * (unsigned)max_blocks);
      const int from = source_of(row);
      old[i] = now[i] = table_in[row * in_stride + c];
      if (from != row) {
        now[i] = -1;
        if (from >= 0) {
          const int page = table_in[from * in_stride + c], len = lens_in[from];
          if ((int64_t)c * block_size < len) now[i] = page;
        }
      }
      table_out[row * out_stride + c] = now[i];
      if (from != row && (old[i] >= num_pages || now[i] >= num_pages)) {
        raise_status(status, OC_STATUS_BAD_PAGE);
        old[i] = now[i] = -1;
      }
    }
    if (base == 0) cooperative_groups::this_cluster().sync();  // refs_out holds the old counts
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      if (old[i] == now[i]) continue;
      if (old[i] >= 0) atomicSub(refs_out + old[i], 1);
      if (now[i] >= 0) atomicAdd(refs_out + now[i], 1);
    }
  }
}

// ------------------------------------------------------------------ reserve
// Workspace: [0] copies, [1] whether the pages were reserved, then
// src[num_seqs], dst[num_seqs], and the free pages handed out, free[num_pages].
struct ReserveSpace {
  int32_t *count, *src, *dst, *free;
  __host__ __device__ ReserveSpace(void* p, int num_seqs)
      : count(static_cast<int32_t*>(p)), src(count + 4), dst(src + num_seqs), free(dst + num_seqs) {}
};

// One CTA.  What a row needs is worked out with rows spread over the threads
// and kept in shared memory; they are then taken in runs, one run per thread,
// so that the prefix sum over threads is the prefix sum over rows.  A row
// writes to the pages from the one that its next token goes to.  Of those,
// shared ones are replaced: the first one copied if it holds tokens of the
// row, the ones behind it (a sequence that was shortened while others held its
// pages) without a copy.
__global__ void __launch_bounds__(kThreads) reserve_kernel(int32_t* table, int64_t stride, const int32_t* lens,
                                                           int32_t* refs, const int32_t* wanted, int num_seqs,
                                                           int max_blocks, int64_t num_pages, int block_size,
                                                           void* workspace, uint32_t* status) {
  // x: the page that the row shares and would write to first, or -1; y: pages that it holds, ~y if it shares some
  // behind that one
  extern __shared__ int2 rows[];
  __shared__ int32_t short_list[kShortList];
  __shared__ int bad;
  pdl_launch_dependents();
  pdl_wait();
  const ReserveSpace ws(workspace, num_seqs);
  // the counts of the first pages, read ahead of the rows that will ask for them
  const int4 first_counts = four_at(refs, (int64_t)threadIdx.x * 4, num_pages, 1);
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  auto shared = [&](int page) { return page >= 0 && page < num_pages && refs[page] > 1; };
  // 1: the page that a growing sequence would write to and others hold too; the pages that it has
  for (int r = threadIdx.x; r < num_seqs; r += blockDim.x) {
    const int len = lens[r], first = len / block_size;
    const int goal = pages_for(max(wanted[r], 0), block_size);
    int page = -1, held = pages_for(max(len, 0), block_size);
    bool later = false;
    if (len < 0 || goal > max_blocks) {
      bad = 1;
    } else if (wanted[r] > len) {  // so first < goal
      const int p = table[r * stride + first];
      for (; held < goal; ++held) {
        const int next = table[r * stride + held];
        if (next < 0) break;
        if (held > first) later |= shared(next);
      }
      if (shared(p)) page = p;
    }
    rows[r] = int2{page, later ? ~held : held};
  }
  __syncthreads();
  // 2: what each row needs
  const int per = (num_seqs + blockDim.x - 1) / blockDim.x, r0 = threadIdx.x * per, r1 = min(num_seqs, r0 + per);
  Two need = {0, 0};  // pages, and copies among them
  unsigned replaced = 0;  // one bit per row of the run: its first page
  int some_later = 0;
  for (int r = r0; r < r1; ++r) {
    const int p = rows[r].x, held = rows[r].y < 0 ? ~rows[r].y : rows[r].y;
    if (p >= 0) {
      int writers = 0, last = -1;
      for (int o = 0; o < num_seqs; ++o)
        if (rows[o].x == p) {
          ++writers;
          last = o;
        }
      // if every holder writes, the last of them keeps the page
      if (!(writers == refs[p] && last == r)) {
        replaced |= 1u << (r - r0);
        ++need.a;
        need.b += lens[r] % block_size != 0;
      }
    }
    if (rows[r].y < 0) {
      some_later = 1;
      for (int c = lens[r] / block_size + 1; c < held; ++c) need.a += shared(table[r * stride + c]);
    }
    const int goal = pages_for(max(wanted[r], 0), block_size);
    need.a += !bad && goal > held ? goal - held : 0;
  }
  Two total;
  const Two before = block_scan(need, total);
  int rank = before.a, copied = before.b;
  // 3: the lowest free pages
  int32_t* const list = total.a <= kShortList ? short_list : ws.free;
  int found = 0;
  for (int64_t base = 0; base < num_pages && found < total.a; base += (int64_t)blockDim.x * 4) {
    const int64_t i = base + threadIdx.x * 4;
    const int4 r = base == 0 ? first_counts : four_at(refs, i, num_pages, 1);
    const int f[4] = {r.x == 0, r.y == 0, r.z == 0, r.w == 0};
    Two sum;
    int at = found + block_scan(Two{f[0] + f[1] + f[2] + f[3], 0}, sum).a;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (f[j]) {
        if (at < total.a) list[at] = (int32_t)(i + j);
        ++at;
      }
    found += sum.a;
  }
  some_later = __syncthreads_or(some_later);  // the list is complete
  if (bad || found < total.a) {
    if (threadIdx.x == 0) {
      raise_status(status, OC_STATUS_PAGES);
      ws.count[0] = ws.count[1] = 0;
    }
    return;
  }
  // 4: hand them out (pages that are handed out were free: no count below is read above)
  if (some_later) {  // which ones are shared is settled before the first count changes: entry -2 - page
    for (int r = r0; r < r1; ++r)
      for (int c = lens[r] / block_size + 1; c < ~rows[r].y; ++c) {
        const int p = table[r * stride + c];
        if (shared(p)) table[r * stride + c] = -2 - p;
      }
    __syncthreads();
  }
  for (int r = r0; r < r1; ++r) {
    const int first = lens[r] / block_size, held = rows[r].y < 0 ? ~rows[r].y : rows[r].y;
    if (replaced >> (r - r0) & 1) {
      const int p = rows[r].x, q = list[rank++];
      table[r * stride + first] = q;
      refs[q] = 1;
      atomicSub(refs + p, 1);
      if (lens[r] % block_size != 0) {
        ws.src[copied] = p;
        ws.dst[copied++] = q;
      }
    }
    for (int c = first + 1; c < ~rows[r].y; ++c) {
      const int p = -2 - table[r * stride + c];
      if (p < 0) continue;
      const int q = list[rank++];
      table[r * stride + c] = q;
      refs[q] = 1;
      atomicSub(refs + p, 1);
    }
    const int goal = pages_for(max(wanted[r], 0), block_size);
    for (int c = held; c < goal; ++c) {
      const int q = list[rank++];
      table[r * stride + c] = q;
      refs[q] = 1;
    }
  }
  if (threadIdx.x == 0) {
    ws.count[0] = total.b;
    ws.count[1] = 1;
  }
}

// ------------------------------------------------------------------ compact
// Workspace: [0] moves, then src[num_pages], dst[num_pages], to[num_pages].
struct CompactSpace {
  int32_t *count, *src, *dst, *to;
  __host__ __device__ CompactSpace(void* p, int64_t num_pages)
      : count(static_cast<int32_t*>(p)), src(count + 4), dst(src + num_pages), to(dst + num_pages) {}
};

__global__ void __launch_bounds__(kThreads) compact_plan_kernel(const int32_t* refs_in, int32_t* refs_out,
                                                                int64_t num_pages, void* workspace) {
  pdl_launch_dependents();
  pdl_wait();
  const CompactSpace ws(workspace, num_pages);
  const int64_t chunk = (int64_t)blockDim.x * 4;
  const int4 first = four_at(refs_in, (int64_t)threadIdx.x * 4, num_pages, 0);
  int live = (first.x > 0) + (first.y > 0) + (first.z > 0) + (first.w > 0);
  for (int64_t i = chunk + threadIdx.x * 4; i < num_pages; i += chunk) {
    const int4 r = four_at(refs_in, i, num_pages, 0);
    live += (r.x > 0) + (r.y > 0) + (r.z > 0) + (r.w > 0);
  }
  Two sum;
  block_scan(Two{live, 0}, sum);
  const int n = sum.a;
  int holes = 0, movers = 0;
  for (int64_t base = 0; base < num_pages; base += chunk) {
    const int64_t i0 = base + threadIdx.x * 4;
    const int4 r = base == 0 ? first : four_at(refs_in, i0, num_pages, 0);
    const int ref[4] = {r.x, r.y, r.z, r.w};
    Two c = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c.a += i0 + j < n && ref[j] <= 0;
      c.b += i0 + j >= n && ref[j] > 0;
    }
    const Two before = block_scan(c, sum);
    int hat = holes + before.a, mat = movers + before.b;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = i0 + j;
      if (i >= num_pages) continue;
      const bool used = ref[j] > 0;
      if (i < n && !used) ws.dst[hat++] = (int32_t)i;
      if (i >= n && used) ws.src[mat++] = (int32_t)i;
      else ws.to[i] = (int32_t)i;
      refs_out[i] = i < n && used ? ref[j] : 0;
    }
    holes += sum.a;
    movers += sum.b;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += blockDim.x) {  // as many holes as movers
    const int32_t s = ws.src[i], d = ws.dst[i];
    ws.to[s] = d;
    refs_out[d] = refs_in[s];
  }
  if (threadIdx.x == 0) *ws.count = movers;
}

bool bad_caches(void* const* caches, const int64_t* strides, int num_caches, int64_t page_bytes) {
  if (num_caches < 0 || page_bytes < 1 || (num_caches && (!caches || !strides))) return true;
  for (int i = 0; i < num_caches; ++i)
    if (!caches[i] || strides[i] < page_bytes) return true;
  return false;
}

constexpr int kMaxSeqs = 4096;  // rows of one reserve call (their needs are held in shared memory)

}  // namespace

extern "C" int oc_copy_pages(void* const* caches, const int64_t* page_strides, int num_caches, int64_t page_bytes,
                             int64_t num_pages, const int32_t* src, const int32_t* dst, int64_t n, uint32_t* status,
                             int num_sms, void* stream) {
  if (bad_caches(caches, page_strides, num_caches, page_bytes) || num_pages < 0 || n < 0 || num_sms < 1 ||
      (n && (!src || !dst)))
    return OC_ERR_INVALID;
  if (n == 0) return OC_OK;
  return copy_all(caches, page_strides, num_caches, page_bytes, num_pages, src, dst, n, nullptr, Renumber{}, status,
                  num_sms, stream);
}

extern "C" int oc_fork_sequences(const int32_t* table_in, int64_t table_in_stride, int32_t* table_out,
                                 int64_t table_out_stride, const int32_t* lens_in, int32_t* lens_out,
                                 const int32_t* refs_in, int32_t* refs_out, const int32_t* source, int num_seqs,
                                 int max_blocks, int64_t num_pages, int block_size, uint32_t* status, void* stream) {
  if (num_seqs < 0 || max_blocks < 0 || num_pages < 0 || block_size < 1 ||
      (num_seqs && (!lens_in || !lens_out || !source)) ||
      (num_seqs && max_blocks && (!table_in || !table_out || table_in == table_out)) ||
      (num_pages && (!refs_in || !refs_out || refs_in == refs_out)))
    return OC_ERR_INVALID;
  if ((int64_t)num_seqs * max_blocks > 0x3fffffff) return OC_ERR_TOO_LARGE;
  if (num_seqs == 0 && num_pages == 0) return OC_OK;
  cudaLaunchConfig_t cfg = {};
  constexpr unsigned ctas = 8;  // one CTA alone is slower even for small tables (10.6 against 6.9 us at 64 x 59 entries)
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = ctas;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, fork_kernel, table_in, table_in_stride, table_out, table_out_stride, lens_in, lens_out,
                         refs_in, refs_out, source, num_seqs, max_blocks, num_pages, block_size,
                         status) != cudaSuccess) {
    cudaGetLastError();
    return OC_ERR_CUDA;
  }
  return OC_OK;
}

extern "C" size_t oc_reserve_workspace_bytes(int num_seqs, int64_t num_pages) {
  if (num_seqs < 0 || num_pages < 0) return 0;
  return 4 * (4 + 2 * (size_t)num_seqs + (size_t)num_pages);
}

extern "C" int oc_reserve_pages(void* const* caches, const int64_t* page_strides, int num_caches, int64_t page_bytes,
                                int32_t* table, int64_t table_stride, const int32_t* lens, int32_t* refs,
                                const int32_t* wanted, int num_seqs, int max_blocks, int64_t num_pages,
                                int block_size, void* workspace, size_t workspace_bytes, uint32_t* status, int num_sms,
                                void* stream) {
  if (bad_caches(caches, page_strides, num_caches, page_bytes) || num_seqs < 0 || max_blocks < 0 || num_pages < 0 ||
      num_pages > 0x7fffffff || block_size < 1 || num_sms < 1 ||
      (num_seqs && (!lens || !wanted || !refs || (max_blocks && !table))))
    return OC_ERR_INVALID;
  if (num_seqs > kMaxSeqs) return OC_ERR_TOO_LARGE;
  if (num_seqs == 0) return OC_OK;
  if (!workspace || !aligned_to(workspace, 4) || workspace_bytes < oc_reserve_workspace_bytes(num_seqs, num_pages))
    return OC_ERR_WORKSPACE;
  const int rc = launch_pdl(reserve_kernel, 1, kThreads, num_seqs * sizeof(int2), stream, table, table_stride, lens,
                            refs, wanted, num_seqs, max_blocks, num_pages, block_size, workspace, status);
  if (rc != OC_OK || num_caches == 0) return rc;
  const ReserveSpace ws(workspace, num_seqs);
  return copy_all(caches, page_strides, num_caches, page_bytes, num_pages, ws.src, ws.dst, num_seqs, ws.count,
                  Renumber{}, status, num_sms, stream);
}

extern "C" size_t oc_compact_workspace_bytes(int64_t num_pages) {
  return num_pages < 0 ? 0 : 4 * (4 + 3 * (size_t)num_pages);
}

extern "C" int oc_compact_pages(void* const* caches, const int64_t* page_strides, int num_caches, int64_t page_bytes,
                                const int32_t* table_in, int64_t table_in_stride, int32_t* table_out,
                                int64_t table_out_stride, const int32_t* refs_in, int32_t* refs_out, int num_seqs,
                                int max_blocks, int64_t num_pages, void* workspace, size_t workspace_bytes,
                                uint32_t* status, int num_sms, void* stream) {
  if (bad_caches(caches, page_strides, num_caches, page_bytes) || num_seqs < 0 || max_blocks < 0 || num_pages < 0 ||
      num_pages > 0x7fffffff || num_sms < 1 || (num_pages && (!refs_in || !refs_out || refs_in == refs_out)) ||
      (num_seqs && max_blocks && (!table_in || !table_out || table_in == table_out)))
    return OC_ERR_INVALID;
  if (num_pages == 0) return OC_OK;
  if (!workspace || !aligned_to(workspace, 4) || workspace_bytes < oc_compact_workspace_bytes(num_pages))
    return OC_ERR_WORKSPACE;
  const CompactSpace ws(workspace, num_pages);
  const int rc = launch_pdl(compact_plan_kernel, 1, kThreads, 0, stream, refs_in, refs_out, num_pages, workspace);
  if (rc != OC_OK) return rc;
  Renumber table = {};
  if (num_seqs > 0 && max_blocks > 0)
    table = Renumber{table_in, ws.to, table_out, table_in_stride, table_out_stride, num_seqs, max_blocks};
  return copy_all(caches, page_strides, num_caches, page_bytes, num_pages, ws.src, ws.dst, num_pages, ws.count, table,
                  status, num_sms, stream);
}
