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
#include <cooperative_groups.h>

#include "oc_ops.cuh"

namespace {

using namespace oc;

constexpr int kMaxCaches = 128;  // pointers that travel in one launch's parameters
constexpr int kThreads = 1024;

struct Caches {
  char* base[kMaxCaches];
  int64_t stride[kMaxCaches];  // bytes from page to page
};

// ------------------------------------------------------------------ block scan
// Exclusive prefix sum of v over the CTA; total returns the sum.
__device__ __forceinline__ int block_scan(int v, int& total) {
  __shared__ int part[33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // part may still be read by an earlier call
  if (lane == 31) part[w] = x;
  __syncthreads();
  if (w == 0) {
    int p = lane < (int)(blockDim.x >> 5) ? part[lane] : 0;
    const int own = p;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, p, o);
      if (lane >= o) p += y;
    }
    part[lane] = p - own;
    if (lane == 31) part[32] = p;
  }
  __syncthreads();
  total = part[32];
  return part[w] + x - v;
}

// ------------------------------------------------------------------ page copies
// Pairs come from arrays of n entries, or of *n_dev entries on the device.
// One warp-group unit = (pair, cache, chunk of a page); a grid-stride loop.
template <int BYTES>
__global__ void __launch_bounds__(256) copy_kernel(const __grid_constant__ Caches caches, int num_caches,
                                                   int64_t page_bytes, int64_t num_pages, const int32_t* src,
                                                   const int32_t* dst, int64_t n, const int32_t* n_dev,
                                                   uint32_t* status) {
  pdl_launch_dependents();
  pdl_wait();
  if (n_dev) n = *n_dev;
  constexpr int64_t kChunk = 256 * 4 * BYTES;
  const int64_t chunks = (page_bytes + kChunk - 1) / kChunk, units = n * num_caches * chunks;
  using V = Vec<uint8_t, BYTES>;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t pc = u / chunks, chunk = u - pc * chunks;
    const int64_t pair = pc / num_caches;
    const int c = (int)(pc - pair * num_caches);
    const int64_t s = src[pair], d = dst[pair];
    if (s < 0 || d < 0) continue;
    if (s >= num_pages || d >= num_pages) {
      if (threadIdx.x == 0) raise_status(status, OC_STATUS_BAD_PAGE);
      continue;
    }
    const char* from = caches.base[c] + s * caches.stride[c];
    char* to = caches.base[c] + d * caches.stride[c];
    const int64_t begin = chunk * kChunk + threadIdx.x * BYTES;
    V v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (begin + i * 256 * BYTES < page_bytes) v[i] = *reinterpret_cast<const V*>(from + begin + i * 256 * BYTES);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (begin + i * 256 * BYTES < page_bytes) *reinterpret_cast<V*>(to + begin + i * 256 * BYTES) = v[i];
  }
}

// Copies over every cache; at most `most` pairs.
int copy_all(void* const* caches, const int64_t* strides, int num_caches, int64_t page_bytes, int64_t num_pages,
             const int32_t* src, const int32_t* dst, int64_t most, const int32_t* n_dev, uint32_t* status, int num_sms,
             void* stream) {
  for (int first = 0; first < num_caches; first += kMaxCaches) {
    const int m = num_caches - first < kMaxCaches ? num_caches - first : kMaxCaches;
    Caches c = {};
    bool vec = page_bytes % 16 == 0;
    for (int i = 0; i < m; ++i) {
      c.base[i] = static_cast<char*>(caches[first + i]);
      c.stride[i] = strides[first + i];
      vec = vec && aligned_to(c.base[i], 16) && c.stride[i] % 16 == 0;
    }
    const int64_t chunk = 256 * 4 * (vec ? 16 : 1);
    const int64_t units = most * m * ((page_bytes + chunk - 1) / chunk);
    const int64_t full = (int64_t)num_sms * 8;
    const unsigned grid = (unsigned)(units < full ? (units < 1 ? 1 : units) : full);
    const int rc = vec ? launch_pdl(copy_kernel<16>, grid, 256, 0, stream, c, m, page_bytes, num_pages, src, dst, most,
                                    n_dev, status)
                       : launch_pdl(copy_kernel<1>, grid, 256, 0, stream, c, m, page_bytes, num_pages, src, dst, most,
                                    n_dev, status);
    if (rc != OC_OK) return rc;
  }
  return OC_OK;
}

// ------------------------------------------------------------------ fork
// One cluster.  Phase 1 copies the counts; after the cluster's barrier, phase
// 2 writes the rows and adds what came and went (integer atomics: any order
// gives the same counts).
__global__ void __launch_bounds__(kThreads) fork_kernel(const int32_t* table_in, int64_t in_stride, int32_t* table_out,
                                                        int64_t out_stride, const int32_t* lens_in, int32_t* lens_out,
                                                        const int32_t* refs_in, int32_t* refs_out,
                                                        const int32_t* source, int num_seqs, int max_blocks,
                                                        int64_t num_pages, int block_size, uint32_t* status) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t me = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, all = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = me; i < num_pages; i += all) refs_out[i] = refs_in[i];
  cooperative_groups::this_cluster().sync();
  // a warp per row
  const int lane = threadIdx.x & 31;
  for (int64_t row = me >> 5; row < num_seqs; row += all >> 5) {
    int from = source[row];
    if (from >= num_seqs) {
      if (lane == 0) raise_status(status, OC_STATUS_POSITION);
      from = (int)row;
    }
    const bool stays = from == row;
    const int len = from >= 0 ? lens_in[from] : 0;
    const int used = stays ? max_blocks : min(max_blocks, (len + block_size - 1) / block_size);
    if (lane == 0) lens_out[row] = len;
    for (int c = lane; c < max_blocks; c += 32) {
      const int old = table_in[row * in_stride + c];
      const int now = stays ? old : from >= 0 && c < used ? table_in[(int64_t)from * in_stride + c] : -1;
      table_out[row * out_stride + c] = now;
      if (stays) continue;
      if (old >= num_pages || now >= num_pages) {
        raise_status(status, OC_STATUS_BAD_PAGE);
        continue;
      }
      if (old == now) continue;
      if (old >= 0) atomicSub(refs_out + old, 1);
      if (now >= 0) atomicAdd(refs_out + now, 1);
    }
  }
}

// ------------------------------------------------------------------ reserve
// Workspace: [0] copies, [1] unused, then src[num_seqs], dst[num_seqs], and
// the free pages handed out, free[num_pages].
struct ReserveSpace {
  int32_t *count, *src, *dst, *free;
  __host__ __device__ ReserveSpace(void* p, int num_seqs)
      : count(static_cast<int32_t*>(p)), src(count + 4), dst(src + num_seqs), free(dst + num_seqs) {}
};

// One CTA.  Rows are taken in runs, one run per thread, so that the prefix sum
// over threads is the prefix sum over rows.  Shared memory: per row the page
// it shares and would write to (or -1), and whether it copies it.
__global__ void __launch_bounds__(kThreads) reserve_kernel(int32_t* table, int64_t stride, const int32_t* lens,
                                                           int32_t* refs, const int32_t* wanted, int num_seqs,
                                                           int max_blocks, int64_t num_pages, int block_size,
                                                           void* workspace, uint32_t* status) {
  extern __shared__ int32_t shared_page[];  // num_seqs
  __shared__ int bad;
  pdl_launch_dependents();
  pdl_wait();
  const ReserveSpace ws(workspace, num_seqs);
  if (threadIdx.x == 0) bad = 0;
  // 1: the page that a growing sequence would write to and others hold too
  for (int r = threadIdx.x; r < num_seqs; r += blockDim.x) {
    const int len = lens[r], part = len / block_size;
    int page = -1;
    if (wanted[r] > len && len > 0 && len % block_size != 0 && part < max_blocks) {
      const int p = table[r * stride + part];
      if (p >= 0 && p < num_pages && refs[p] > 1) page = p;
    }
    shared_page[r] = page;
  }
  __syncthreads();
  // 2: what each row needs
  const int per = (num_seqs + blockDim.x - 1) / blockDim.x, r0 = threadIdx.x * per, r1 = min(num_seqs, r0 + per);
  int need = 0;
  unsigned long long copies = 0;  // one bit per row of the run (per <= 64)
  for (int r = r0; r < r1; ++r) {
    const int p = shared_page[r];
    if (p >= 0) {
      int writers = 0, last = -1;
      for (int o = 0; o < num_seqs; ++o)
        if (shared_page[o] == p) {
          ++writers;
          last = o;
        }
      // if every holder writes, the last of them keeps the page
      if (!(writers == refs[p] && last == r)) {
        copies |= 1ull << (r - r0);
        ++need;
      }
    }
    const int len = lens[r], goal = (int)(((int64_t)wanted[r] + block_size - 1) / block_size);
    if (len < 0 || goal > max_blocks) {
      bad = 1;
      continue;
    }
    int held = (len + block_size - 1) / block_size;
    while (held < goal && table[r * stride + held] >= 0) ++held;
    need += goal > held ? goal - held : 0;
  }
  int total;
  int rank = block_scan(need, total);
  // 3: the lowest free pages
  int found = 0;
  for (int64_t base = 0; base < num_pages && found < total; base += (int64_t)blockDim.x * 4) {
    const int64_t i = base + threadIdx.x * 4;
    int f[4], n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = i + j < num_pages && refs[i + j] == 0;
      n += f[j];
    }
    int sum;
    int at = found + block_scan(n, sum);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (f[j]) {
        if (at < total) ws.free[at] = (int32_t)(i + j);
        ++at;
      }
    found += sum;
  }
  __syncthreads();  // ws.free and bad are complete
  int copied_before, all_copies;
  copied_before = block_scan(__popcll(copies), all_copies);
  if (bad || found < total) {
    if (threadIdx.x == 0) {
      raise_status(status, OC_STATUS_PAGES);
      *ws.count = 0;
    }
    return;
  }
  // 4: hand them out (pages that are handed out were free: no count below is read above)
  for (int r = r0; r < r1; ++r) {
    const int len = lens[r], goal = (int)(((int64_t)wanted[r] + block_size - 1) / block_size);
    if (copies >> (r - r0) & 1) {
      const int p = shared_page[r], q = ws.free[rank++];
      table[r * stride + len / block_size] = q;
      refs[q] = 1;
      atomicSub(refs + p, 1);
      ws.src[copied_before] = p;
      ws.dst[copied_before++] = q;
    }
    int held = (len + block_size - 1) / block_size;
    while (held < goal && table[r * stride + held] >= 0) ++held;
    for (; held < goal; ++held) {
      const int q = ws.free[rank++];
      table[r * stride + held] = q;
      refs[q] = 1;
    }
  }
  if (threadIdx.x == 0) *ws.count = all_copies;
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
  int live = 0;
  for (int64_t i = threadIdx.x; i < num_pages; i += blockDim.x) live += refs_in[i] > 0;
  int n;
  block_scan(live, n);
  int holes = 0, movers = 0;
  for (int64_t base = 0; base < num_pages; base += (int64_t)blockDim.x * 4) {
    const int64_t i0 = base + threadIdx.x * 4;
    int h = 0, m = 0;
    int32_t ref[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = i0 + j;
      ref[j] = i < num_pages ? refs_in[i] : 0;
      h += i < n && ref[j] <= 0;
      m += i >= n && ref[j] > 0;
    }
    int hs, ms;
    int hat = holes + block_scan(h, hs), mat = movers + block_scan(m, ms);
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
    holes += hs;
    movers += ms;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += blockDim.x) {  // as many holes as movers
    const int32_t s = ws.src[i], d = ws.dst[i];
    ws.to[s] = d;
    refs_out[d] = refs_in[s];
  }
  if (threadIdx.x == 0) *ws.count = movers;
}

__global__ void __launch_bounds__(256) renumber_kernel(const int32_t* table_in, int64_t in_stride, int32_t* table_out,
                                                       int64_t out_stride, int num_seqs, int max_blocks,
                                                       int64_t num_pages, const int32_t* to, uint32_t* status) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t entries = (int64_t)num_seqs * max_blocks;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < entries; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = e / max_blocks, c = e - r * max_blocks;
    const int32_t p = table_in[r * in_stride + c];
    if (p >= num_pages) raise_status(status, OC_STATUS_BAD_PAGE);
    table_out[r * out_stride + c] = p < 0 || p >= num_pages ? -1 : to[p];
  }
}

bool bad_caches(void* const* caches, const int64_t* strides, int num_caches, int64_t page_bytes) {
  if (num_caches < 0 || page_bytes < 1 || (num_caches && (!caches || !strides))) return true;
  for (int i = 0; i < num_caches; ++i)
    if (!caches[i] || strides[i] < page_bytes) return true;
  return false;
}

constexpr int kMaxSeqs = 8192;  // rows of one reserve call (their shared pages are held in shared memory)

}  // namespace

extern "C" int oc_copy_pages(void* const* caches, const int64_t* page_strides, int num_caches, int64_t page_bytes,
                             int64_t num_pages, const int32_t* src, const int32_t* dst, int64_t n, uint32_t* status,
                             int num_sms, void* stream) {
  if (bad_caches(caches, page_strides, num_caches, page_bytes) || num_pages < 0 || n < 0 || num_sms < 1 ||
      (n && (!src || !dst)))
    return OC_ERR_INVALID;
  if (n == 0) return OC_OK;
  return copy_all(caches, page_strides, num_caches, page_bytes, num_pages, src, dst, n, nullptr, status, num_sms,
                  stream);
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
  if (num_seqs == 0 && num_pages == 0) return OC_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(8);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 8;
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
  const int rc = launch_pdl(reserve_kernel, 1, kThreads, num_seqs * sizeof(int32_t), stream, table, table_stride, lens,
                            refs, wanted, num_seqs, max_blocks, num_pages, block_size, workspace, status);
  if (rc != OC_OK || num_caches == 0) return rc;
  const ReserveSpace ws(workspace, num_seqs);
  return copy_all(caches, page_strides, num_caches, page_bytes, num_pages, ws.src, ws.dst, num_seqs, ws.count, status,
                  num_sms, stream);
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
  int rc = launch_pdl(compact_plan_kernel, 1, kThreads, 0, stream, refs_in, refs_out, num_pages, workspace);
  const int64_t entries = (int64_t)num_seqs * max_blocks;
  if (rc == OC_OK && entries > 0) {
    const int64_t blocks = (entries + 255) / 256;
    rc = launch_pdl(renumber_kernel, (unsigned)(blocks < num_sms * 8 ? blocks : num_sms * 8), 256, 0, stream, table_in,
                    table_in_stride, table_out, table_out_stride, num_seqs, max_blocks, num_pages, ws.to, status);
  }
  if (rc == OC_OK && num_caches > 0)
    rc = copy_all(caches, page_strides, num_caches, page_bytes, num_pages, ws.src, ws.dst, num_pages, ws.count, status,
                  num_sms, stream);
  return rc;
}
