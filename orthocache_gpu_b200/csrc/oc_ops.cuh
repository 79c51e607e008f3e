// Helpers shared by the paged-serving operators (oc_rotary.cu, oc_pages.cu,
// oc_paged_attn.cu, oc_prompt_attn.cu): element conversion, 16-byte vectors,
// and programmatic dependent launches.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/orthocache_b200.h"

namespace oc {

// Bound of a wait for a copy (a build option: with 0 every wait runs out), and
// of the waits after one has run out: for the copies that are still in flight,
// which must land before the CTA's memory is given back.
#ifndef OC_WAIT_POLLS
#define OC_WAIT_POLLS (1u << 22)
#endif
constexpr uint32_t kPolls = OC_WAIT_POLLS, kLandPolls = 1u << 22;

struct fp8_t {
  uint8_t b;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(fp8_t x) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(x.b, __NV_E4M3)));
}

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ fp8_t from_f32<fp8_t>(float x) {  // saturating, NaN stays NaN
  return fp8_t{static_cast<uint8_t>(__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3))};
}

// N elements moved as one access where ALIGNED (N * sizeof(T) is 4, 8 or 16).
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T e[N];
};

// Programmatic dependent launch: a kernel launched with launch_pdl() may
// start while the kernel before it on the stream drains; it touches no
// global memory before pdl_wait(), which returns when that kernel has
// completed and its writes are visible.  Every CTA of every kernel launched
// this way calls pdl_wait() first, so completion is transitive along a stream.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename... P, typename... A>
inline int launch_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, void* stream, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  if (e != cudaSuccess) {
    cudaGetLastError();  // the error is reported here, not by a later launch
    return OC_ERR_CUDA;
  }
  return OC_OK;
}

// Lets a kernel use `bytes` of dynamic shared memory on the current device.
// The attribute outlives the call: `done` (one per kernel) remembers the
// devices that have it.
inline bool allow_smem(const void* kernel, std::atomic<uint64_t>& done, int bytes) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return true;
}

__device__ __forceinline__ void raise_status(uint32_t* status, uint32_t bits) {
  if (status) atomicOr(status, bits);
}

inline bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline int type_bytes(int dt) {
  return dt == OC_F32 ? 4 : dt == OC_F16 || dt == OC_BF16 ? 2 : dt == OC_F8E4M3 ? 1 : 0;
}

}  // namespace oc
