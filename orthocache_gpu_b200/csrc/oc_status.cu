// The status word that the library keeps on each device for callers that want
// one word for everything that runs there, whatever stream or graph it runs
// in: zero when the library is loaded, and it lasts as long as the process.
#include <cstdint>

#include <cuda_runtime.h>

#include "../../include/orthocache_b200.h"

namespace {

__device__ uint32_t device_word;

__global__ void clear_kernel(uint32_t* word, uint32_t bits) { atomicAnd(word, ~bits); }

}  // namespace

extern "C" int oc_device_status(uint32_t** word) {
  if (!word) return OC_ERR_INVALID;
  // the first call may load the module, which a stream capture of this thread must not mind
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  void* p = nullptr;
  if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) {
    cudaGetLastError();
    return OC_ERR_CUDA;
  }
  const bool found = cudaGetSymbolAddress(&p, device_word) == cudaSuccess;
  if (!found) cudaGetLastError();
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (!found) return OC_ERR_CUDA;
  *word = static_cast<uint32_t*>(p);
  return OC_OK;
}

extern "C" int oc_clear_status(uint32_t* word, uint32_t bits, void* stream) {
  if (!word) return OC_ERR_INVALID;
  clear_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(word, bits);
  if (cudaGetLastError() != cudaSuccess) return OC_ERR_CUDA;
  return OC_OK;
}
