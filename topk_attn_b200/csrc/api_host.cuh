// What the host sources of the C ABI share: the error text of the calling thread, the device's
// multiprocessor count and the driver's tensor-map encoder (defined in api.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

namespace ra {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int host_fail(int status, const char* why);             // records the text, returns the status
int host_cuda_fail(cudaError_t e, const char* what);    // RA_ERR_CUDA with the runtime's text
int host_sm_count();                                    // of the current device
EncodeTiledFn host_encode_fn();                         // null where the driver has none


// Raises a kernel's dynamic shared memory limit, once for each device (`done`: a bit for each).
template <typename Kernel>
cudaError_t allow_smem(Kernel kern, size_t bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace ra
