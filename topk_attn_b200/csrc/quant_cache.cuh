// Parameters of the kernels that write and read back quantised key/value caches, and the element
// types shared by the kernels that work on such caches.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace ra {

// Formats of a cache's rows of 128 values (the RA_CACHE_* numbers of the C ABI).
enum CacheFormat { kCacheFp16 = 0, kCacheBf16 = 1, kCacheInt8 = 2, kCacheFp8 = 3, kCacheInt4 = 4 };

__host__ __device__ constexpr int cache_row_bytes(int format) {
  return format <= kCacheBf16 ? 256 : (format == kCacheInt4 ? 64 : 128);
}
// scales of one row: one, or one for each 32 values
__host__ __device__ constexpr int cache_row_scales(int format) {
  return format <= kCacheBf16 ? 0 : (format == kCacheInt4 ? 4 : 1);
}

// A key/value cache as the kernels see it: strides in bytes for the rows and in floats for the scales.
struct CacheView {
  unsigned char* k;
  unsigned char* v;
  float* k_scale;
  float* v_scale;
  int n_tokens;
  long long bstride, tstride, hstride;
  long long sbstride, shstride;
};

// Loads of what an earlier kernel may have written while this one, launched early, was already there: after
// griddepcontrol.wait, and not through the read-only path, which is for data that nobody writes as long as the
// kernel lives.  Volatile, so that they stay behind the wait.
__device__ __forceinline__ uint4 ld128(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint2 ld64(const void* p) {
  uint2 r;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t ld32(const void* p) {
  uint32_t r;
  asm volatile("ld.global.u32 %0, [%1];" : "=r"(r) : "l"(p));
  return r;
}

constexpr int kQuantMaxHeads = 1024;

struct QuantParams {
  CacheView cache;
  void* rows[2];            // K and V rows, fp16 or bf16
  long long rb[2], rt[2], rh[2];   // their strides in elements
  int caches, heads, n_rows;
  int tile;                 // tokens of a CTA (set by the launch)
  const int* positions;     // [caches] or null
  int position;
  const int* counts;        // [caches] or null
  int early;                // launched while the kernel before it still runs, which the kernel waits for
  unsigned* status;
};

cudaError_t launch_kv_quantize(const QuantParams& P, int format, bool bf16, cudaStream_t stream);
cudaError_t launch_kv_dequantize(const QuantParams& P, int format, bool bf16, cudaStream_t stream);

}  // namespace ra
