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
