// Parameters of decode attention over a prefix shared by the batch and each row's own cache.
#pragma once
#include "quant_cache.cuh"

namespace ra {

constexpr int kPartialFloats = kHeadDim + 2;   // un-normalised sums, weight, maximum (log2 domain)

struct CacheAttendParams {
  CacheView cache;          // of the segment that is attended to
  const void* q;            // fp16 or bf16 [batch, hq, 128]
  float* partials;
  const int* seq_lens;      // [batch] or null: every row sees all tokens of the segment
  unsigned* status;
  int batch, hq, hkv, group;
  int splits, split_len;
  float scale_log2e;
};

cudaError_t launch_cache_attend(const CacheAttendParams& P, int format, bool bf16, cudaStream_t stream);
cudaError_t launch_cache_combine(const float* a, int na, const float* b, int nb, int rows, void* out, bool bf16,
                                 cudaStream_t stream);

}  // namespace ra
