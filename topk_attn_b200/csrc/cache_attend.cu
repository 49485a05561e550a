// Decode attention over one segment (a prefix shared by the batch, or each row's own cache) in any
// of the cache formats, and the joining of the segments' partials.
//
// Simple form: one CTA per (batch row, query head, split of the tokens), a warp per token with four
// dimensions in each lane, online softmax, partials (sums, weight, maximum) joined by their maxima.
#include "cache_attend.cuh"

namespace ra {

constexpr int kAttendWarps = 4;

template <int FMT>
__device__ __forceinline__ void load4(const unsigned char* row, const float* scale, int lane, float (&x)[4]) {
  if (FMT == kCacheFp16 || FMT == kCacheBf16) {
    const uint2 u = *reinterpret_cast<const uint2*>(row + 8 * lane);
    if (FMT == kCacheBf16) {
      x[0] = __uint_as_float(u.x << 16);
      x[1] = __uint_as_float(u.x & 0xffff0000u);
      x[2] = __uint_as_float(u.y << 16);
      x[3] = __uint_as_float(u.y & 0xffff0000u);
    } else {
      const float2 a = h2f2(u.x), b = h2f2(u.y);
      x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    }
  } else if (FMT == kCacheInt4) {
    const uint32_t w = *reinterpret_cast<const uint16_t*>(row + 2 * lane);
    const float s = scale[lane >> 3];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)((int)((w >> (4 * i)) & 15u) - 8) * s;
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(row + 4 * lane);
    const float s = scale[0];
    if (FMT == kCacheInt8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i)) * s;
    } else {
      uint32_t a, b;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"((uint16_t)w));
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"((uint16_t)(w >> 16)));
      const float2 f = h2f2(a), g = h2f2(b);
      x[0] = f.x * s; x[1] = f.y * s; x[2] = g.x * s; x[3] = g.y * s;
    }
  }
}

template <int FMT, bool BF16>
__global__ void __launch_bounds__(32 * kAttendWarps)
cache_attend_kernel(const __grid_constant__ CacheAttendParams P) {
  __shared__ float sm_o[kAttendWarps][kHeadDim], sm_m[kAttendWarps], sm_l[kAttendWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x, row = blockIdx.y, b = row / P.hq, h = (row % P.hq) / P.group;
  int len = P.cache.n_tokens;
  if (P.seq_lens) {
    const int asked = P.seq_lens[b];
    if ((asked < 0 || asked > len) && threadIdx.x == 0 && split == 0) atomicOr(P.status, kStatusBadToken);
    len = max(0, min(len, asked));
  }
  const int lo = split * P.split_len, hi = min(len, lo + P.split_len);
  float q[4];
  load4<BF16 ? kCacheBf16 : kCacheFp16>(static_cast<const unsigned char*>(P.q) + (size_t)row * kRowBytes, nullptr,
                                        lane, q);
  constexpr int kScales = cache_row_scales(FMT);
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t = lo + warp; t < hi; t += kAttendWarps) {
    const long long at = b * P.cache.bstride + t * P.cache.tstride + h * P.cache.hstride;
    const long long sat = b * P.cache.sbstride + h * P.cache.shstride + (long long)t * kScales;
    float k[4], v[4];
    load4<FMT>(P.cache.k + at, P.cache.k_scale + sat, lane, k);
    load4<FMT>(P.cache.v + at, P.cache.v_scale + sat, lane, v);
    float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
    for (int i = 16; i; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    s *= P.scale_log2e;
    const float m_new = fmaxf(m, s), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float a = exp2f(m - m_use), p = exp2f(s - m_use);
    l = l * a + p;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * a + p * v[i];
    m = m_new;
  }
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sm_o[warp][4 * lane + i] = o[i];
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kAttendWarps; ++w) top = fmaxf(top, sm_m[w]);
  const float use = top == -INFINITY ? 0.f : top;
  float sum = 0.f, wsum = 0.f;
#pragma unroll
  for (int w = 0; w < kAttendWarps; ++w) {
    const float f = exp2f(sm_m[w] - use);
    sum += f * sm_o[w][threadIdx.x];
    wsum += f * sm_l[w];
  }
  float* out = P.partials + ((size_t)row * P.splits + split) * kPartialFloats;
  out[threadIdx.x] = sum;
  if (threadIdx.x == 0) {
    out[kHeadDim] = wsum;
    out[kHeadDim + 1] = top;
  }
}

// out[row] = sum over both segments' partials, joined by their maxima; zeros where nothing was seen.
template <bool BF16>
__global__ void __launch_bounds__(kHeadDim)
cache_combine_kernel(const float* a, int na, const float* b, int nb, void* out) {
  const int row = blockIdx.x, d = threadIdx.x;
  float m = -INFINITY;
  for (int i = 0; i < na + nb; ++i) {
    const float* p = i < na ? a + ((size_t)row * na + i) * kPartialFloats : b + ((size_t)row * nb + i - na) * kPartialFloats;
    m = fmaxf(m, p[kHeadDim + 1]);
  }
  const float use = m == -INFINITY ? 0.f : m;
  float sum = 0.f, w = 0.f;
  for (int i = 0; i < na + nb; ++i) {
    const float* p = i < na ? a + ((size_t)row * na + i) * kPartialFloats : b + ((size_t)row * nb + i - na) * kPartialFloats;
    const float f = exp2f(p[kHeadDim + 1] - use);
    sum += f * p[d];
    w += f * p[kHeadDim];
  }
  const float r = w == 0.f ? 0.f : sum / w;
  if (BF16) static_cast<__nv_bfloat16*>(out)[(size_t)row * kHeadDim + d] = __float2bfloat16_rn(r);
  else static_cast<__half*>(out)[(size_t)row * kHeadDim + d] = __float2half_rn(r);
}

namespace {

template <int FMT>
cudaError_t launch_one(const CacheAttendParams& P, bool bf16, cudaStream_t stream) {
  const dim3 grid(P.splits, P.batch * P.hq);
  note_launch();
  if (bf16) cache_attend_kernel<FMT, true><<<grid, 32 * kAttendWarps, 0, stream>>>(P);
  else cache_attend_kernel<FMT, false><<<grid, 32 * kAttendWarps, 0, stream>>>(P);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_cache_attend(const CacheAttendParams& P, int format, bool bf16, cudaStream_t stream) {
  switch (format) {
    case kCacheFp16: return launch_one<kCacheFp16>(P, bf16, stream);
    case kCacheBf16: return launch_one<kCacheBf16>(P, bf16, stream);
    case kCacheInt8: return launch_one<kCacheInt8>(P, bf16, stream);
    case kCacheFp8: return launch_one<kCacheFp8>(P, bf16, stream);
    default: return launch_one<kCacheInt4>(P, bf16, stream);
  }
}

cudaError_t launch_cache_combine(const float* a, int na, const float* b, int nb, int rows, void* out, bool bf16,
                                 cudaStream_t stream) {
  note_launch();
  if (bf16) cache_combine_kernel<true><<<rows, kHeadDim, 0, stream>>>(a, na, b, nb, out);
  else cache_combine_kernel<false><<<rows, kHeadDim, 0, stream>>>(a, na, b, nb, out);
  return cudaGetLastError();
}

}  // namespace ra
