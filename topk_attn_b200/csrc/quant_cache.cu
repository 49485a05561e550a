// Quantising key/value rows as they are written into a cache, and reading them back.
//
// One scale s for a row x of 128 values (int8, fp8 e4m3) or for each 32 of them (int4):
//   int8  s = amax / 127     c = rne(x / s)       int4  s = amax / 7, likewise, stored as c + 8
//   fp8   s = 2^k, the least with amax <= 448 s   c = e4m3(x / s), exact but for the one rounding
// and the value read back is c s.  A row (a group) whose largest magnitude is below 2^-100 is stored
// as zeros with s = 0; one that holds an infinity or a NaN is stored with s = NaN, so that it reads
// back as NaN throughout instead of as wrong finite values.
//
// Both kernels are bound by memory: 256 bytes on one side and 132 (80 for int4) on the other for
// each row.  16 lanes share a row, 16 bytes of it each.
#include "quant_cache.cuh"

namespace ra {

constexpr int kQuantThreads = 256;
constexpr float kTiny = 7.8886090522101181e-31f;   // 2^-100

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (BF16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = h2f2(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// rne(x / s) of the exact quotient, |x| <= M s: q is the rounded product with 1/s, and the remainder
// x - q s is exact (s has 24 bits, x at most 11), so comparing it with s/2 settles the last step and
// the ties, which the rounded quotient alone gets wrong next to them.
__device__ __forceinline__ int exact_code(float x, float s, float inv, int top) {
  constexpr float kMagic = 12582912.f;   // 1.5 * 2^23: adding it rounds to the nearest integer
  float q = __fmaf_rn(x, inv, kMagic) - kMagic;
  const float r = __fmaf_rn(-q, s, x);
  const float half = 0.5f * s;
  if (fabsf(r) >= half) {
    const bool odd = (static_cast<int>(q) & 1) != 0;
    if (r > half || (r == half && odd)) q += 1.f;
    if (r < -half || (r == -half && odd)) q -= 1.f;
  }
  return max(-top, min(top, static_cast<int>(q)));
}

__device__ __forceinline__ int first_token(const QuantParams& P, int b) {
  return P.positions ? P.positions[b] : P.position;
}

template <int FMT, bool BF16>
__global__ void __launch_bounds__(kQuantThreads)
kv_quantize_kernel(const __grid_constant__ QuantParams P) {
  const int lane16 = threadIdx.x & 15;
  const int which = blockIdx.y;
  const long long total = (long long)P.caches * P.n_rows * P.heads;
  const long long stride = (long long)gridDim.x * (kQuantThreads / 16);
  unsigned char* codes = which ? P.cache.v : P.cache.k;
  float* scales = which ? P.cache.v_scale : P.cache.k_scale;
  const unsigned char* src = static_cast<const unsigned char*>(P.rows[which]);
  // every lane of a warp takes the same number of turns: the two rows of a warp share its shuffles
  const long long first = (long long)blockIdx.x * (kQuantThreads / 16) + (threadIdx.x >> 4);
  const long long warp_first = first - ((threadIdx.x >> 4) & 1);
  for (long long wr = warp_first, r = first; wr < total; wr += stride, r += stride) {
    bool live = r < total;
    const long long rr = live ? r : total - 1;
    const int h = (int)(rr % P.heads);
    const long long bt = rr / P.heads;
    const int t = (int)(bt % P.n_rows), b = (int)(bt / P.n_rows);
    if (P.counts && t >= P.counts[b]) live = false;
    const long long tok = (long long)first_token(P, b) + t;
    if (tok < 0 || tok >= P.cache.n_tokens) {
      if (live && lane16 == 0 && h == 0) atomicOr(P.status, kStatusBadToken);
      live = false;
    }
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live)
      unpack8<BF16>(ldg128_nc(src + 2 * (b * P.rb[which] + t * P.rt[which] + h * P.rh[which]) + 16 * lane16), x);
    // the largest magnitude by its bits, which infinities and NaN win
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    if (FMT != kCacheInt4) {
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 4));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 8));
    }
    if (!live) continue;
    const float amax = __uint_as_float(top);
    const bool bad = top >= 0x7f800000u;
    const bool zero = amax < kTiny;
    const bool dead = bad || zero;
    float s;
    unsigned char* dst = codes + b * P.cache.bstride + tok * P.cache.tstride + h * P.cache.hstride;
    if (FMT == kCacheFp8) {
      // 448 = 1.75 * 2^8: amax = m * 2^e needs 2^(e-8), one more where m > 1.75
      int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
      s = __uint_as_float((uint32_t)(e + 127) << 23);
      const float inv = dead ? 0.f : __uint_as_float((uint32_t)(127 - e) << 23);
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        uint16_t p;
        const float lo = dead ? 0.f : x[i] * inv, hi = dead ? 0.f : x[i + 1] * inv;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p) : "f"(hi), "f"(lo));
        w[i >> 2] |= (uint32_t)p << (8 * (i & 2));
      }
      *reinterpret_cast<uint2*>(dst + 8 * lane16) = make_uint2(w[0], w[1]);
    } else {
      constexpr int kTop = FMT == kCacheInt8 ? 127 : 7;
      s = __fdiv_rn(amax, (float)kTop);
      const float inv = dead ? 0.f : __frcp_rn(s);
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = dead ? 0 : exact_code(x[i], s, inv, kTop);
        if (FMT == kCacheInt8)
          w[i >> 2] |= (uint32_t)(c & 255) << (8 * (i & 3));
        else
          w[0] |= (uint32_t)(c + 8) << (4 * i);
      }
      if (FMT == kCacheInt8)
        *reinterpret_cast<uint2*>(dst + 8 * lane16) = make_uint2(w[0], w[1]);
      else
        *reinterpret_cast<uint32_t*>(dst + 4 * lane16) = w[0];
    }
    if (bad) s = __uint_as_float(0x7fc00000u);
    else if (zero) s = 0.f;
    constexpr int kScales = cache_row_scales(FMT);
    float* sp = scales + b * P.cache.sbstride + h * P.cache.shstride + tok * kScales;
    if (kScales == 1 ? lane16 == 0 : (lane16 & 3) == 0) sp[kScales == 1 ? 0 : lane16 >> 2] = s;
  }
}

template <int FMT, bool BF16>
__global__ void __launch_bounds__(kQuantThreads)
kv_dequantize_kernel(const __grid_constant__ QuantParams P) {
  const int lane16 = threadIdx.x & 15;
  const int which = blockIdx.y;
  const long long total = (long long)P.caches * P.n_rows * P.heads;
  const long long stride = (long long)gridDim.x * (kQuantThreads / 16);
  const unsigned char* codes = which ? P.cache.v : P.cache.k;
  const float* scales = which ? P.cache.v_scale : P.cache.k_scale;
  unsigned char* out = static_cast<unsigned char*>(P.rows[which]);
  constexpr int kScales = cache_row_scales(FMT);
  for (long long r = (long long)blockIdx.x * (kQuantThreads / 16) + (threadIdx.x >> 4); r < total; r += stride) {
    const int h = (int)(r % P.heads);
    const long long bt = r / P.heads;
    const int t = (int)(bt % P.n_rows), b = (int)(bt / P.n_rows);
    const long long tok = (long long)first_token(P, b) + t;
    uint4 res = make_uint4(0u, 0u, 0u, 0u);
    if (tok >= 0 && tok < P.cache.n_tokens) {
      const unsigned char* src = codes + b * P.cache.bstride + tok * P.cache.tstride + h * P.cache.hstride;
      const float s = scales[b * P.cache.sbstride + h * P.cache.shstride + tok * kScales +
                             (kScales == 1 ? 0 : lane16 >> 2)];
      float x[8];
      if (FMT == kCacheInt4) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(src + 4 * lane16);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)((int)((w >> (4 * i)) & 15u) - 8) * s;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(src + 8 * lane16);
        const uint32_t w[2] = {u.x, u.y};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (FMT == kCacheInt8) {
            x[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * s;
          } else if ((i & 1) == 0) {
            uint32_t p;
            const uint16_t pair = (uint16_t)(w[i >> 2] >> (8 * (i & 2)));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(p) : "h"(pair));
            const float2 f = h2f2(p);
            x[i] = f.x * s;
            x[i + 1] = f.y * s;
          }
        }
      }
      res = make_uint4(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]),
                       pack2<BF16>(x[6], x[7]));
    } else if (lane16 == 0 && h == 0) {
      atomicOr(P.status, kStatusBadToken);
    }
    *reinterpret_cast<uint4*>(out + 2 * (b * P.rb[which] + t * P.rt[which] + h * P.rh[which]) + 16 * lane16) = res;
  }
}

namespace {

int quant_grid(const QuantParams& P) {
  const long long rows = (long long)P.caches * P.n_rows * P.heads;
  const long long blocks = (rows + kQuantThreads / 16 - 1) / (kQuantThreads / 16);
  return (int)(blocks < 148 * 16 ? blocks : 148 * 16);
}

template <int FMT>
cudaError_t launch_one(const QuantParams& P, bool bf16, bool back, cudaStream_t stream) {
  const dim3 grid(quant_grid(P), 2);
  note_launch();
  if (back) {
    if (bf16) kv_dequantize_kernel<FMT, true><<<grid, kQuantThreads, 0, stream>>>(P);
    else kv_dequantize_kernel<FMT, false><<<grid, kQuantThreads, 0, stream>>>(P);
  } else {
    if (bf16) kv_quantize_kernel<FMT, true><<<grid, kQuantThreads, 0, stream>>>(P);
    else kv_quantize_kernel<FMT, false><<<grid, kQuantThreads, 0, stream>>>(P);
  }
  return cudaGetLastError();
}

cudaError_t launch_format(const QuantParams& P, int format, bool bf16, bool back, cudaStream_t stream) {
  switch (format) {
    case kCacheInt8: return launch_one<kCacheInt8>(P, bf16, back, stream);
    case kCacheFp8: return launch_one<kCacheFp8>(P, bf16, back, stream);
    default: return launch_one<kCacheInt4>(P, bf16, back, stream);
  }
}

}  // namespace

cudaError_t launch_kv_quantize(const QuantParams& P, int format, bool bf16, cudaStream_t stream) {
  return launch_format(P, format, bf16, false, stream);
}
cudaError_t launch_kv_dequantize(const QuantParams& P, int format, bool bf16, cudaStream_t stream) {
  return launch_format(P, format, bf16, true, stream);
}

}  // namespace ra
