// Quantising key/value rows as they are written into a cache, and reading them back.
//
// One scale s for a row x of 128 values (int8, fp8 e4m3) or for each 32 of them (int4):
//   int8  s = amax / 127     c = rne(x / s)       int4  s = amax / 7, likewise, stored as c + 8
//   fp8   s = 2^k, the least with amax <= 448 s   c = e4m3(x / s), exact but for the one rounding
// and the value read back is c s.  A row (a group) whose largest magnitude is below 2^-100 is stored
// as zeros with s = 0; one that holds an infinity or a NaN is stored with s = NaN, so that it reads
// back as NaN throughout instead of as wrong finite values.
//
// Both kernels are bound by memory: 256 bytes on one side and 132 (80 for int4) on the other for each row.
// 2 x 16384 bf16 rows of 8 heads, K and V, take 66 us into fp8 and back (406 MB moved, 6.1 TB/s), 85 into int8 or
// int4, whose exact quotients cost more.  Eight lanes share a row rather than sixteen: the work on addresses and
// scales halves (77 us with sixteen).
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

// rne(x / s) of the exact quotient, |x| <= amax, in the low bits (two's complement) of the result: q is
// the rounded product with 1/s, got by adding 1.5 * 2^23, which leaves the integer in the low mantissa
// bits.  The remainder x - q s is exact (s has 24 bits, x at most 11), so comparing it with s/2 settles
// the last step and the ties, which the rounded quotient alone gets wrong next to them.  |q| never
// exceeds the format's largest code: amax / s is at most that times 1 + 2^-24.
__device__ __forceinline__ uint32_t exact_code(float x, float s, float inv, float half) {
  constexpr float kMagic = 12582912.f;
  float t = __fmaf_rn(x, inv, kMagic);
  const float r = __fmaf_rn(kMagic - t, s, x);
  if (fabsf(r) >= half) {
    const bool odd = (__float_as_uint(t) & 1u) != 0;
    if (r > half || (r == half && odd)) t += 1.f;
    if (r < -half || (r == -half && odd)) t -= 1.f;
  }
  return __float_as_uint(t);
}

__device__ __forceinline__ int first_token(const QuantParams& P, int b) {
  return P.positions ? P.positions[b] : P.position;
}

// A CTA's rows: tokens [t0, t0 + tile) of cache b, all heads, K (blockIdx.y = 0) or V.  Eight lanes share a
// row, with 16 bytes of either half each; slot w of 32 takes rows w, w + 32, .. , heads fastest, by
// additions only.  The tokens' scales pass through shared memory so that a head's leave, or come, side by
// side.
constexpr int kSlots = kQuantThreads / 8;

struct RowWalk {
  int t, h;
  __device__ RowWalk(int row, int heads) : t(row / heads), h(row % heads) {}
  __device__ void step(int dt, int dh, int heads) {
    t += dt;
    h += dh;
    if (h >= heads) {
      h -= heads;
      ++t;
    }
  }
};

template <int FMT, bool BF16>
__global__ void __launch_bounds__(kQuantThreads)
kv_quantize_kernel(const __grid_constant__ QuantParams P) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ float sm_scale[];               // [heads][tokens][scales of a row]
  constexpr int kScales = cache_row_scales(FMT);
  constexpr int kDeep = 2;                          // rows whose loads are under way together
  const int lane8 = threadIdx.x & 7, which = blockIdx.y, b = blockIdx.z;
  const int t0 = blockIdx.x * P.tile;
  int n = min(P.tile, P.n_rows - t0);
  if (P.counts) n = min(n, max(P.counts[b], 0) - t0);
  const long long first = (long long)first_token(P, b) + t0;   // token of row t0
  if (n > 0 && (first < 0 || first + n > P.cache.n_tokens) && threadIdx.x == 0) atomicOr(P.status, kStatusBadToken);
  if (n <= 0 || first >= P.cache.n_tokens || first + n <= 0) return;
  // tokens outside the cache are left out
  const int lo = first < 0 ? (int)-first : 0, hi = (int)min((long long)n, P.cache.n_tokens - first);
  unsigned char* codes = (which ? P.cache.v : P.cache.k) + b * P.cache.bstride + (first + lo) * P.cache.tstride;
  const unsigned char* src = static_cast<const unsigned char*>(P.rows[which]) +
                             2 * (b * P.rb[which] + (long long)(t0 + lo) * P.rt[which]) + 16 * lane8;
  const int heads = P.heads, tokens = hi - lo, rows = tokens * heads;
  const long long rt = 2 * P.rt[which], rh = 2 * P.rh[which];
  const int slot = threadIdx.x >> 3, dt = kSlots / heads, dh = kSlots % heads;
  RowWalk load(slot, heads), store = load;
  // every lane of a warp takes the same number of turns: its rows share the shuffles
  for (int r0 = 0; r0 < rows; r0 += kDeep * kSlots) {
    uint4 u[kDeep][2];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      u[i][0] = u[i][1] = make_uint4(0u, 0u, 0u, 0u);
      if (r0 + i * kSlots + slot < rows) {
        const unsigned char* at = src + load.t * rt + load.h * rh;
        u[i][0] = ld128(at);
        u[i][1] = ld128(at + 128);
      }
      load.step(dt, dh, heads);
    }
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const bool live = r0 + i * kSlots + slot < rows;
      float x[2][8];
      uint32_t tops[2];          // the largest magnitude by its bits, which infinities and NaN win
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        unpack8<BF16>(u[i][c], x[c]);
        tops[c] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) tops[c] = max(tops[c], __float_as_uint(x[c][j]) & 0x7fffffffu);
      }
      if (FMT != kCacheInt4) tops[0] = max(tops[0], tops[1]);
#pragma unroll
      for (int c = 0; c < (FMT == kCacheInt4 ? 2 : 1); ++c) {
        tops[c] = max(tops[c], __shfl_xor_sync(0xffffffffu, tops[c], 1));
        tops[c] = max(tops[c], __shfl_xor_sync(0xffffffffu, tops[c], 2));
        if (FMT != kCacheInt4) tops[c] = max(tops[c], __shfl_xor_sync(0xffffffffu, tops[c], 4));
      }
      unsigned char* dst = codes + store.t * P.cache.tstride + store.h * P.cache.hstride;
      float* sp = sm_scale + (store.h * tokens + store.t) * kScales;
      float s = 0.f, inv = 0.f;
      bool dead = false;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (c == 0 || FMT == kCacheInt4) {
          const uint32_t top = tops[c];
          const float amax = __uint_as_float(top);
          const bool bad = top >= 0x7f800000u;
          dead = bad || amax < kTiny;
          float keep;
          if (FMT == kCacheFp8) {
            // 448 = 1.75 * 2^8: amax = m * 2^e needs 2^(e-8), one more where m > 1.75
            const uint32_t e = (top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
            s = __uint_as_float(e << 23);
            inv = __uint_as_float((254u - e) << 23);
          } else {
            s = __fdiv_rn(amax, FMT == kCacheInt8 ? 127.f : 7.f);
            inv = __frcp_rn(s);
          }
          keep = dead ? (bad ? __uint_as_float(0x7fc00000u) : 0.f) : s;
          if (live) {
            if (FMT == kCacheInt4) {
              if ((lane8 & 3) == 0) sp[2 * c + (lane8 >> 2)] = keep;
            } else if (lane8 == 0) {
              sp[0] = keep;
            }
          }
        }
        uint32_t w[2] = {0u, 0u};
        if (FMT == kCacheFp8) {
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            uint16_t p;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p) : "f"(x[c][j + 1] * inv), "f"(x[c][j] * inv));
            w[j >> 2] |= (uint32_t)p << (8 * (j & 2));
          }
        } else {
          const float half = 0.5f * s;
          uint32_t q[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) q[j] = exact_code(x[c][j], s, inv, half);
          if (FMT == kCacheInt8) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              w[j] = __byte_perm(__byte_perm(q[4 * j], q[4 * j + 1], 0x0040),
                                 __byte_perm(q[4 * j + 2], q[4 * j + 3], 0x0040), 0x5410);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[0] |= ((q[j] + 8u) & 15u) << (4 * j);
          }
        }
        if (dead) w[0] = w[1] = FMT == kCacheInt4 ? 0x88888888u : 0u;
        if (live) {
          if (FMT == kCacheInt4) *reinterpret_cast<uint32_t*>(dst + 4 * lane8 + 32 * c) = w[0];
          else *reinterpret_cast<uint2*>(dst + 8 * lane8 + 64 * c) = make_uint2(w[0], w[1]);
        }
      }
      store.step(dt, dh, heads);
    }
  }
  __syncthreads();
  float* scales = (which ? P.cache.v_scale : P.cache.k_scale) + b * P.cache.sbstride + (first + lo) * kScales;
  const int run = tokens * kScales, dk = kQuantThreads % run, ds = kQuantThreads / run;
  for (int i = threadIdx.x, h = i / run, k = i % run; i < rows * kScales; i += kQuantThreads) {
    scales[h * P.cache.shstride + k] = sm_scale[i];
    h += ds;
    k += dk;
    if (k >= run) {
      k -= run;
      ++h;
    }
  }
}

// eight values of codes (int4: one word, else two) times their scale
template <int FMT>
__device__ __forceinline__ void values_of(uint2 u, float s, float (&x)[8]) {
  // an integer below 2^23 in the low mantissa bits of 2^23
  if (FMT == kCacheInt4) {
    const uint32_t w[2] = {u.x & 0x0f0f0f0fu, (u.x >> 4) & 0x0f0f0f0fu};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x[j] = (__uint_as_float(__byte_perm(w[j & 1], 0x4b000000u, 0x7650 | (j >> 1))) - 8388616.f) * s;
  } else if (FMT == kCacheInt8) {
    const uint32_t w[2] = {u.x ^ 0x80808080u, u.y ^ 0x80808080u};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x[j] = (__uint_as_float(__byte_perm(w[j >> 2], 0x4b000000u, 0x7650 | (j & 3))) - 8388736.f) * s;
  } else {
    const uint32_t w[2] = {u.x, u.y};
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      uint32_t p;
      const uint16_t pair = (uint16_t)(w[j >> 2] >> (8 * (j & 2)));
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(p) : "h"(pair));
      const float2 f = h2f2(p);
      x[j] = f.x * s;
      x[j + 1] = f.y * s;
    }
  }
}

template <int FMT, bool BF16>
__global__ void __launch_bounds__(kQuantThreads)
kv_dequantize_kernel(const __grid_constant__ QuantParams P) {
  // launched while the kernel before it still runs
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ float sm_scale[];               // [heads][tokens][scales of a row]
  constexpr int kScales = cache_row_scales(FMT);
  constexpr int kDeep = 4;
  const int lane8 = threadIdx.x & 7, which = blockIdx.y, b = blockIdx.z;
  const int t0 = blockIdx.x * P.tile;
  const int n = min(P.tile, P.n_rows - t0);
  const long long first = (long long)first_token(P, b) + t0;
  if ((first < 0 || first + n > P.cache.n_tokens) && threadIdx.x == 0) atomicOr(P.status, kStatusBadToken);
  // tokens of this tile inside the cache; the others read as zeros
  const int lo = (int)max(0ll, min((long long)n, -first)), hi = (int)max(0ll, min((long long)n, P.cache.n_tokens - first));
  const unsigned char* codes = (which ? P.cache.v : P.cache.k) + b * P.cache.bstride + first * P.cache.tstride;
  const float* scales = (which ? P.cache.v_scale : P.cache.k_scale) + b * P.cache.sbstride + first * kScales;
  const int heads = P.heads, run = n * kScales, rows = n * heads;
  const int dk = kQuantThreads % run, ds = kQuantThreads / run;
  for (int i = threadIdx.x, h = i / run, k = i % run; i < rows * kScales; i += kQuantThreads) {
    const int t = k / kScales;
    sm_scale[i] = t >= lo && t < hi ? __uint_as_float(ld32(scales + h * P.cache.shstride + k)) : 0.f;
    h += ds;
    k += dk;
    if (k >= run) {
      k -= run;
      ++h;
    }
  }
  __syncthreads();
  unsigned char* out = static_cast<unsigned char*>(P.rows[which]) +
                       2 * (b * P.rb[which] + (long long)t0 * P.rt[which]) + 16 * lane8;
  const long long rt = 2 * P.rt[which], rh = 2 * P.rh[which];
  const int slot = threadIdx.x >> 3, dt = kSlots / heads, dh = kSlots % heads;
  RowWalk load(slot, heads), store = load;
  for (int r0 = 0; r0 < rows; r0 += kDeep * kSlots) {
    uint2 u[kDeep][2];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      u[i][0] = u[i][1] = make_uint2(FMT == kCacheInt4 ? 0x88888888u : 0u, 0u);
      if (r0 + i * kSlots + slot < rows && load.t >= lo && load.t < hi) {
        const unsigned char* at = codes + load.t * P.cache.tstride + load.h * P.cache.hstride;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (FMT == kCacheInt4) u[i][c].x = ld32(at + 4 * lane8 + 32 * c);
          else u[i][c] = ld64(at + 8 * lane8 + 64 * c);
        }
      }
      load.step(dt, dh, heads);
    }
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      if (r0 + i * kSlots + slot < rows) {
        const float* sp = sm_scale + (store.h * n + store.t) * kScales;
        unsigned char* dst = out + store.t * rt + store.h * rh;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x[8];
          values_of<FMT>(u[i][c], sp[FMT == kCacheInt4 ? 2 * c + (lane8 >> 2) : 0], x);
          *reinterpret_cast<uint4*>(dst + 128 * c) =
              make_uint4(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]), pack2<BF16>(x[6], x[7]));
        }
      }
      store.step(dt, dh, heads);
    }
  }
}

namespace {

// Tokens of a CTA: about 256 rows, so that a padded batch's longest rows still spread over the device,
// but 8 tokens at least (a whole sector of a head's scales) and 32 at most; fewer than 8 only where the
// call is too small to occupy the device.  kQuantMaxHeads keeps the scales within 32 KiB.
int quant_tile(const QuantParams& P) {
  int tile = 32;
  while (tile > 8 && tile * P.heads > 256) tile >>= 1;
  while (tile > 1 && ((long long)P.caches * ((P.n_rows + tile - 1) / tile) * 2 < 2 * 148 ||
                      tile * P.heads > 2 * kQuantMaxHeads))
    tile >>= 1;
  return tile;
}

template <int FMT>
cudaError_t launch_one(QuantParams P, bool bf16, bool back, cudaStream_t stream) {
  P.tile = quant_tile(P);
  const size_t smem = (size_t)P.tile * P.heads * cache_row_scales(FMT) * sizeof(float);
  const dim3 grid((unsigned)((P.n_rows + P.tile - 1) / P.tile), 2, (unsigned)P.caches);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kQuantThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = P.early ? 1 : 0;
  note_launch();
  if (back)
    return bf16 ? cudaLaunchKernelEx(&cfg, kv_dequantize_kernel<FMT, true>, P)
                : cudaLaunchKernelEx(&cfg, kv_dequantize_kernel<FMT, false>, P);
  return bf16 ? cudaLaunchKernelEx(&cfg, kv_quantize_kernel<FMT, true>, P)
              : cudaLaunchKernelEx(&cfg, kv_quantize_kernel<FMT, false>, P);
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
