// Decode attention over one segment (a prefix shared by the batch, or each row's own cache) in any
// of the cache formats, and the joining of the segments' partials.
//
// A tile of 64 tokens arrives by TMA in a ring of stages; four consumer warps take 16 tokens each.
// Both products run on the tensor cores with the tokens (then the dims) as the 16 rows of
// m16n8k16 and the queries as its 8 columns, so that a group of up to 8 query heads costs one MMA
// where the other orientation would pad it to 16:
//     S^T[token, query] = K Q^T          O^T[dim, query] += V^T P^T
// Codes become fp16 (every int8, e4m3 and int4 code is exact in it) in registers on the way to the
// MMA and are multiplied as they are; the scales stay outside in fp32: a token's K scale multiplies its
// scores, its V scale (relative to the largest seen, a power of two) its weights.  int4 has a scale for
// each 32 dims: the scores of the four groups are accumulated apart, and the weights multiplied once
// for each group.  K's dims may go through the MMA in any order, so a lane takes them as they lie in
// 16 (int4: 4) bytes of a row; V's dims come out in the order the lanes hold them.
//
// The running maximum moves only when a score exceeds it by 2^4 (a vote, no reduction).  Weights are
// exp2(score - maximum + 10), at most 2^14 (2^15 with a V scale): fp32 sums do not mind.  For the product
// they are split into a 16-bit value and the 16-bit rest of it, which takes two MMAs: fp16 (bf16 for a bf16
// cache) alone would add an error of the size of the result's own rounding, both parts leave 2^-21 (2^-15)
// of a weight, and fp16's least number 2^-35 of the largest weight times the largest V scale.  The second MMA
// costs fp8 and 16-bit caches up to 2 %, int8 up to 9 % (113 against 104 us for 8 x 32768 tokens on 384 CTAs), int4
// 13 % (365 against 322 us for 1 Mi tokens).
// Bytes bound it where arithmetic does not: 512 per token and kv head in 16 bits, 264 in 8, 160 in 4.  16
// rows behind 131072 fp16 tokens of 32 heads take 330 us (2.17 GB at 6.6 TB/s, the copy rate); 8 x 32768
// tokens of 8 heads take 100 to 107 us in int8 (5.2 to 5.5 TB/s), where turning codes into fp16 keeps the integer
// pipe busy 60 % of the time, and 94 in fp8 (5.9); 1 Mi tokens of 8 heads take 365 us in int4 (3.7 TB/s), with no
// pipe above 53 % and 2.4 instructions a clock.
// Three CTAs of 160 threads to a multiprocessor: with four (96 registers) registers spill, and what then took
// 105 us in int8 and 411 in int4 took 111 and 525.
#include "cache_attend.cuh"

#include "api_host.cuh"

namespace ra {

template <int NQ>
struct AttendCtrl {
  uint64_t full[kAttendMaxStages];
  uint64_t empty[kAttendMaxStages];
  long long before;                 // tiles before cache `start`
  long long total;
  long long sums[kAttendThreads / 32 + 1];
  float m[kAttendWarps][8 * NQ];
  float l[kAttendWarps][8 * NQ];
  float c[kAttendWarps];
  int start;
  int timeout;
};
constexpr int kMergePitch = 68;     // floats of one query's half row in the merge buffer
constexpr int kMergeBytes = kAttendWarps * 8 * kMergePitch * 4;
// Where fp32 holds scores no finer than 1/8, the maximum is not lifted: 10 less may be 16 less after rounding.
constexpr float kLazyLog2 = 4.f, kLiftLog2 = 10.f, kFarLog2 = 1048576.f;

__device__ __forceinline__ void attend_consumer_sync() {
  asm volatile("bar.sync 1, %0;" ::"r"(32 * kAttendWarps) : "memory");
}
__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF16>
__device__ __forceinline__ void mma_any(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16) mma_bf16_16816(d, a, b0, b1);
  else mma_16816(d, a, b0, b1);
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// asynchronous copy of 4 or 16 bytes, or as many zeros
template <int BYTES>
__device__ __forceinline__ void cp_async_zfill(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(live ? BYTES : 0)
               : "memory");
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  uint32_t r;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  uint16_t r;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ uint32_t hsub2_bits(uint32_t a, uint32_t b) {
  __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}

// Two pairs of fp16 codes out of the four bytes of a word, (0,2) and (1,3) for int8: a byte with its
// sign bit flipped, put into the low mantissa bits of 1024.0, is 1024 + 128 + code.  e4m3: (0,1) and
// (2,3) by the hardware's conversion.
template <int FMT>
__device__ __forceinline__ void codes_of(uint32_t w, uint32_t& first, uint32_t& second) {
  if (FMT == kCacheInt8) {
    first = hsub2_bits((w & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u);
    second = hsub2_bits(((w >> 8) & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u);
  } else {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(first), "=r"(second)
        : "r"(w));
  }
}
// A pair of weights as 16-bit values and the 16-bit rests of them.  FINITE: they meet codes, which are finite;
// both parts are rounded to nearest.  Otherwise the value is cut off a little below the weight, so that neither
// part of a weight that counts is zero or negative: zero times an infinity of V would make a NaN of it.
template <bool BF16, bool FINITE>
__device__ __forceinline__ void split_pair(float lo, float hi, uint32_t& value, uint32_t& rest) {
  constexpr float kBelow = 0.99999904632568359375f;     // 1 - 2^-20
  float2 y;
  if (FINITE) {
    value = pack_pair<BF16>(lo, hi);
  } else if (BF16) {
    value = __byte_perm(__float_as_uint(lo * kBelow), __float_as_uint(hi * kBelow), 0x7632);
  } else {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(value) : "f"(hi * kBelow), "f"(lo * kBelow));
  }
  if (BF16) y = make_float2(__uint_as_float(value << 16), __uint_as_float(value & 0xffff0000u));
  else y = h2f2(value);
  rest = pack_pair<BF16>(lo - y.x, hi - y.y);
}
// The same pairs of an int8 word as fp16 subnormals of (code + 128) 2^-24: for the scores, whose sum of q
// times 128 goes into the accumulators beforehand.  (For the values it would not do: their long sums
// would lose in the difference.)
__device__ __forceinline__ void int8_raw(uint32_t w, uint32_t& first, uint32_t& second) {
  first = (w & 0x00ff00ffu) ^ 0x00800080u;
  second = ((w >> 8) & 0x00ff00ffu) ^ 0x00800080u;
}
// Nibbles (i, i + 4) of a word hold code + 8.  raw: as they are, an fp16 subnormal of (code + 8) 2^-24,
// the odd ones 16 times that; otherwise exact codes, the odd ones 16 times.
__device__ __forceinline__ uint32_t nibbles_raw(uint32_t w, int i) {
  return (i < 2 ? w : w >> 8) & ((i & 1) ? 0x00f000f0u : 0x000f000fu);
}
__device__ __forceinline__ uint32_t nibbles_of(uint32_t w, int i) {
  return (i & 1) ? hsub2_bits(nibbles_raw(w, i) | 0x64006400u, 0x64806480u)
                 : hsub2_bits(nibbles_raw(w, i) | 0x64006400u, 0x64086408u);
}

// My part of one work row: tiles [first, first + count) of (cache b, kv head h, query tile qt), and the
// units of the line that it stands for.
struct AttendRow {
  int b, inner, h, qt, len, first, count, units;
};

constexpr float kNoMax = -3e38f;    // below every score that counts, and finite: no special cases

template <int FMT, bool BF16, int NQ>
__global__ void __launch_bounds__(kAttendThreads, attend_ctas(NQ))
cache_attend_kernel(const __grid_constant__ CacheAttendParams P) {
  constexpr bool kDense = FMT <= kCacheBf16;
  constexpr bool kPBf16 = kDense && BF16;           // type of the weights in the product
  constexpr int kHalf = kAttendTile * 128;          // one swizzled [64 tokens][128 bytes] block
  constexpr int kKBytes = kAttendTile * cache_row_bytes(FMT);
  constexpr int kStage = 2 * kKBytes;
  constexpr int kNS = kDense ? 1 : cache_row_scales(FMT);
  constexpr int kScaleFloats = attend_scale_floats(FMT);
  constexpr int QT = 8 * NQ;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const AttendSegment& G = P.seg;
  const int S = G.nstages;
  float* sm_sc = reinterpret_cast<float*>(smem + (size_t)S * kStage);  // [stages][K, V][64 tokens][scales]
  float* sm_o = sm_sc + S * kScaleFloats;                               // [4 warps][8 queries][68]
  AttendCtrl<NQ>* ctrl = reinterpret_cast<AttendCtrl<NQ>*>(reinterpret_cast<unsigned char*>(sm_o) + kMergeBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per_cache = P.hkv * G.query_tiles;

  if (tid == 0) {
    tma_prefetch_desc(&G.kmap);
    tma_prefetch_desc(&G.vmap);
    for (int s = 0; s < S; ++s) {
      mbar_init(&ctrl->full[s], kDense ? 1 : 33);      // the TMA's arrival and each lane's scales
      mbar_init(&ctrl->empty[s], kAttendWarps);
    }
    ctrl->timeout = 0;
    fence_barrier_init();
  }
  // a call's first kernel is launched while the one before it still runs, and touches no memory before this
  if (!P.after) asm volatile("griddepcontrol.wait;" ::: "memory");
  auto length_of = [&](int b) {
    int len = G.cache.n_tokens;
    if (G.lens) len = max(0, min(len, G.lens[b]));
    return len;
  };
  auto units_of_length = [](int len) { return len > 0 ? ceil_div(len, kAttendTile) + kAttendRowUnits : 0; };
  auto units_of = [&](int b) { return units_of_length(length_of(b)); };

  // ---- my share of the line.  Equal lengths need a division; otherwise every thread sums a run of
  // caches and a block-wide scan does the rest.
  if (!G.lens) {
    const long long n = units_of(0), all = n * G.caches * per_cache, ctas = min((long long)G.grid, all);
    if (tid == 0) {
      ctrl->total = n * G.caches;
      ctrl->start = blockIdx.x < ctas ? (int)(all * blockIdx.x / ctas / (n * per_cache)) : 0;
      ctrl->before = ctrl->start * n;
    }
  } else {
    const int run = ceil_div(G.caches, kAttendThreads);
    const int lo = min(G.caches, tid * run), hi = min(G.caches, lo + run);
    long long mine = 0;
    for (int b = lo; b < hi; ++b) {
      mine += units_of(b);
      if (blockIdx.x == 0 && (G.lens[b] < 0 || G.lens[b] > G.cache.n_tokens)) atomicOr(P.status, kStatusBadToken);
    }
    long long incl = mine;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, incl, i);
      if (lane >= i) incl += o;
    }
    if (lane == 31) ctrl->sums[warp] = incl;
    __syncthreads();
    long long base = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kAttendThreads / 32; ++w) {
      if (w < warp) base += ctrl->sums[w];
      total += ctrl->sums[w];
    }
    long long at = base + incl - mine;          // units of one (kv head, query tile) before cache lo
    const long long all = total * per_cache;
    const long long ctas = min((long long)G.grid, all);   // every one of them has a unit
    const long long first = blockIdx.x < ctas ? all * blockIdx.x / ctas : all;
    for (int b = lo; b < hi; ++b) {
      const int n = units_of(b);
      if (first >= at * per_cache && first < (at + n) * per_cache) {
        ctrl->start = b;
        ctrl->before = at;
      }
      at += n;
    }
    if (tid == 0) ctrl->total = total;
  }
  __syncthreads();
  // lets the next kernel start its launch; it waits for this grid's end before it reads
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const long long total = ctrl->total * per_cache;
  const long long ctas = min((long long)G.grid, total);
  if (blockIdx.x >= ctas) {
    if (P.after) asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const long long t0 = total * blockIdx.x / ctas, t1 = total * (blockIdx.x + 1) / ctas;
  int left = (int)(t1 - t0);          // units of mine in this row and behind it

  // r's units from `pos` on, of which n are mine or behind
  auto take = [&](AttendRow& r, int pos, int n) {
    r.units = min(n, units_of_length(r.len) - pos);
    r.first = max(0, pos - kAttendRowUnits);
    r.count = max(0, pos + r.units - kAttendRowUnits - r.first);
  };
  AttendRow row;
  {
    row.b = ctrl->start;
    row.len = length_of(row.b);
    const int units = units_of_length(row.len);
    const long long off = t0 - ctrl->before * per_cache;
    row.inner = (int)(off / units);
    row.h = row.inner / G.query_tiles;
    row.qt = row.inner % G.query_tiles;
    take(row, (int)(off % units), left);
  }
  // the row behind `r`, of which n > 0 units are mine or behind
  auto row_behind = [&](AttendRow r, int n) {
    ++r.inner;
    if (++r.qt == G.query_tiles) {
      r.qt = 0;
      ++r.h;
    }
    if (r.inner == per_cache) {
      r.inner = r.h = r.qt = 0;
      do r.len = length_of(++r.b);
      while (r.len == 0);
    }
    take(r, 0, n);
    return r;
  };

  if (warp == kAttendWarps) {
    // ---------------------------------------------------------------- producer warp
    // lane 0 starts the TMA copies; all lanes fetch the scales, which would otherwise come one tile
    // ahead at most and pay the memory's loaded latency for every tile
    int s = 0, issued = 0;
    unsigned parity = 1;          // of the phase before the first: an unused stage is free
    bool ok = true;
    while (ok) {
      const long long sbase = (long long)row.b * G.cache.sbstride + (long long)row.h * G.cache.shstride;
      for (int i = 0; ok && i < row.count; ++i) {
        ok = __all_sync(0xffffffffu, mbar_wait(&ctrl->empty[s], parity, &ctrl->timeout));
        if (!ok) break;
        unsigned char* dst = smem + (size_t)s * kStage;
        const int tok = (row.first + i) * kAttendTile;
        if (lane == 0) {
          mbar_expect_tx(&ctrl->full[s], kStage);
          if (kDense) {
            tma_load_4d(dst, &G.kmap, &ctrl->full[s], 0, row.h, tok, row.b);
            tma_load_4d(dst + kHalf, &G.kmap, &ctrl->full[s], 64, row.h, tok, row.b);
            tma_load_4d(dst + 2 * kHalf, &G.vmap, &ctrl->full[s], 0, row.h, tok, row.b);
            tma_load_4d(dst + 3 * kHalf, &G.vmap, &ctrl->full[s], 64, row.h, tok, row.b);
          } else {
            tma_load_4d(dst, &G.kmap, &ctrl->full[s], 0, row.h, tok, row.b);
            tma_load_4d(dst + kKBytes, &G.vmap, &ctrl->full[s], 0, row.h, tok, row.b);
          }
        }
        if (!kDense) {
          const uint32_t sc = smem_u32(sm_sc + s * kScaleFloats);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int t = lane + 32 * (j & 1);      // token of the tile; K for j < 2, then V
            const bool live = tok + t < row.len;    // zeros for the others
            const float* src = ((j >> 1) ? G.cache.v_scale : G.cache.k_scale) + (live ? sbase + (long long)(tok + t) * kNS : 0);
            cp_async_zfill<4 * kNS>(sc + ((j >> 1) * kAttendTile + t) * 4 * kNS, src, live);
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&ctrl->full[s])) : "memory");
        }
        ++issued;
        if (++s == S) {
          s = 0;
          parity ^= 1;
        }
      }
      left -= row.units;
      if (left <= 0) break;
      row = row_behind(row, left);
    }
    if (!ok) {
      // a wait ran out: the consumers carry on, but no copy may still be under way when the CTA ends
      if (lane == 0) atomicOr(P.status, kStatusTimeout);
      asm volatile("cp.async.wait_all;" ::: "memory");
      int own = 0;
      for (int i = max(0, issued - S); i < issued; ++i)
        mbar_wait(&ctrl->full[i % S], (unsigned)((i / S) & 1), &own, kWaitLimitNs / 4);
    }
    if (P.after) asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }

  // ------------------------------------------------------------------ consumer warps
  const int g = lane >> 2, t = lane & 3;
  const int r0 = warp * 16;
  const uint32_t stage0 = smem_u32(smem);
  const int mi = lane >> 3, lr = lane & 7;
  int s = 0;
  unsigned parity = 0;
  for (;;) {
    // ---- one work row
    left -= row.units;
    AttendRow behind = row;
    if (left > 0) behind = row_behind(row, left);
    if (row.count == 0) {             // none of its tiles, only of the units before them
      if (left <= 0) break;
      row = behind;
      continue;
    }
    const int b = row.b, h = row.h, q0 = row.qt * QT, len = row.len;
    const long long slot = (long long)b * per_cache + row.inner + blockIdx.x;
    // B fragments of Q^T: column g is query q0 + 8 nq + g; the dims of lane t in the order K's lanes hold them
    uint32_t qb[NQ][8][2];
    constexpr int kOff = FMT == kCacheInt4 ? 4 : 1;
    float k_off[NQ][kOff][2];
    float fac[NQ][2];      // what turns a raw score of my two columns into the log2 domain
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      const int qi = q0 + 8 * nq + g;
      const bool live = qi < G.queries;
      // of the prefix (one cache) query qi is of batch row qi / group
      const int qrow = live ? (b + qi / P.group) * P.hq + h * P.group + qi % P.group : 0;
      const unsigned char* qp = static_cast<const unsigned char*>(P.q) + (size_t)qrow * kRowBytes;
      if (kDense) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          qb[nq][kk][0] = live ? *reinterpret_cast<const uint32_t*>(qp + 32 * kk + 4 * t) : 0u;
          qb[nq][kk][1] = live ? *reinterpret_cast<const uint32_t*>(qp + 32 * kk + 16 + 4 * t) : 0u;
        }
        fac[nq][0] = fac[nq][1] = P.scale_log2e;
      } else {
        // the row is brought to a magnitude of 1 by a power of two, so that fp16 holds a bf16 row too
        // dims of step kk: int8: bytes (0,2), (1,3) of word kk of my 32 dims; e4m3: bytes (0,1), (2,3);
        // int4: of group kk / 2, nibbles (0,4), (1,5) or (2,6), (3,7) of my word
        float x[32];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 u = live ? *reinterpret_cast<const uint4*>(qp + (FMT == kCacheInt4 ? 64 * i + 16 * t : 64 * t + 16 * i))
                               : make_uint4(0u, 0u, 0u, 0u);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (BF16) {
              x[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
              x[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            } else {
              const float2 f = h2f2(w[j]);
              x[8 * i + 2 * j] = f.x;
              x[8 * i + 2 * j + 1] = f.y;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(x[i]) & 0x7f800000u);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // zeros and rows with an infinity or a NaN stay as they are
        if (top == 0u || top == 0x7f800000u) top = 0x3f800000u;
        top = min(top, 0x7e800000u);
        const float down = __uint_as_float(0x7f000000u - top);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const float* y = FMT == kCacheInt4 ? x + 8 * (kk >> 1) + 2 * (kk & 1) : x + 4 * kk;
          constexpr int i1 = FMT == kCacheInt4 ? 4 : FMT == kCacheInt8 ? 2 : 1;
          constexpr int i2 = FMT == kCacheFp8 ? 2 : 1;
          qb[nq][kk][0] = pack_pair<false>(y[0] * down, y[i1] * down);
          constexpr float kOdd = FMT == kCacheInt4 ? 0.0625f : 1.f;     // K's odd nibbles come 16 times as large
          qb[nq][kk][1] = pack_pair<false>(y[i2] * down * kOdd, y[i2 + i1] * down * kOdd);
        }
        if (FMT != kCacheFp8) {
          // the sum of q (code + bias) less bias times the sum of q: what the accumulators start from
          constexpr int kPer = 32 / kOff;
#pragma unroll
          for (int j = 0; j < kOff; ++j) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < kPer; ++i) sum += x[kPer * j + i];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            sum *= down * (FMT == kCacheInt4 ? -8.f / 16777216.f : -128.f / 16777216.f);
            k_off[nq][j][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
            k_off[nq][j][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
          }
        }
        const float up = __uint_as_float(top) * P.scale_log2e * (FMT == kCacheFp8 ? 1.f : 16777216.f);
        fac[nq][0] = __shfl_sync(0xffffffffu, up, 8 * t);
        fac[nq][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
      }
    }
    float o[NQ][8][4];
    float m_ref[NQ][2], l_run[NQ][2];
    float c_ref = 1.1754944e-38f;       // power of two that V scales are taken relative to
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[nq][i][0] = o[nq][i][1] = o[nq][i][2] = o[nq][i][3] = 0.f;
      m_ref[nq][0] = m_ref[nq][1] = kNoMax;
      l_run[nq][0] = l_run[nq][1] = 0.f;
    }

    for (int i_tile = 0; i_tile < row.count; ++i_tile) {
      const int tok0 = (row.first + i_tile) * kAttendTile + r0;     // my 16 tokens
      if (!mbar_wait(&ctrl->full[s], parity, &ctrl->timeout)) {
        if (lane == 0) atomicOr(P.status, kStatusTimeout);
      }
      if (tok0 < len) {
        const uint32_t kbase = stage0 + (uint32_t)s * kStage, vbase = kbase + kKBytes;
        const bool tail = tok0 + 16 > len;
        float ks[2][kNS], vs[2][kNS];     // of tokens g and g + 8 of my 16
        if (!kDense) {
          const float* sc = sm_sc + s * kScaleFloats + (r0 + g) * kNS;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (kNS == 4) {
              const float4 a = *reinterpret_cast<const float4*>(sc + 8 * i * kNS);
              const float4 c = *reinterpret_cast<const float4*>(sc + (kAttendTile + 8 * i) * kNS);
              ks[i][0] = a.x; ks[i][kNS > 1 ? 1 : 0] = a.y; ks[i][kNS > 2 ? 2 : 0] = a.z; ks[i][kNS - 1] = a.w;
              vs[i][0] = c.x; vs[i][kNS > 1 ? 1 : 0] = c.y; vs[i][kNS > 2 ? 2 : 0] = c.z; vs[i][kNS - 1] = c.w;
            } else {
              ks[i][0] = sc[8 * i];
              vs[i][0] = sc[kAttendTile + 8 * i];
            }
          }
        }
        // ---- S^T = K Q^T
        float x[NQ][4];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) x[nq][0] = x[nq][1] = x[nq][2] = x[nq][3] = 0.f;
        if (kDense) {
          const int tk = r0 + (mi & 1) * 8 + lr;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const int c8 = 2 * kk + (mi >> 1);
            uint32_t a[4];
            ldmatrix_x4(a, kbase + (c8 >> 3) * kHalf + tk * 128 + (((c8 & 7) ^ (tk & 7)) << 4));
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) mma_any<kPBf16>(x[nq], a, qb[nq][kk][0], qb[nq][kk][1]);
          }
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[nq][i] *= P.scale_log2e;
        } else if (FMT == kCacheInt4) {
          const int ta = r0 + g, tb = ta + 8;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t wa = lds32(kbase + ta * 64 + ((j ^ ((ta >> 1) & 3)) << 4) + 4 * t);
            const uint32_t wb = lds32(kbase + tb * 64 + ((j ^ ((tb >> 1) & 3)) << 4) + 4 * t);
            float part[NQ][4];
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) {
              part[nq][0] = part[nq][2] = k_off[nq][j % kOff][0];
              part[nq][1] = part[nq][3] = k_off[nq][j % kOff][1];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t a[4] = {nibbles_raw(wa, 2 * i), nibbles_raw(wb, 2 * i), nibbles_raw(wa, 2 * i + 1),
                                     nibbles_raw(wb, 2 * i + 1)};
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq) mma_16816(part[nq], a, qb[nq][2 * j + i][0], qb[nq][2 * j + i][1]);
            }
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
              for (int i = 0; i < 4; ++i) x[nq][i] += part[nq][i] * ks[i >> 1][j < kNS ? j : 0];
          }
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[nq][i] *= fac[nq][i & 1];
        } else {
          const int ta = r0 + g, tb = ta + 8;
          float y[NQ][4];
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq) {
            y[nq][0] = y[nq][1] = y[nq][2] = y[nq][3] = 0.f;
            if (FMT == kCacheInt8) {
              x[nq][0] = x[nq][2] = k_off[nq][0][0];
              x[nq][1] = x[nq][3] = k_off[nq][0][1];
            }
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint4 ua = lds128(kbase + ta * 128 + (((2 * t + half) ^ (ta & 7)) << 4));
            const uint4 ub = lds128(kbase + tb * 128 + (((2 * t + half) ^ (tb & 7)) << 4));
            const uint32_t wa[4] = {ua.x, ua.y, ua.z, ua.w}, wb[4] = {ub.x, ub.y, ub.z, ub.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t a[4];
              if (FMT == kCacheInt8) {
                int8_raw(wa[i], a[0], a[2]);
                int8_raw(wb[i], a[1], a[3]);
              } else {
                codes_of<FMT>(wa[i], a[0], a[2]);
                codes_of<FMT>(wb[i], a[1], a[3]);
              }
              const int kk = 4 * half + i;
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq)
                mma_16816(half ? y[nq] : x[nq], a, qb[nq][kk][0], qb[nq][kk][1]);
            }
          }
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[nq][i] = (x[nq][i] + y[nq][i]) * (ks[i >> 1][0] * fac[nq][i & 1]);
        }
        if (tail) {
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (tok0 + g + 8 * (i >> 1) >= len) x[nq][i] = -INFINITY;
        }
        // ---- the running maximum less the lift; a score has to exceed it by 2^4 to move it
        bool rise = false;
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            rise |= fmaxf(x[nq][i], x[nq][i + 2]) - m_ref[nq][i] > kLazyLog2 + kLiftLog2;
        float c_new = c_ref;
        if (!kDense) {
          float vm = 0.f;
#pragma unroll
          for (int j = 0; j < kNS; ++j) vm = fmaxf(vm, fmaxf(fabsf(vs[0][j]), fabsf(vs[1][j])));
          if (vm >= 2.f * c_ref) {
            c_new = __uint_as_float(min(__float_as_uint(vm) & 0x7f800000u, 0x7e800000u));
            rise = true;
          }
        }
        if (__any_sync(0xffffffffu, rise)) {
          float back = 1.f;
          if (!kDense) {
#pragma unroll
            for (int i = 16; i; i >>= 1) c_new = fmaxf(c_new, __shfl_xor_sync(0xffffffffu, c_new, i));
            back = c_ref / c_new;
            c_ref = c_new;
          }
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float mx = fmaxf(x[nq][i], x[nq][i + 2]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              const float m_new = fmaxf(m_ref[nq][i], fabsf(mx) < kFarLog2 ? mx - kLiftLog2 : mx);
              const float alpha = fast_exp2(m_ref[nq][i] - m_new);
              m_ref[nq][i] = m_new;
              l_run[nq][i] *= alpha;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                o[nq][j][i] *= alpha * back;
                o[nq][j][i + 2] *= alpha * back;
              }
            }
        }
        // ---- weights, scaled by V's scales, as B fragments (tokens along k)
        uint32_t pb[NQ][kNS][2], pr[NQ][kNS][2];
        const float down = kDense ? 1.f : __uint_as_float(0x7f000000u - __float_as_uint(c_ref));
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
          float p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = fast_exp2(x[nq][i] - m_ref[nq][i & 1]);
          l_run[nq][0] += p[0] + p[2];
          l_run[nq][1] += p[1] + p[3];
#pragma unroll
          for (int j = 0; j < kNS; ++j) {
            const float f0 = kDense ? 1.f : vs[0][j] * down, f1 = kDense ? 1.f : vs[1][j] * down;
            uint32_t a, ar, c, cr;
            split_pair<kPBf16, !kDense>(p[0] * f0, p[1] * f0, a, ar);
            split_pair<kPBf16, !kDense>(p[2] * f1, p[3] * f1, c, cr);
            pb[nq][j][0] = movmatrix_trans(a);
            pb[nq][j][1] = movmatrix_trans(c);
            pr[nq][j][0] = movmatrix_trans(ar);
            pr[nq][j][1] = movmatrix_trans(cr);
          }
        }
        // ---- O^T += V^T P^T
        // values behind the length may be anything, and a weight of zero does not hide an infinity or a
        // NaN: they are cut out of the fragments (int8 and int4 codes are always finite)
        const int seen = len - tok0;
        const uint32_t k0 = !tail ? 0xffffffffu : (2 * t < seen ? 0xffffu : 0u) | (2 * t + 1 < seen ? 0xffff0000u : 0u);
        const uint32_t k1 = !tail ? 0xffffffffu : (2 * t + 8 < seen ? 0xffffu : 0u) | (2 * t + 9 < seen ? 0xffff0000u : 0u);
        if (kDense) {
          const int tv = r0 + (mi >> 1) * 8 + lr;
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            const int c8 = 2 * mt + (mi & 1);
            uint32_t a[4];
            ldmatrix_x4_trans(a, vbase + (c8 >> 3) * kHalf + tv * 128 + (((c8 & 7) ^ (tv & 7)) << 4));
            if (tail) {
              a[0] &= k0; a[1] &= k0; a[2] &= k1; a[3] &= k1;
            }
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) {
              mma_any<kPBf16>(o[nq][mt], a, pb[nq][0][0], pb[nq][0][1]);
              mma_any<kPBf16>(o[nq][mt], a, pr[nq][0][0], pr[nq][0][1]);
            }
          }
        } else if (FMT == kCacheInt4) {
          // lane g: dims 32 j + 4 g .. + 3 of group j, two bytes of a token
          const int ta = r0 + 2 * t;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int tk = ta + 8 * i;    // even: tk and tk + 1 have the same swizzle
              const uint32_t at = vbase + tk * 64 + ((j ^ ((tk >> 1) & 3)) << 4) + 2 * g;
              w[i] = lds16(at) | (lds16(at + 64) << 16);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t a[4] = {nibbles_of(w[0], 2 * i), nibbles_of(w[0], 2 * i + 1), nibbles_of(w[1], 2 * i),
                                     nibbles_of(w[1], 2 * i + 1)};
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq) {
                mma_16816(o[nq][2 * j + i], a, pb[nq][j < kNS ? j : 0][0], pb[nq][j < kNS ? j : 0][1]);
                mma_16816(o[nq][2 * j + i], a, pr[nq][j < kNS ? j : 0][0], pr[nq][j < kNS ? j : 0][1]);
              }
            }
          }
        } else {
          // lane g: dims 16 g .. 16 g + 15; tile mt takes bytes 2 mt and 2 mt + 1
          const int ta = r0 + 2 * t;
          uint4 u[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tk = ta + (i & 1) + 8 * (i >> 1);
            u[i] = lds128(vbase + tk * 128 + ((g ^ (tk & 7)) << 4));
          }
          const uint32_t w[4][4] = {{u[0].x, u[0].y, u[0].z, u[0].w}, {u[1].x, u[1].y, u[1].z, u[1].w},
                                    {u[2].x, u[2].y, u[2].z, u[2].w}, {u[3].x, u[3].y, u[3].z, u[3].w}};
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            // bytes 2 mt and 2 mt + 1 of both tokens, paired as codes_of takes them
            const uint32_t sel = FMT == kCacheInt8 ? ((mt & 1) ? 0x7632u : 0x5410u) : ((mt & 1) ? 0x7362u : 0x5140u);
            uint32_t a[4];
            codes_of<FMT>(__byte_perm(w[0][mt >> 1], w[1][mt >> 1], sel), a[0], a[1]);
            codes_of<FMT>(__byte_perm(w[2][mt >> 1], w[3][mt >> 1], sel), a[2], a[3]);
            if (FMT == kCacheFp8 && tail) {
              a[0] &= k0; a[1] &= k0; a[2] &= k1; a[3] &= k1;
            }
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) {
              mma_16816(o[nq][mt], a, pb[nq][0][0], pb[nq][0][1]);
              mma_16816(o[nq][mt], a, pr[nq][0][0], pr[nq][0][1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctrl->empty[s]);
      if (++s == S) {
        s = 0;
        parity ^= 1;
      }
    }

    // ---- merge the warps' partials and leave them in the row's slot
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float l = l_run[nq][i];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (g == 0) {
          ctrl->m[warp][8 * nq + 2 * t + i] = m_ref[nq][i];
          ctrl->l[warp][8 * nq + 2 * t + i] = l;
        }
      }
    attend_consumer_sync();
    if (tid == 0) {
      // the first and the last CTA with tiles of this row say so
      int* span = G.span + 2 * ((long long)b * per_cache + row.inner);
      if (row.first == 0) span[0] = blockIdx.x;
      if ((row.first + row.count) * kAttendTile >= len) span[1] = blockIdx.x;
    }
    if (tid < QT) {
      float m = kNoMax, l = 0.f;
#pragma unroll
      for (int w = 0; w < kAttendWarps; ++w) m = fmaxf(m, ctrl->m[w][tid]);
#pragma unroll
      for (int w = 0; w < kAttendWarps; ++w) l += ctrl->l[w][tid] * fast_exp2(ctrl->m[w][tid] - m);
      float* ml = G.part_ml + (slot * QT + tid) * 2;
      ml[0] = m;
      ml[1] = l;
    }
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      float f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int qi = 8 * nq + 2 * t + i;
        float m = kNoMax;
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) m = fmaxf(m, ctrl->m[w][qi]);
        f[i] = fast_exp2(m_ref[nq][i] - m);
        if (!kDense) f[i] *= c_ref;
      }
      // dims of the accumulators: 16-bit: 16 mt + g (+ 8); 8 bits: 16 g + 2 mt (+ 1); 4 bits: of group
      // mt / 2: 4 g + 2 (mt & 1) (+ 1).  One half of the dims after the other through the buffer.
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (nq || half) attend_consumer_sync();
        float* dst = sm_o + (warp * 8) * kMergePitch;
        if (FMT == kCacheInt8 || FMT == kCacheFp8) {
          if ((g >> 2) == half) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int mt = 0; mt < 8; ++mt)
                *reinterpret_cast<float2*>(dst + (2 * t + i) * kMergePitch + 16 * (g & 3) + 2 * mt) =
                    make_float2(o[nq][mt][i] * f[i], o[nq][mt][i + 2] * f[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int m4 = 0; m4 < 4; ++m4) {
              const int mt = 4 * half + m4;
              float* p = dst + (2 * t + i) * kMergePitch;
              if (FMT == kCacheInt4) {
                *reinterpret_cast<float2*>(p + 32 * (m4 >> 1) + 4 * g + 2 * (m4 & 1)) =
                    make_float2(o[nq][mt][i] * f[i], o[nq][mt][i + 2] * (f[i] * 0.0625f));   // odd nibble
              } else {
                p[16 * m4 + g] = o[nq][mt][i] * f[i];
                p[16 * m4 + g + 8] = o[nq][mt][i + 2] * f[i];
              }
            }
        }
        attend_consumer_sync();
        // 8 queries x 64 dims: 128 threads, one float4 each
        const int qi = tid >> 4, d4 = tid & 15;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) {
          const float4 v = *reinterpret_cast<const float4*>(sm_o + (w * 8 + qi) * kMergePitch + 4 * d4);
          sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        *reinterpret_cast<float4*>(G.part_o + ((slot * QT + 8 * nq + qi) * kHeadDim + 64 * half + 4 * d4)) = sum;
      }
    }
    if (left <= 0) break;
    row = behind;
    attend_consumer_sync();   // the buffers are reused by the next row
  }
  // a kernel that waits for this one's end then has everything before it too
  if (P.after) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Joins the partials of both segments for one (row, head): weights by the common maximum, sums in
// slot order (the same bits every time), zeros where nothing was seen.  A warp takes up to 32 partials
// at once: a lane for the maximum and weight of each, then four dims per lane.  WARPS warps share the
// partials of a row where rows are few, or each has a row of its own.
constexpr int kCombineWarps = 8;

template <bool BF16, int WARPS>
__global__ void __launch_bounds__(32 * kCombineWarps)
cache_combine_kernel(const __grid_constant__ CombineParams P) {
  __shared__ float4 sm_sum[kCombineWarps][32];
  __shared__ float2 sm_ml[kCombineWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long r = (long long)blockIdx.x * (kCombineWarps / WARPS) + warp / WARPS;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the next call's first kernel, which waits too
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (r >= (long long)P.batch * P.hq) return;
  const int b = (int)(r / P.hq), hq = (int)(r % P.hq), h = hq / P.group;
  // the partials of either segment that are mine: [at, at + n) of the slots, strided by a row's query tile
  long long at[2];
  int n[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const CombineSegment& G = P.seg[i];
    at[i] = 0;
    n[i] = 0;
    if (!G.part_o) continue;
    const int cache = G.prefix ? 0 : b;
    if (G.lens && G.lens[cache] <= 0) continue;
    const int qi = hq % P.group + (G.prefix ? b * P.group : 0);
    const long long row = (long long)cache * P.hkv * G.query_tiles + h * G.query_tiles + qi / G.qt;
    const int2 span = G.splits ? make_int2(0, G.splits - 1) : *reinterpret_cast<const int2*>(G.span + 2 * row);
    const int parts = span.y - span.x + 1, per = (parts + WARPS - 1) / WARPS, mine = per * (warp % WARPS);
    at[i] = ((G.splits ? row * G.splits : row) + span.x + mine) * G.qt + qi % G.qt;
    n[i] = max(0, min(per, parts - mine));
  }
  // maxima and weights of the first 32 of both under way together
  float2 ml[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    ml[i] = make_float2(kNoMax, 0.f);
    if (lane < n[i]) ml[i] = *reinterpret_cast<const float2*>(P.seg[i].part_ml + 2 * (at[i] + (long long)lane * P.seg[i].qt));
  }
  float m = fmaxf(ml[0].x, ml[1].x), w = 0.f;
#pragma unroll
  for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const CombineSegment& G = P.seg[i];
    for (int c = 0; c < n[i]; c += 32) {
      if (c) {           // a row of more than 32 partials to a warp: one long context alone
        ml[i] = make_float2(kNoMax, 0.f);
        if (c + lane < n[i]) ml[i] = *reinterpret_cast<const float2*>(G.part_ml + 2 * (at[i] + (long long)(c + lane) * G.qt));
        float top = fmaxf(m, ml[i].x);
#pragma unroll
        for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        const float keep = fast_exp2(m - top);
        m = top;
        w *= keep;
        sum.x *= keep; sum.y *= keep; sum.z *= keep; sum.w *= keep;
      }
      const float f = fast_exp2(ml[i].x - m);
      w += ml[i].y * f;              // of this lane's partials; summed over the lanes at the end
      const float* src = G.part_o + (at[i] + (long long)c * G.qt) * kHeadDim + 4 * lane;
      const int here = min(32, n[i] - c);
#pragma unroll 8
      for (int k = 0; k < here; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(src + (long long)k * G.qt * kHeadDim);
        const float fk = __shfl_sync(0xffffffffu, f, k);
        sum.x += v.x * fk; sum.y += v.y * fk; sum.z += v.z * fk; sum.w += v.w * fk;
      }
    }
  }
#pragma unroll
  for (int k = 16; k; k >>= 1) w += __shfl_xor_sync(0xffffffffu, w, k);
  if (WARPS > 1) {
    sm_sum[warp][lane] = sum;
    if (lane == 0) sm_ml[warp] = make_float2(m, w);
    __syncthreads();
    if (warp) return;
    m = kNoMax;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) m = fmaxf(m, sm_ml[k].x);
    w = 0.f;
    sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      const float f = fast_exp2(sm_ml[k].x - m);
      const float4 v = sm_sum[k][lane];
      w += sm_ml[k].y * f;
      sum.x += v.x * f; sum.y += v.y * f; sum.z += v.z * f; sum.w += v.w * f;
    }
  }
  const float inv = w == 0.f ? 0.f : 1.f / w;
  const uint2 u = make_uint2(pack_pair<BF16>(sum.x * inv, sum.y * inv), pack_pair<BF16>(sum.z * inv, sum.w * inv));
  *reinterpret_cast<uint2*>(static_cast<unsigned char*>(P.out) + (size_t)r * kRowBytes + 8 * lane) = u;
}

namespace {
int stage_bytes(int format) { return 2 * kAttendTile * cache_row_bytes(format); }
}  // namespace

// Three CTAs of a multiprocessor share 228 KiB, or two.
int cache_attend_stages(int format, int nq) {
  const int n = (nq == 1 ? 65536 : 98304) / (stage_bytes(format) + 4 * attend_scale_floats(format));
  return n < kAttendMaxStages ? n : kAttendMaxStages;
}

namespace {

template <int FMT, bool BF16, int NQ>
cudaError_t launch_one(const CacheAttendParams& P, cudaStream_t stream) {
  auto kern = cache_attend_kernel<FMT, BF16, NQ>;
  const size_t smem = (size_t)P.seg.nstages * (stage_bytes(FMT) + 4 * attend_scale_floats(FMT)) + kMergeBytes + sizeof(AttendCtrl<NQ>) + 1024;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = allow_smem(kern, smem, done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)P.seg.grid);
  cfg.blockDim = dim3(kAttendThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = P.early ? 1 : 0;
  note_launch();
  return cudaLaunchKernelEx(&cfg, kern, P);
}

template <int FMT>
cudaError_t launch_format(const CacheAttendParams& P, bool bf16, int nq, cudaStream_t stream) {
  if (bf16) return nq == 1 ? launch_one<FMT, true, 1>(P, stream) : launch_one<FMT, true, 2>(P, stream);
  return nq == 1 ? launch_one<FMT, false, 1>(P, stream) : launch_one<FMT, false, 2>(P, stream);
}

}  // namespace

cudaError_t launch_cache_attend(const CacheAttendParams& P, int format, bool bf16, int nq, cudaStream_t stream) {
  switch (format) {
    case kCacheFp16:
      return nq == 1 ? launch_one<kCacheFp16, false, 1>(P, stream) : launch_one<kCacheFp16, false, 2>(P, stream);
    case kCacheBf16:
      return nq == 1 ? launch_one<kCacheBf16, true, 1>(P, stream) : launch_one<kCacheBf16, true, 2>(P, stream);
    case kCacheInt8: return launch_format<kCacheInt8>(P, bf16, nq, stream);
    case kCacheFp8: return launch_format<kCacheFp8>(P, bf16, nq, stream);
    default: return launch_format<kCacheInt4>(P, bf16, nq, stream);
  }
}

cudaError_t launch_cache_combine(const CombineParams& P, bool bf16, cudaStream_t stream) {
  // launched while the attention kernel before it still runs; it waits for that kernel's end itself
  const long long rows = (long long)P.batch * P.hq;
  const bool share = rows <= 1024;      // up to about one wave of CTAs with all their warps on one row
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(share ? rows : (rows + kCombineWarps - 1) / kCombineWarps));
  cfg.blockDim = dim3(32 * kCombineWarps);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  if (share)
    return bf16 ? cudaLaunchKernelEx(&cfg, cache_combine_kernel<true, kCombineWarps>, P)
                : cudaLaunchKernelEx(&cfg, cache_combine_kernel<false, kCombineWarps>, P);
  return bf16 ? cudaLaunchKernelEx(&cfg, cache_combine_kernel<true, 1>, P)
              : cudaLaunchKernelEx(&cfg, cache_combine_kernel<false, 1>, P);
}

}  // namespace ra
