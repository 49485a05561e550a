// Attention of all batch rows' queries over the prefix that they share, on the 5th-generation tensor
// cores: with R = batch * group queries for every key of a kv head the work is two matrix products,
//     S = Q K^T   [128 queries x 128 tokens]        O += P V   [128 queries x 128 dims]
// bound by arithmetic from about 256 queries on and by the keys' bytes below.
//
// A CTA takes one kv head, up to two tiles of 128 queries and a range of the tokens.  It runs two
// streams, each with its own S and O in TMEM and its own softmax warpgroup, so that the tensor cores
// work on one while the other's softmax runs.  With two query tiles both streams walk the same K/V
// tiles; with one, they take the tiles in turn and join their sums at the end.
//   warp 0      TMA: K and V tiles of 32 KiB in one ring
//   warps 1, 2  one thread of each issues a stream's MMAs; its commits release tiles and hand over S
//   warps 12-15 for 8-bit caches: codes into fp16 or bf16 tiles, and the scales beside them; a token's K
//               scale multiplies its column of S, its V scale its column of P, both in fp32
//   warps 4-11  softmax: a thread owns one query (one TMEM lane), so maximum and sum need no exchange;
//               P goes back into S's columns as the A operand of the second product
// The maximum moves only when a score exceeds it by 2^4, and only then O is rescaled in TMEM; no wait
// is needed for that: S(k) is committed after O's product k-1.  Weights go through the product as a value of V's
// type and, in the other half of S's columns, the rest of it in the same type, so that the result's own rounding
// is the only one that counts.
//
// 256 batch rows x 32 heads behind 32768 bf16 tokens of 8 kv heads: 185 us for this kernel, 0.74 PFLOP/s of the
// formula's operations and half as many again for the rests, with the tensor pipe at 63 %: a pair of steps takes
// about 4750 cycles, two thirds of them products, and what bounds it is each stream's chain of S, maximum, exponentials
// (about 1300 cycles for 128 x 128 on the 16 results a clock of the special-function unit), rests and O.  Without
// the rests it took 134-150 us, and then a share of the exponentials on the FMA pipe changed nothing and handing P
// over in four parts instead of two made it slower (170 against 149 us).
// With 128 queries and 16385 int8 tokens it takes about 35 us, with no pipe above 23 %: one query tile leaves each
// stream one stage for K and one for V, so the conversion of codes, the products and the softmax follow one another.
#include "prefix_attend.cuh"

#include "api_host.cuh"

namespace ra {

// Dense tiles go straight from TMA to the MMAs.  8-bit codes pass a warpgroup that turns them into tiles
// of fp16 or bf16, which hold every code exactly.
__host__ __device__ constexpr int pf_stages(bool codes) { return codes ? 3 : 5; }      // of 32 KiB, one more where
                                                                   // only one query tile is held
constexpr int kCodeStages = 3;                                     // of 16 KiB
constexpr int kCodeBytes = kPrefixTile * 128;
constexpr int kScaleTiles = 4;                                     // tiles whose scales are kept
__host__ __device__ constexpr int pf_threads(bool codes) { return codes ? 512 : 384; }
// registers: the softmax's 256 threads take over what the others give up
//   dense: 256 * 232 + 128 * 40 = 384 * 168     codes: 256 * 184 + 128 * 40 + 128 * 104 = 512 * 128
__host__ __device__ constexpr int pf_soft_regs(bool codes) { return codes ? 184 : 232; }
constexpr int kPfOtherRegs = 40, kPfConvertRegs = 104;
constexpr int kPrefixEarly = 64;                // tokens of P whose product starts while the rest is computed
// Quarter of P after which the other stream's turn at the exponentials begins.  At the sizes above a whole call takes
// 230 to 233 us with this quarter, the one before it or the last.
constexpr int kPrefixYield = 2;
// From kPfFar on fp32 holds scores no finer than 1/8: the maximum is not lifted there, since 10 less may be 16 less
// after rounding.
constexpr float kPfFar = 1048576.f, kPfLazy = 4.f, kPfLift = 10.f, kPfNoMax = -3e38f, kPfLeastScale = -60.f;

struct PrefixScales {
  float k[kScaleTiles][kPrefixTile];    // times the score scale
  float v[kScaleTiles][kPrefixTile];
  float top[kScaleTiles][4];            // largest |v| of 32 tokens
};
struct PrefixCtrl {
  uint64_t full[6], empty[6], code_full[kCodeStages], code_empty[kCodeStages], scales_full[kScaleTiles];
  uint64_t q_full, s_full[2], p_full[2][2], o_full[2], turn[2], drain[2];
  uint32_t tmem;
  int timeout;
};

// ---- tcgen05 wrappers (cta_group::1)
__device__ __forceinline__ void tc_alloc512(uint32_t* dst) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(dst)) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_free512(uint32_t tmem) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
#define RA_TC_R8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
#define RA_TC_W8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
// 32 consecutive columns of this thread's lane
__device__ __forceinline__ void tc_ld32(uint32_t* v, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : RA_TC_W8(v, 0), RA_TC_W8(v, 8), RA_TC_W8(v, 16), RA_TC_W8(v, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::RA_TC_R8(v, 0),
      RA_TC_R8(v, 8), RA_TC_R8(v, 16), RA_TC_R8(v, 24), "r"(addr)
      : "memory");
}

__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::RA_TC_R8(v, 0),
      RA_TC_R8(v, 8), "r"(addr)
      : "memory");
}

// two fp32 operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Shared-memory matrix descriptor, 128-byte swizzle.  Rows along K (Q, K tiles): groups of 8 rows are
// 1024 bytes apart, the leading offset is not used.  Rows along the other dimension (V as [token][dim],
// 64 dims to a row): the leading offset leads to the next 64 dims, the stride to the next 8 tokens.
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t leading, uint32_t stride) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(stride >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// Instruction descriptor of kind::f16: fp32 accumulators, 128 x 128.
__device__ __forceinline__ constexpr uint32_t tc_idesc(bool bf16, bool b_mn_major) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn_major ? 1u : 0u) << 16) |
         ((128u >> 3) << 17) | ((128u >> 4) << 24);
}

template <bool BF16>
__device__ __forceinline__ uint32_t pf_pack(float lo, float hi) {
  uint32_t r;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// A pair of weights as 16-bit values and the 16-bit rests of them.  FINITE: they meet codes, which are finite;
// both parts are rounded to nearest.  Otherwise the value is cut off a little below the weight, so that neither
// part of a weight that counts is zero or negative: zero times an infinity of V would make a NaN of it.
template <bool BF16, bool FINITE>
__device__ __forceinline__ void pf_split(float2 x, uint32_t& value, uint32_t& rest) {
  if (FINITE) {
    value = pf_pack<BF16>(x.x, x.y);
  } else {
    const float2 y = mul2(x, make_float2(0.99999904632568359375f, 0.99999904632568359375f));   // 1 - 2^-20
    if (BF16) value = __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x7632);
    else asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(value) : "f"(y.y), "f"(y.x));
  }
  const float2 z = BF16 ? make_float2(__uint_as_float(value << 16), __uint_as_float(value & 0xffff0000u)) : h2f2(value);
  rest = pf_pack<BF16>(x.x - z.x, x.y - z.y);
}

// Sixteen codes as eight pairs of fp16 or bf16.
template <int FMT, bool BF16>
__device__ __forceinline__ void pf_codes(const uint4& u, uint32_t (&r)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t lo, hi;
    if (FMT == kCacheInt8) {
      // a byte with its sign bit flipped in the low mantissa bits of 1024.0 is 1024 + 128 + code
      const uint32_t x = w[i] ^ 0x80808080u, bias = 0x64806480u;
      const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
      __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
      __half2 hb = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&bias));
      lo = *reinterpret_cast<uint32_t*>(&ha);
      hi = *reinterpret_cast<uint32_t*>(&hb);
    } else {
      asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
          : "=r"(lo), "=r"(hi)
          : "r"(w[i]));
    }
    if (BF16) {
      const float2 a = h2f2(lo), b = h2f2(hi);
      lo = pf_pack<true>(a.x, a.y);
      hi = pf_pack<true>(b.x, b.y);
    }
    r[2 * i] = lo;
    r[2 * i + 1] = hi;
  }
}

template <int FMT, bool BF16>
__global__ void __launch_bounds__(pf_threads(FMT >= kCacheInt8), 1)
prefix_attend_kernel(const __grid_constant__ PrefixAttendParams P) {
  constexpr bool kCodes = FMT >= kCacheInt8;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sm_q = smem;                                   // two query tiles
  unsigned char* sm_codes = smem + (2 + pf_stages(kCodes)) * kPrefixTileBytes;
  PrefixScales* scales = reinterpret_cast<PrefixScales*>(sm_codes + (kCodes ? kCodeStages * kCodeBytes : 0));
  PrefixCtrl* ctrl = reinterpret_cast<PrefixCtrl*>(reinterpret_cast<unsigned char*>(scales) + (kCodes ? sizeof(PrefixScales) : 0));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // ---- what this CTA works on; splits fastest, so that neighbours stream different tokens
  const int split = blockIdx.x % P.splits, rest = blockIdx.x / P.splits;
  const int h = rest % P.hkv, qt0 = 2 * (rest / P.hkv);
  const bool pair = qt0 + 1 < P.query_tiles;
  // ring of K and V tiles; the second query tile's place is one of them where there is none
  unsigned char* sm_kv = smem + (pair ? 2 : 1) * kPrefixTileBytes;
  const int stages = pf_stages(kCodes) + (pair ? 0 : 1);
  const int all_tiles = ceil_div(P.n_tokens, kPrefixTile);
  const int tile0 = (int)((long long)all_tiles * split / P.splits);
  const int tiles = (int)((long long)all_tiles * (split + 1) / P.splits) - tile0;
  // stream s walks the tiles s, s + 2, .. of one query tile, or all of them for query tile s.  Tiles are
  // loaded in the order of their first use: K of the first `stride` tiles, then V of tile j and K of
  // tile j + stride for each j, as far as there are any.
  const int stride = pair ? 1 : 2;
  // Each stream has stages of its own where it has tiles of its own: a barrier's parity tells two phases
  // apart, so whoever waits for a stage's next load has to have waited for the one before it.
  // Loads of a stream: K of its i-th tile is number 2 i, V number 2 i + 1.
  const int per_stream = pair ? stages : stages / 2;
  auto index_of = [&](int j, int v) { return 2 * (pair ? j : j >> 1) + v; };
  auto stage_of = [&](int j, int v) { return index_of(j, v) % per_stream + (pair ? 0 : (j & 1) * per_stream); };
  auto round_of = [&](int j, int v) { return (index_of(j, v) / per_stream) & 1; };

  if (tid == 0) {
    tma_prefetch_desc(&P.kmap);
    tma_prefetch_desc(&P.vmap);
    for (int s = 0; s < stages; ++s) {
      mbar_init(&ctrl->full[s], kCodes ? 128 : 1);
      mbar_init(&ctrl->empty[s], pair ? 2 : 1);
    }
    for (int s = 0; s < kCodeStages; ++s) {
      mbar_init(&ctrl->code_full[s], 1);
      mbar_init(&ctrl->code_empty[s], 128);
    }
    for (int s = 0; s < kScaleTiles; ++s) mbar_init(&ctrl->scales_full[s], 128);
    mbar_init(&ctrl->q_full, 256);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&ctrl->s_full[s], 1);
      mbar_init(&ctrl->p_full[s][0], 128);
      mbar_init(&ctrl->p_full[s][1], 128);
      mbar_init(&ctrl->o_full[s], 1);
      mbar_init(&ctrl->turn[s], 128);
      mbar_init(&ctrl->drain[s], 1);
    }
    ctrl->timeout = 0;
    fence_barrier_init();
  }
  if (warp == 1) tc_alloc512(&ctrl->tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // nothing of the kernels before is touched before this; and what is launched after this one, which may
  // not wait for it, must not start before it has passed
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = ctrl->tmem;
  // TMEM columns of stream st: S at 128 st, P in its first half; O at 256 + 128 st
  // false: a wait ran out, here or elsewhere in the CTA; the role that sees it stops
  auto wait = [&](uint64_t* bar, unsigned parity) {
    if (mbar_wait(bar, parity, &ctrl->timeout)) return true;
    atomicOr(P.status, kStatusTimeout);
    return false;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPfOtherRegs));
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- TMA
      constexpr int kBytes = kCodes ? kCodeBytes : kPrefixTileBytes;
      int n = 0;                                     // loads so far
      auto load = [&](int tile, int v) {
        const int st = kCodes ? n % kCodeStages : stage_of(tile, v);
        const unsigned round = kCodes ? (n / kCodeStages) & 1 : round_of(tile, v);
        uint64_t* full = kCodes ? &ctrl->code_full[st] : &ctrl->full[st];
        if (!wait(kCodes ? &ctrl->code_empty[st] : &ctrl->empty[st], round ^ 1)) return false;
        unsigned char* dst = (kCodes ? sm_codes : sm_kv) + st * kBytes;
        const CUtensorMap* map = v ? &P.vmap : &P.kmap;
        const int tok = (tile0 + tile) * kPrefixTile;
        mbar_expect_tx(full, kBytes);
        tma_load_4d(dst, map, full, 0, h, tok, 0);
        if (!kCodes) tma_load_4d(dst + kPrefixHalf, map, full, 64, h, tok, 0);
        ++n;
        return true;
      };
      bool ok = true;
      for (int j = -stride; ok && j < tiles; ++j) {
        if (j >= 0) ok = load(j, 1);
        if (ok && j + stride < tiles) ok = load(j + stride, 0);
      }
      // after a wait that ran out: no load may still be under way when the CTA ends
      if (!ok) {
        int own = 0, i = 0;
        auto settle = [&](int tile, int v) {
          if (i < n && i + 6 >= n)                   // of the loads that may be under way
            mbar_wait(kCodes ? &ctrl->code_full[i % kCodeStages] : &ctrl->full[stage_of(tile, v)],
                      kCodes ? (i / kCodeStages) & 1 : round_of(tile, v), &own, kWaitLimitNs / 8);
          ++i;
        };
        for (int j = -stride; i < n && j < tiles; ++j) {
          if (j >= 0) settle(j, 1);
          if (j + stride < tiles) settle(j + stride, 0);
        }
      }
    } else if (warp == 1 || warp == 2) {
      // ---------------------------------------------------------------- MMA, stream warp - 1
      // The whole warp walks the steps, so that descriptors and addresses are uniform values; one
      // elected thread issues.  (From a branch of one lane every MMA took about 100 cycles to issue, and
      // with one warp for both streams each stream waited for the other's issue.)
      constexpr uint32_t kIdS = tc_idesc(BF16, false), kIdO = tc_idesc(BF16, true);
      const int st = warp - 1;
      const uint32_t tm_s = __shfl_sync(0xffffffffu, tmem, 0) + 128u * st, tm_o = tm_s + 256u;
      const uint64_t q_desc = tc_desc(smem_u32(sm_q) + (pair ? st * kPrefixTileBytes : 0), 16, 1024);
      const uint64_t k_desc = tc_desc(smem_u32(sm_kv), 16, 1024);
      const uint64_t v_desc = tc_desc(smem_u32(sm_kv), kPrefixHalf, 1024);
      auto ready = [&](int j, int v) { return wait(&ctrl->full[stage_of(j, v)], round_of(j, v)); };
      auto scores = [&](int j) {
        const int s = stage_of(j, 0);
        const uint64_t b = k_desc + (uint64_t)(s * (kPrefixTileBytes >> 4));
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint64_t off = ((k >> 2) * kPrefixHalf + (k & 3) * 32) >> 4;
            tc_mma_ss(tm_s, q_desc + off, b + off, kIdS, k > 0);
          }
          tc_commit(&ctrl->empty[s]);
          tc_commit(&ctrl->s_full[st]);
        }
        __syncwarp();
      };
      int j = pair ? 0 : st;
      bool ok = wait(&ctrl->q_full, 0) && (j >= tiles || ready(j, 0));
      if (ok && j < tiles) scores(j);
      for (unsigned k = 0; ok && j < tiles; j += stride, ++k) {
        // the tiles first, so that the products follow one another once P is there
        const bool more = j + stride < tiles;
        ok = ready(j, 1) && (!more || ready(j + stride, 0));
        const int s = stage_of(j, 1);
        const uint64_t b = v_desc + (uint64_t)(s * (kPrefixTileBytes >> 4));
        ok = ok && wait(&ctrl->p_full[st][0], k & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t add = k > 0;
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < kPrefixEarly / 16; ++c) {
            tc_mma_ts(tm_o, tm_s + 8 * c, b + (uint64_t)(c * 2048 >> 4), kIdO, c > 0 ? 1u : add);
            tc_mma_ts(tm_o, tm_s + 64 + 8 * c, b + (uint64_t)(c * 2048 >> 4), kIdO, 1u);
          }
        }
        __syncwarp();
        ok = wait(&ctrl->p_full[st][1], k & 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int c = kPrefixEarly / 16; c < 8; ++c) {
            tc_mma_ts(tm_o, tm_s + 8 * c, b + (uint64_t)(c * 2048 >> 4), kIdO, 1u);
            tc_mma_ts(tm_o, tm_s + 64 + 8 * c, b + (uint64_t)(c * 2048 >> 4), kIdO, 1u);
          }
          tc_commit(&ctrl->empty[s]);
          if (!more) tc_commit(&ctrl->o_full[st]);
        }
        __syncwarp();
        if (more) scores(j + stride);
      }
      if (!ok) {   // no product may still be under way when TMEM is given back
        if (elect_one()) tc_commit(&ctrl->drain[st]);
        __syncwarp();
        int own = 0;
        mbar_wait(&ctrl->drain[st], 0, &own, kWaitLimitNs / 4);
      }
    }
    __syncwarp();
  } else if (kCodes && warp >= 12) {
    // ---------------------------------------------------------------- codes into tiles: a thread per token
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPfConvertRegs));
    const int t = tid - 384;
    const long long at = (long long)h * P.scale_hstride + (long long)tile0 * kPrefixTile + t;
    const int left = P.n_tokens - tile0 * kPrefixTile - t;       // tokens from mine on
    auto scale = [](const float* p) { return __uint_as_float(ld32(p)); };
    float ks = left > 0 ? scale(P.k_scale + at) : 0.f, vs = left > 0 ? scale(P.v_scale + at) : 0.f;
    // V of tile j and K of tile j + stride together: one round of waits, one fence
    int n = 0;                                       // code tiles so far
    for (int j = -stride; j < tiles; ++j) {
      const int jk = j + stride, sj = jk % kScaleTiles;
      const bool has[2] = {j >= 0, jk < tiles};
      const int tile[2] = {max(j, 0), jk};
      bool go = true;
#pragma unroll
      for (int i = 0, next = n; i < 2; ++i)
        if (has[i]) {
          go = go && wait(&ctrl->code_full[next % kCodeStages], (next / kCodeStages) & 1) &&
               wait(&ctrl->empty[stage_of(tile[i], 1 - i)], round_of(tile[i], 1 - i) ^ 1);
          ++next;
        }
      if (!__all_sync(0xffffffffu, go)) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!has[i]) continue;
        const int c = n++ % kCodeStages;
        const uint32_t src = smem_u32(sm_codes) + c * kCodeBytes + t * 128;
        unsigned char* dst = sm_kv + stage_of(tile[i], 1 - i) * kPrefixTileBytes;
        uint4 u[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) u[d] = lds128(src + ((d ^ (t & 7)) << 4));
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          uint32_t r[8];
          pf_codes<FMT, BF16>(u[d], r);
          *reinterpret_cast<uint4*>(dst + swz128(t, 2 * d)) = make_uint4(r[0], r[1], r[2], r[3]);
          *reinterpret_cast<uint4*>(dst + swz128(t, 2 * d + 1)) = make_uint4(r[4], r[5], r[6], r[7]);
        }
        // only now that the values have been used: with the arrival directly behind the loads 820 of 2000 calls on
        // tiles in L2 gave other results, in this order none of 3000
        mbar_arrive(&ctrl->code_empty[c]);
      }
      fence_proxy_async();
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (has[i]) mbar_arrive(&ctrl->full[stage_of(tile[i], 1 - i)]);
      if (has[1]) {
        // both scales of tile jk.  Their slot of four was tile jk - 4's, whose weights are done: the stage
        // of V of tile jk - stride had V of a tile of jk - 4 or later of the same stream, or K of one after
        // it (of both streams, where both walk all tiles), and was released by a product behind them.
        scales->k[sj][t] = ks * P.scale_log2e;
        scales->v[sj][t] = vs;
        float top = fabsf(vs);
#pragma unroll
        for (int i = 16; i; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
        if (lane == 0) scales->top[sj][t >> 5] = top;
        mbar_arrive(&ctrl->scales_full[sj]);
        const bool next = left > (jk + 1) * kPrefixTile;
        ks = next ? scale(P.k_scale + at + (long long)(jk + 1) * kPrefixTile) : 0.f;
        vs = next ? scale(P.v_scale + at + (long long)(jk + 1) * kPrefixTile) : 0.f;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(pf_soft_regs(kCodes)));
    // ---------------------------------------------------------------- queries into shared memory
    const int st = (warp >> 2) - 1;           // stream
    const int soft = tid - 128;
    {
      // 16 lanes to a row; all of a thread's loads are under way before the first is stored
      const int c = soft & 15, n = pair ? 16 : 8;
      const int first = qt0 * kPrefixTile + (soft >> 4);
      const int step_b = 16 / P.group, step_g = 16 % P.group;
      int qb = first / P.group, qg = first % P.group;
      uint4 u[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        u[i] = make_uint4(0u, 0u, 0u, 0u);
        if (i < n && first + 16 * i < P.queries) {
          const long long row = (long long)qb * P.hq + h * P.group + qg;
          u[i] = ld128(static_cast<const unsigned char*>(P.q) + row * kRowBytes + 16 * c);
        }
        qb += step_b;
        qg += step_g;
        if (qg >= P.group) {
          qg -= P.group;
          ++qb;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = (soft >> 4) + 16 * i;
        if (i < n) *reinterpret_cast<uint4*>(sm_q + (r >> 7) * kPrefixTileBytes + swz128(r & 127, c)) = u[i];
      }
      fence_proxy_async();
      mbar_arrive(&ctrl->q_full);
    }
    // ---------------------------------------------------------------- softmax
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;    // my warp's 32 TMEM lanes
    const uint32_t tms = tmem + 128u * st + lanes, tmo = tms + 256u;
    // the running maximum in units of S (log2 units of codes, whose scale is in K's): its difference to a score is
    // exact where it matters, however large the two are
    const float unit = kCodes ? 1.f : P.scale_log2e, lift = kCodes ? kPfLift : fminf(kPfLift / unit, 1e38f);
    float m_ref = kPfNoMax, l = 0.f;
    int k = 0;
    bool ok = true;
    for (int j = pair ? 0 : st; j < tiles; j += stride, ++k) {
      ok = __all_sync(0xffffffffu, wait(&ctrl->s_full[st], k & 1));
      if (!ok) break;
      tc_fence_after();
      uint32_t s[128];
      tc_ld32(s, tms);
      tc_ld32(s + 32, tms + 32);
      tc_ld32(s + 64, tms + 64);
      tc_ld32(s + 96, tms + 96);
      tc_wait_ld();
      const int sj = j % kScaleTiles;
      if (kCodes) {
        ok = __all_sync(0xffffffffu, wait(&ctrl->scales_full[sj], (j / kScaleTiles) & 1));
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < 128; c += 4) {
          const float4 f = *reinterpret_cast<const float4*>(&scales->k[sj][c]);
          const float2 a = mul2(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), make_float2(f.x, f.y));
          const float2 b = mul2(make_float2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), make_float2(f.z, f.w));
          s[c] = __float_as_uint(a.x);
          s[c + 1] = __float_as_uint(a.y);
          s[c + 2] = __float_as_uint(b.x);
          s[c + 3] = __float_as_uint(b.y);
        }
      }
      const int valid = P.n_tokens - (tile0 + j) * kPrefixTile;
      if (valid < kPrefixTile) {
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if (c >= valid) s[c] = 0xff800000u;
      }
      float mx4[4] = {kPfNoMax, kPfNoMax, kPfNoMax, kPfNoMax};
#pragma unroll
      for (int c = 0; c < 128; c += 8)
#pragma unroll
        for (int d = 0; d < 4; ++d)
          mx4[d] = max3(mx4[d], __uint_as_float(s[c + d]), __uint_as_float(s[c + d + 4]));
      float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      const bool far = !(fabsf(mx) * unit < kPfFar);
      if (kCodes) {
        // the weights are multiplied by V's scales: the reference counts their largest in, and since sums
        // and weights share the reference, it drops out in the end.  No less than 2^-60 of it: a weight is at most
        // 2^(14 + 60) then, and 2^31 of them, of rows that are all zeros, are still a finite sum
        const float top = fmaxf(fmaxf(scales->top[sj][0], scales->top[sj][1]), fmaxf(scales->top[sj][2], scales->top[sj][3]));
        if (!far) mx += fmaxf(kPfLeastScale, (float)((int)(__float_as_uint(top) >> 23) - 126));
      }
      if (__any_sync(0xffffffffu, (mx - m_ref) * unit > kPfLazy + kPfLift)) {
        const float m_new = fmaxf(m_ref, far ? mx : mx - lift), alpha = fast_exp2((m_ref - m_new) * unit);
        m_ref = m_new;
        l *= alpha;
        if (k) {
#pragma unroll 1
          for (int c = 0; c < 128; c += 32) {
            uint32_t o[32];
            tc_ld32(o, tmo + c);
            tc_wait_ld();
#pragma unroll
            for (int d = 0; d < 32; ++d) o[d] = __float_as_uint(__uint_as_float(o[d]) * alpha);
            tc_st32(tmo + c, o);
          }
        }
      }
      // the streams take turns at the exponentials: left alone they fall into step, and then the
      // tensor cores idle while both compute, and the other way round
      if (st ? true : k > 0) ok = __all_sync(0xffffffffu, wait(&ctrl->turn[st], (st ? k : k - 1) & 1));
      if (!ok) break;
      const float2 scale2 = make_float2(P.scale_log2e, P.scale_log2e), neg_m = make_float2(-m_ref, -m_ref);
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int part = 0; part < 4; ++part) {
        uint32_t p[16], rest[16];
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          const int e = 32 * part + 2 * c;
          float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
          if (kCodes) f = *reinterpret_cast<const float4*>(&scales->v[sj][e]);
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            float2 x = make_float2(__uint_as_float(s[e + 2 * d]), __uint_as_float(s[e + 2 * d + 1]));
            x = add2(x, neg_m);
            if (!kCodes) x = mul2(x, scale2);
            x.x = fast_exp2(x.x);
            x.y = fast_exp2(x.y);
            sum[d] = add2(sum[d], x);
            if (kCodes) x = mul2(x, d ? make_float2(f.z, f.w) : make_float2(f.x, f.y));
            pf_split<BF16, kCodes>(x, p[c + d], rest[c + d]);
          }
        }
        tc_st16(tms + 16 * part, p);
        tc_st16(tms + 64 + 16 * part, rest);
        if (part == kPrefixYield) mbar_arrive(&ctrl->turn[st ^ 1]);
        if (part == kPrefixEarly / 32 - 1 || part == 3) {
          tc_wait_st();
          tc_fence_before();
          mbar_arrive(&ctrl->p_full[st][part == 3]);
        }
      }
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    }
    // ---------------------------------------------------------------- partial
    m_ref = fmaxf(m_ref * unit, kPfNoMax);
    const int qt = pair ? qt0 + st : qt0;
    const long long slot = ((long long)h * P.query_tiles + qt) * P.splits + split;
    const int row0 = (warp & 3) * 32;                      // my warp's rows
    const int live = P.queries - qt * kPrefixTile - row0;  // of them, how many are queries
    float* out = P.part_o + (slot * kPrefixTile + row0) * kHeadDim;
    if (k && ok) {
      wait(&ctrl->o_full[st], 0);
      __syncwarp();
      tc_fence_after();
    }
    auto stage = [&](uint32_t buf, const uint32_t* o) {    // 32 dims of my row; a row is 128 bytes, swizzled
#pragma unroll
      for (int d = 0; d < 8; ++d)
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(buf + lane * 128 + ((d ^ (lane & 7)) << 4)),
                     "r"(o[4 * d]), "r"(o[4 * d + 1]), "r"(o[4 * d + 2]), "r"(o[4 * d + 3])
                     : "memory");
    };
    if (pair) {
      // 32 rows x 32 dims at a time through the stream's query tile, so that rows leave in whole lines
      const uint32_t buf = smem_u32(sm_q) + st * kPrefixTileBytes + (warp & 3) * 4096;
#pragma unroll 1
      for (int c = 0; c < 128; c += 32) {
        uint32_t o[32];
        tc_ld32(o, tmo + c);
        tc_wait_ld();
        stage(buf, o);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 4 * i + (lane >> 3), d = lane & 7;
          const uint4 v = lds128(buf + r * 128 + ((d ^ (r & 7)) << 4));
          if (r < live) *reinterpret_cast<uint4*>(out + r * kHeadDim + c + 4 * d) = v;
        }
        __syncwarp();
      }
      *reinterpret_cast<float2*>(P.part_ml + (slot * kPrefixTile + row0 + lane) * 2) = make_float2(m_ref, l);
    } else {
      // both streams saw the same queries: their sums are joined here, through the ring, where nothing is
      // under way once both are done
      float2* sm_ml = reinterpret_cast<float2*>(sm_q);     // [2][128]
      asm volatile("bar.sync 2, 256;" ::: "memory");
      sm_ml[st * kPrefixTile + row0 + lane] = make_float2(m_ref, l);
      asm volatile("bar.sync 2, 256;" ::: "memory");
      const float2 other = sm_ml[(st ^ 1) * kPrefixTile + row0 + lane];
      const float top = fmaxf(m_ref, other.x), f = fast_exp2(m_ref - top);
      const uint32_t buf = smem_u32(sm_kv) + (warp & 3) * 16384;   // [4 blocks of 32 dims][32 rows]; stream 1 at + 64 KiB
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        if (k) {
          tc_ld32(o, tmo + 32 * c);
          tc_wait_ld();
#pragma unroll
          for (int d = 0; d < 32; ++d) o[d] = __float_as_uint(__uint_as_float(o[d]) * f);
        } else {
#pragma unroll
          for (int d = 0; d < 32; ++d) o[d] = 0u;
        }
        stage(buf + st * 65536 + c * 4096, o);
      }
      asm volatile("bar.sync 2, 256;" ::: "memory");
      // half of the 32 rows each
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const int c = i & 3, r = 16 * st + 4 * (i >> 2) + (lane >> 3), d = lane & 7;
        const uint32_t at = buf + c * 4096 + r * 128 + ((d ^ (r & 7)) << 4);
        const uint4 x = lds128(at), y = lds128(at + 65536);
        if (r < live)
          *reinterpret_cast<float4*>(out + r * kHeadDim + 32 * c + 4 * d) =
              make_float4(__uint_as_float(x.x) + __uint_as_float(y.x), __uint_as_float(x.y) + __uint_as_float(y.y),
                          __uint_as_float(x.z) + __uint_as_float(y.z), __uint_as_float(x.w) + __uint_as_float(y.w));
      }
      if (st == 0)
        *reinterpret_cast<float2*>(P.part_ml + (slot * kPrefixTile + row0 + lane) * 2) =
            make_float2(top, l * f + other.y * fast_exp2(other.x - top));
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tc_free512(tmem);
}

namespace {

template <int FMT, bool BF16>
cudaError_t launch_one(const PrefixAttendParams& P, cudaStream_t stream) {
  constexpr bool kCodes = FMT >= kCacheInt8;
  auto kern = prefix_attend_kernel<FMT, BF16>;
  const size_t smem = (size_t)(2 + pf_stages(kCodes)) * kPrefixTileBytes +
                      (kCodes ? kCodeStages * kCodeBytes + sizeof(PrefixScales) : 0) + sizeof(PrefixCtrl) + 1024;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = allow_smem(kern, smem, done);
  if (e != cudaSuccess) return e;
  const int blocks = (P.query_tiles + 1) / 2 * P.hkv * P.splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(pf_threads(kCodes));
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

}  // namespace

cudaError_t launch_prefix_attend(const PrefixAttendParams& P, int format, bool bf16, cudaStream_t stream) {
  switch (format) {
    case kCacheFp16: return launch_one<kCacheFp16, false>(P, stream);
    case kCacheBf16: return launch_one<kCacheBf16, true>(P, stream);
    case kCacheInt8: return bf16 ? launch_one<kCacheInt8, true>(P, stream) : launch_one<kCacheInt8, false>(P, stream);
    default: return bf16 ? launch_one<kCacheFp8, true>(P, stream) : launch_one<kCacheFp8, false>(P, stream);
  }
}

}  // namespace ra
