// Attention of all batch rows' queries over the prefix that they share, on the 5th-generation tensor
// cores: with R = batch * group queries for every key of a kv head the work is two matrix products,
//     S = Q K^T   [128 queries x 128 tokens]        O += P V   [128 queries x 128 dims]
// bound by arithmetic from about 256 queries on and by the keys' bytes below.
//
// A CTA takes one kv head, up to two tiles of 128 queries and a range of the tokens.  It runs two
// streams, each with its own S and O in TMEM and its own softmax warpgroup, so that the tensor cores
// work on one while the other's softmax runs.  With two query tiles both streams walk the same K/V
// tiles; with one, they take the tiles in turn and leave a partial each.
//   warp 0      TMA: K and V tiles of 32 KiB in one ring, in the order of their first use
//   warp 1      one thread issues the MMAs; its commits release tiles and hand over S
//   warps 4-11  softmax: a thread owns one query (one TMEM lane), so maximum and sum need no exchange;
//               P goes back into S's columns as the A operand of the second product
// The maximum moves only when a score exceeds it by 2^4, and only then O is rescaled in TMEM; no wait
// is needed for that: S(k) is committed after O's product k-1.  Weights are rounded to the type of V.
#include "prefix_attend.cuh"

namespace ra {

constexpr int kPrefixStages = 5;
constexpr int kPrefixThreads = 384;
constexpr int kPrefixSoftRegs = 232, kPrefixOtherRegs = 40;   // 256 * 232 + 128 * 40 = 384 * 168
constexpr float kPfLazy = 4.f, kPfLift = 10.f, kPfNoMax = -3e38f;

struct PrefixCtrl {
  uint64_t full[kPrefixStages], empty[kPrefixStages];
  uint64_t q_full, s_full[2], p_full[2], o_full[2];
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

template <bool BF16>
__global__ void __launch_bounds__(kPrefixThreads, 1)
prefix_attend_kernel(const __grid_constant__ PrefixAttendParams P) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sm_q = smem;                                   // two query tiles
  unsigned char* sm_kv = smem + 2 * kPrefixTileBytes;           // ring of K and V tiles
  PrefixCtrl* ctrl = reinterpret_cast<PrefixCtrl*>(sm_kv + kPrefixStages * kPrefixTileBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // ---- what this CTA works on; splits fastest, so that neighbours stream different tokens
  const int split = blockIdx.x % P.splits, rest = blockIdx.x / P.splits;
  const int h = rest % P.hkv, qt0 = 2 * (rest / P.hkv);
  const bool pair = qt0 + 1 < P.query_tiles;
  const int all_tiles = ceil_div(P.n_tokens, kPrefixTile);
  const int tile0 = (int)((long long)all_tiles * split / P.splits);
  const int tiles = (int)((long long)all_tiles * (split + 1) / P.splits) - tile0;
  // step i: stream i & 1, tile i / 2 (two query tiles) or i (one)
  const int steps = pair ? 2 * tiles : tiles;

  if (tid == 0) {
    tma_prefetch_desc(&P.kmap);
    tma_prefetch_desc(&P.vmap);
    for (int s = 0; s < kPrefixStages; ++s) {
      mbar_init(&ctrl->full[s], 1);
      mbar_init(&ctrl->empty[s], 1);
    }
    mbar_init(&ctrl->q_full, 256);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&ctrl->s_full[s], 1);
      mbar_init(&ctrl->p_full[s], 128);
      mbar_init(&ctrl->o_full[s], 1);
    }
    ctrl->timeout = 0;
    fence_barrier_init();
  }
  if (warp == 1) tc_alloc512(&ctrl->tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = ctrl->tmem;
  auto tm_s = [&](int stream) { return tmem + 128u * stream; };          // S, then P in its first half
  auto tm_o = [&](int stream) { return tmem + 256u + 128u * stream; };
  auto wait = [&](uint64_t* bar, unsigned parity) {
    if (!mbar_wait(bar, parity, &ctrl->timeout)) atomicOr(P.status, kStatusTimeout);
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPrefixOtherRegs));
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- TMA
      int n = 0;
      auto load = [&](const CUtensorMap* map, int tile) {
        const int s = n % kPrefixStages;
        wait(&ctrl->empty[s], ((n / kPrefixStages) & 1) ^ 1);
        unsigned char* dst = sm_kv + s * kPrefixTileBytes;
        const int tok = (tile0 + tile) * kPrefixTile;
        mbar_expect_tx(&ctrl->full[s], kPrefixTileBytes);
        tma_load_4d(dst, map, &ctrl->full[s], 0, h, tok, 0);
        tma_load_4d(dst + kPrefixHalf, map, &ctrl->full[s], 64, h, tok, 0);
        ++n;
      };
      load(&P.kmap, 0);
      if (!pair && steps > 1) load(&P.kmap, 1);
      for (int i = 0; i < steps; ++i) {
        const bool fresh = !pair || !(i & 1);
        const int j = pair ? i >> 1 : i, ahead = pair ? j + 1 : j + 2;
        if (fresh) load(&P.vmap, j);
        if (fresh && ahead < tiles) load(&P.kmap, ahead);
      }
    } else if (warp == 1 && lane == 0) {
      // ---------------------------------------------------------------- MMA
      constexpr uint32_t kIdS = tc_idesc(BF16, false), kIdO = tc_idesc(BF16, true);
      int n = 0, ks = 0, vs = 0;
      const uint32_t kv = smem_u32(sm_kv), sq = smem_u32(sm_q);
      auto take = [&]() {
        const int s = n % kPrefixStages;
        wait(&ctrl->full[s], (n / kPrefixStages) & 1);
        ++n;
        return s;
      };
      auto scores = [&](int i) {
        const bool fresh = !pair || !(i & 1);
        if (fresh) ks = take();
        tc_fence_after();
        const uint32_t a = sq + (pair ? (i & 1) * kPrefixTileBytes : 0), b = kv + ks * kPrefixTileBytes;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = (k >> 2) * kPrefixHalf + (k & 3) * 32;
          tc_mma_ss(tm_s(i & 1), tc_desc(a + off, 16, 1024), tc_desc(b + off, 16, 1024), kIdS, k > 0);
        }
        if (!pair || (i & 1)) tc_commit(&ctrl->empty[ks]);
        tc_commit(&ctrl->s_full[i & 1]);
      };
      wait(&ctrl->q_full, 0);
      scores(0);
      if (steps > 1) scores(1);
      for (int i = 0; i < steps; ++i) {
        if (!pair || !(i & 1)) vs = take();
        wait(&ctrl->p_full[i & 1], (i >> 1) & 1);
        tc_fence_after();
        const uint32_t b = kv + vs * kPrefixTileBytes;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          tc_mma_ts(tm_o(i & 1), tm_s(i & 1) + 8 * k, tc_desc(b + k * 2048, kPrefixHalf, 1024), kIdO, i > 1 || k > 0);
        if (!pair || (i & 1)) tc_commit(&ctrl->empty[vs]);
        if (i + 2 >= steps) tc_commit(&ctrl->o_full[i & 1]);
        if (i + 2 < steps) scores(i + 2);
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPrefixSoftRegs));
    // ---------------------------------------------------------------- queries into shared memory
    const int st = (warp >> 2) - 1;           // stream
    const int soft = tid - 128;
    {
      const int rows = pair ? 256 : 128;
      const int c = soft & 15;
#pragma unroll 4
      for (int r = soft >> 4; r < rows; r += 16) {
        const int qi = qt0 * kPrefixTile + r;
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (qi < P.queries) {
          const long long row = (long long)(qi / P.group) * P.hq + h * P.group + qi % P.group;
          u = *reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(P.q) + row * kRowBytes + 16 * c);
        }
        *reinterpret_cast<uint4*>(sm_q + (r >> 7) * kPrefixTileBytes + swz128(r & 127, c)) = u;
      }
      fence_proxy_async();
      mbar_arrive(&ctrl->q_full);
    }
    // ---------------------------------------------------------------- softmax
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;    // my warp's 32 TMEM lanes
    const uint32_t tms = tm_s(st) + lanes, tmo = tm_o(st) + lanes;
    float m_ref = kPfNoMax, l = 0.f;
    int k = 0;
    for (int i = st; i < steps; i += 2, ++k) {
      wait(&ctrl->s_full[st], k & 1);
      tc_fence_after();
      uint32_t s[128];
      tc_ld32(s, tms);
      tc_ld32(s + 32, tms + 32);
      tc_ld32(s + 64, tms + 64);
      tc_ld32(s + 96, tms + 96);
      tc_wait_ld();
      const int tile = tile0 + (pair ? i >> 1 : i);
      const int valid = P.n_tokens - tile * kPrefixTile;
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
          mx4[d] = fmaxf(mx4[d], fmaxf(__uint_as_float(s[c + d]), __uint_as_float(s[c + d + 4])));
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * P.scale_log2e;
      if (__any_sync(0xffffffffu, mx > m_ref + (kPfLazy + kPfLift))) {
        const float m_new = fmaxf(m_ref, mx - kPfLift), alpha = fast_exp2(m_ref - m_new);
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
      float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t p[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float a = fast_exp2(__fmaf_rn(__uint_as_float(s[64 * half + 2 * c]), P.scale_log2e, -m_ref));
          const float b = fast_exp2(__fmaf_rn(__uint_as_float(s[64 * half + 2 * c + 1]), P.scale_log2e, -m_ref));
          l4[(2 * c) & 3] += a;
          l4[(2 * c + 1) & 3] += b;
          p[c] = pf_pack<BF16>(a, b);
        }
        tc_st32(tms + 32 * half, p);
      }
      l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&ctrl->p_full[st]);
    }
    // ---------------------------------------------------------------- partial
    const int qt = pair ? qt0 + st : qt0;
    const long long slot = ((long long)h * P.query_tiles + qt) * (2 * P.splits) + (pair ? split : 2 * split + st);
    const int row = (warp & 3) * 32 + lane;
    float* out = P.part_o + (slot * kPrefixTile + row) * kHeadDim;
    if (k) {
      wait(&ctrl->o_full[st], 0);
      tc_fence_after();
    }
#pragma unroll
    for (int c = 0; c < 128; c += 32) {
      uint32_t o[32];
      if (k) {
        tc_ld32(o, tmo + c);
        tc_wait_ld();
      } else {
#pragma unroll
        for (int d = 0; d < 32; ++d) o[d] = 0u;
      }
      if (qt * kPrefixTile + row < P.queries) {
#pragma unroll
        for (int d = 0; d < 32; d += 4)
          *reinterpret_cast<uint4*>(out + c + d) = make_uint4(o[d], o[d + 1], o[d + 2], o[d + 3]);
      }
    }
    float* ml = P.part_ml + (slot * kPrefixTile + row) * 2;
    *reinterpret_cast<float2*>(ml) = make_float2(m_ref, l);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tc_free512(tmem);
}

cudaError_t launch_prefix_attend(const PrefixAttendParams& P, bool bf16, cudaStream_t stream) {
  auto kern = bf16 ? prefix_attend_kernel<true> : prefix_attend_kernel<false>;
  const size_t smem = (size_t)(2 + kPrefixStages) * kPrefixTileBytes + sizeof(PrefixCtrl) + 1024;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const int blocks = (P.query_tiles + 1) / 2 * P.hkv * P.splits;
  note_launch();
  kern<<<blocks, kPrefixThreads, smem, stream>>>(P);
  return cudaGetLastError();
}

}  // namespace ra
