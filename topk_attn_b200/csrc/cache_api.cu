// Entry points of the C ABI for quantised caches and attention behind a shared prefix: argument
// validation and launches.  Nothing here allocates device memory or synchronises.
#include "topk_attn_b200.h"

#include <cstdio>
#include <cstring>

#include <algorithm>

#include "api_host.cuh"
#include "cache_attend.cuh"
#include "prefix_attend.cuh"

namespace {

using namespace ra;

constexpr float kLog2e = 1.4426950408889634f;

int invalid(const char* why) { return host_fail(RA_ERR_INVALID_ARGUMENT, why); }
int unsupported(const char* why) { return host_fail(RA_ERR_UNSUPPORTED, why); }

constexpr int kMaxTokens = INT32_MAX - 4095;   // tiles are counted in 32 bits, rounding up
constexpr int kMaxQueryRows = 1 << 24;

bool misaligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// Checks a cache description and turns it into the kernels' view of it.
int view_of(const ra_kv_cache& c, bool per_row, int caches, CacheView& v) {
  if (c.format < RA_CACHE_FP16 || c.format > RA_CACHE_INT4) return invalid("unknown cache format");
  if (!c.k || !c.v) return invalid("a cache pointer is null");
  if (misaligned(c.k, 16) || misaligned(c.v, 16)) return invalid("cache pointers must be 16-byte aligned");
  if (c.num_tokens > kMaxTokens) return unsupported("more than 2^31 - 4096 tokens in a cache");
  const long long esz = c.format <= RA_CACHE_BF16 ? 2 : 1;
  const int row = cache_row_bytes(c.format);
  v.k = static_cast<unsigned char*>(c.k);
  v.v = static_cast<unsigned char*>(c.v);
  v.n_tokens = c.num_tokens;
  v.tstride = c.token_stride * esz;
  v.hstride = c.head_stride * esz;
  v.bstride = per_row ? c.batch_stride * esz : 0;
  if (v.tstride < row || v.hstride < row || v.tstride % 16 || v.hstride % 16)
    return invalid("cache strides must hold a row and be multiples of 16 bytes");
  if (per_row && caches > 1 && (v.bstride <= 0 || v.bstride % 16))
    return invalid("one cache for each row needs a batch stride that is a multiple of 16 bytes");
  if (per_row && caches > 1 && v.bstride < row) return invalid("the batch stride must hold a row");
  v.k_scale = v.v_scale = nullptr;
  v.sbstride = v.shstride = 0;
  const int ns = cache_row_scales(c.format);
  if (ns) {
    if (!c.k_scale || !c.v_scale) return invalid("a quantised cache needs its scales");
    if (misaligned(c.k_scale, 4 * ns) || misaligned(c.v_scale, 4 * ns)) return invalid("scales are misaligned");
    v.k_scale = c.k_scale;
    v.v_scale = c.v_scale;
    v.shstride = c.scale_head_stride;
    v.sbstride = per_row ? c.scale_batch_stride : 0;
    if (v.shstride < (long long)ns * c.num_tokens || v.shstride % ns || v.sbstride % ns)
      return invalid("scale strides must hold every token's scales");
    if (per_row && caches > 1 && v.sbstride <= 0) return invalid("scales need a batch stride");
  }
  return RA_OK;
}

// A call's first kernel is launched so that its launch overlaps the end of whatever runs before it (it waits
// for that end itself), except in a capture, where what is before it need not be a kernel.
bool capturing(cudaStream_t stream) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  return cudaStreamIsCapturing(stream, &st) != cudaSuccess || st != cudaStreamCaptureStatusNone;
}

int check_rows(const ra_kv_rows_params* p, QuantParams& q) {
  if (!p) return invalid("params is null");
  if (p->head_dim != kHeadDim) return unsupported("head_dim must be 128");
  if (p->caches < 1 || p->num_kv_heads < 1 || p->num_rows < 0) return invalid("sizes must be positive");
  if (p->caches > 65535 || p->num_kv_heads > kQuantMaxHeads)
    return unsupported("more than 65535 caches or 1024 kv heads");
  if (p->num_rows > kMaxTokens) return unsupported("more than 2^31 - 4096 rows for a cache");
  if (p->cache.num_tokens < 1) return invalid("the cache has no tokens");
  if (p->cache.format < RA_CACHE_INT8) return invalid("the cache must be int8, fp8 or int4");
  if (p->row_type != RA_TYPE_FP16 && p->row_type != RA_TYPE_BF16) return invalid("rows must be fp16 or bf16");
  memset(&q, 0, sizeof q);
  const int st = view_of(p->cache, true, p->caches, q.cache);
  if (st != RA_OK) return st;
  if (!p->k_rows || !p->v_rows || !p->status) return invalid("a required pointer is null");
  if (misaligned(p->k_rows, 16) || misaligned(p->v_rows, 16)) return invalid("rows must be 16-byte aligned");
  q.rows[0] = p->k_rows;
  q.rows[1] = p->v_rows;
  const int64_t s[6] = {p->k_batch_stride, p->k_token_stride, p->k_head_stride,
                        p->v_batch_stride, p->v_token_stride, p->v_head_stride};
  for (int i = 0; i < 6; ++i)
    if (s[i] < 0 || s[i] % 8) return invalid("row strides must be multiples of 8 elements");
  for (int i = 0; i < 2; ++i) {
    q.rb[i] = s[3 * i];
    q.rt[i] = s[3 * i + 1];
    q.rh[i] = s[3 * i + 2];
  }
  q.caches = p->caches;
  q.heads = p->num_kv_heads;
  q.n_rows = p->num_rows;
  q.positions = p->positions;
  q.position = p->position;
  q.counts = p->counts;
  q.status = static_cast<unsigned*>(p->status);
  return RA_OK;
}

// Tensor map over K or V: boxes of `rows` tokens of one head, swizzled over the 128 (int4: 64) bytes of a
// row or half row.
int encode_map(CUtensorMap* map, const void* base, const CacheView& v, int format, int heads, int caches, int rows) {
  EncodeTiledFn enc = host_encode_fn();
  if (!enc) return host_fail(RA_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const bool dense = format <= RA_CACHE_BF16;
  const cuuint64_t row = dense ? kHeadDim : cache_row_bytes(format);
  const cuuint64_t dims[4] = {row, (cuuint64_t)heads, (cuuint64_t)v.n_tokens, (cuuint64_t)caches};
  const cuuint64_t strides[3] = {(cuuint64_t)v.hstride, (cuuint64_t)v.tstride,
                                 (cuuint64_t)(caches > 1 ? v.bstride : v.tstride)};
  const cuuint32_t box[4] = {(cuuint32_t)(dense ? 64 : row), 1, (cuuint32_t)rows, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = format == RA_CACHE_FP16   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                   : format == RA_CACHE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                             : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const CUresult r = enc(map, type, 4, const_cast<void*>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE,
                         format == RA_CACHE_INT4 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                         // no more than the row: what lies behind it is another head's
                         dense                       ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B
                         : format == RA_CACHE_INT4 ? CU_TENSOR_MAP_L2_PROMOTION_L2_64B
                                                   : CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return RA_OK;
  char buf[96];
  snprintf(buf, sizeof buf, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  return host_fail(RA_ERR_CUDA, buf);
}

// How one segment is worked on, and where its partials lie in the scratch.
struct SegmentPlan {
  int caches, queries, qt, query_tiles;
  int nq, grid;        // of the line of work rows (cache_attend)
  int splits;          // > 0: the prefix goes to prefix_attend, its tokens cut into so many ranges
  size_t ml_at, span_at, bytes;   // part_o at 0
};

// Ranges that the prefix's tokens are cut into: the fewest rounds of CTAs, one to a multiprocessor, by
// what each costs (its tiles, and about four for its beginning and end).
int prefix_splits(int blocks, int tiles, int sms) {
  int best = 1;
  long long best_cost = -1;
  for (int s = 1; s <= std::min(tiles, std::max(1, 2 * sms / blocks)); ++s) {
    const long long rounds = ((long long)blocks * s + sms - 1) / sms;
    const long long cost = rounds * ((tiles + s - 1) / s + 4);
    if (best_cost < 0 || cost < best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  return best;
}

// Queries per key up to which a prefix goes to cache_attend, 16 of them at a time; above, to prefix_attend, 128 at
// a time.  8 kv heads, us by the one and the other: 65536 fp16 tokens, 17 to 32 queries 90 and 57; int8 76 and 114
// to 120, 48 queries 106 and 114, 64 queries 137 and 114; fp8 64 and 83, 48 queries 90 and 83.  8192 tokens: fp16
// 18 and 17, int8 19 and 28, fp8 17 and 20, 64 queries 25 and 18, 29 and 23, 23 and 20.  int4 has scales along the
// dims, which prefix_attend cannot apply to S.
int most_narrow_queries(int format) {
  return format == RA_CACHE_INT4 ? INT32_MAX : format <= RA_CACHE_BF16 ? 16 : 32;
}

// Where every cache is equally long and held in fp8, the grid is a multiple of the rows, so that the heads,
// whose 128-byte rows lie side by side in memory, are walked in step: 8 x 32768 tokens of 8 heads take 94 us
// so, with 384 CTAs, and 107 with all 444; with 4 and 2 heads, whose rows fill less of a page, 90 either way.  Not
// below 5/6 of the CTAs that fit.  256-byte rows do not need it; int8 and int4, bound by their arithmetic, need
// the CTAs (8 heads, in step: int8 113 against 107, int4 113 against 99).
int grid_in_step(long long rows, int grid, int format, bool equal) {
  if (!equal || format != RA_CACHE_FP8 || rows > grid) return grid;
  const int whole = (int)(grid / rows * rows);
  return 6 * whole >= 5 * grid ? whole : grid;
}

SegmentPlan plan_segment(bool prefix, int format, bool equal, int batch, int hq, int hkv, int tokens, int sms) {
  SegmentPlan s;
  memset(&s, 0, sizeof s);
  if (tokens <= 0) return s;
  const int group = hq / hkv;
  s.caches = prefix ? 1 : batch;
  s.queries = prefix ? batch * group : group;
  s.nq = s.queries <= 8 ? 1 : 2;
  const bool wide = prefix && s.queries > most_narrow_queries(format);
  s.qt = wide ? kPrefixTile : 8 * s.nq;
  s.query_tiles = (s.queries + s.qt - 1) / s.qt;
  const long long rows = (long long)s.caches * hkv * s.query_tiles;
  size_t slots;
  if (wide) {
    const int blocks = (s.query_tiles + 1) / 2 * hkv;
    s.splits = prefix_splits(blocks, (tokens + kPrefixTile - 1) / kPrefixTile, sms);
    slots = (size_t)rows * s.splits;
  } else {
    const long long units = rows * ((tokens + kAttendTile - 1) / kAttendTile + kAttendRowUnits);
    s.grid = (int)std::min<long long>(units, (long long)attend_ctas(s.nq) * sms);
    slots = (size_t)rows + s.grid;      // room for the full grid, whatever the lengths
    s.grid = grid_in_step(rows, s.grid, format, equal);
  }
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  s.ml_at = up(slots * s.qt * kHeadDim * sizeof(float));
  s.span_at = s.ml_at + up(slots * s.qt * 2 * sizeof(float));
  s.bytes = s.span_at + up((size_t)rows * 2 * sizeof(int));
  return s;
}

}  // namespace

extern "C" {

int ra_kv_append_quantized(const ra_kv_rows_params* p) {
  QuantParams q;
  const int st = check_rows(p, q);
  if (st != RA_OK) return st;
  // counts may keep the last rows of a padded batch out of the cache's end: then the kernel looks
  if (!p->positions && (p->position < 0 || (!p->counts && (int64_t)p->position + p->num_rows > p->cache.num_tokens)))
    return invalid("rows outside the cache");
  if (p->num_rows == 0) return RA_OK;
  q.early = !capturing(static_cast<cudaStream_t>(p->stream));
  const cudaError_t e = launch_kv_quantize(q, p->cache.format, p->row_type == RA_TYPE_BF16,
                                           static_cast<cudaStream_t>(p->stream));
  return e == cudaSuccess ? RA_OK : host_cuda_fail(e, "kv_append_quantized launch");
}

int ra_kv_dequantize(const ra_kv_rows_params* p) {
  QuantParams q;
  const int st = check_rows(p, q);
  if (st != RA_OK) return st;
  if (!p->positions && (p->position < 0 || (int64_t)p->position + p->num_rows > p->cache.num_tokens))
    return invalid("rows outside the cache");
  if (p->num_rows == 0) return RA_OK;
  q.early = !capturing(static_cast<cudaStream_t>(p->stream));
  const cudaError_t e = launch_kv_dequantize(q, p->cache.format, p->row_type == RA_TYPE_BF16,
                                             static_cast<cudaStream_t>(p->stream));
  return e == cudaSuccess ? RA_OK : host_cuda_fail(e, "kv_dequantize launch");
}

size_t ra_cache_attention_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                          int32_t prefix_tokens, int32_t cache_tokens) {
  if (batch < 1 || num_kv_heads < 1 || num_q_heads < num_kv_heads || prefix_tokens < 0 || cache_tokens < 0) return 0;
  // what ra_cache_attention refuses; the plans count rows and tiles in 32 bits
  if (num_q_heads % num_kv_heads || (long long)batch * num_q_heads > kMaxQueryRows || prefix_tokens > kMaxTokens ||
      cache_tokens > kMaxTokens)
    return 0;
  // room for either kind of cache
  const int sms = host_sm_count();
  size_t need = 0;
  for (int format : {RA_CACHE_FP16, RA_CACHE_INT4})
    need = std::max(need, plan_segment(true, format, true, batch, num_q_heads, num_kv_heads, prefix_tokens, sms).bytes +
                              plan_segment(false, format, true, batch, num_q_heads, num_kv_heads, cache_tokens, sms).bytes);
  return 256 + need;
}

int ra_cache_attention(const ra_cache_attention_params* p) {
  if (!p) return invalid("params is null");
  if (p->head_dim != kHeadDim) return unsupported("head_dim must be 128");
  if (p->batch < 1 || p->num_q_heads < 1 || p->num_kv_heads < 1) return invalid("sizes must be positive");
  if (p->num_q_heads % p->num_kv_heads) return invalid("num_kv_heads must divide num_q_heads");
  if (p->type != RA_TYPE_FP16 && p->type != RA_TYPE_BF16) return invalid("type must be fp16 or bf16");
  if (!(p->sm_scale > 0.f)) return invalid("sm_scale must be positive");
  if (!p->q || !p->out || !p->status) return invalid("a required pointer is null");
  if (misaligned(p->q, 16) || misaligned(p->out, 16)) return invalid("q and out must be 16-byte aligned");
  const bool has[2] = {p->prefix.num_tokens > 0, p->cache.num_tokens > 0};
  if (p->prefix.num_tokens < 0 || p->cache.num_tokens < 0) return invalid("sizes must not be negative");
  if (has[0] && has[1] && p->prefix.format != p->cache.format)
    return invalid("prefix and cache must have one format");
  if ((long long)p->batch * p->num_q_heads > kMaxQueryRows) return unsupported("more than 2^24 query rows");
  CacheView view[2];
  for (int i = 0; i < 2; ++i) {
    const ra_kv_cache& kv = i ? p->cache : p->prefix;
    if (!has[i]) continue;
    if (kv.format <= RA_CACHE_BF16 && kv.format != p->type) return invalid("the cache must have the type of q");
    const int st = view_of(kv, i == 1, p->batch, view[i]);
    if (st != RA_OK) return st;
  }
  const size_t need = ra_cache_attention_workspace_bytes(p->batch, p->num_q_heads, p->num_kv_heads,
                                                         p->prefix.num_tokens, p->cache.num_tokens);
  if (!p->workspace || p->workspace_bytes < need || misaligned(p->workspace, 256))
    return host_fail(RA_ERR_WORKSPACE,
                     "workspace missing, misaligned or smaller than ra_cache_attention_workspace_bytes()");
  cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
  const bool bf16 = p->type == RA_TYPE_BF16;
  const int sms = host_sm_count();
  CombineParams cp;
  memset(&cp, 0, sizeof cp);
  cp.out = p->out;
  cp.batch = p->batch;
  cp.hq = p->num_q_heads;
  cp.hkv = p->num_kv_heads;
  cp.group = p->num_q_heads / p->num_kv_heads;
  const bool early = !capturing(stream);
  char* at = static_cast<char*>(p->workspace);
  for (int i = 0; i < 2; ++i) {
    if (!has[i]) continue;
    const int format = (i ? p->cache : p->prefix).format;
    const SegmentPlan s =
        plan_segment(i == 0, format, i == 0 || !p->seq_lens, p->batch, p->num_q_heads, p->num_kv_heads, view[i].n_tokens, sms);
    float* part_o = reinterpret_cast<float*>(at);
    float* part_ml = reinterpret_cast<float*>(at + s.ml_at);
    CombineSegment& c = cp.seg[i];
    c.part_o = part_o;
    c.part_ml = part_ml;
    c.span = reinterpret_cast<int*>(at + s.span_at);
    c.lens = i ? p->seq_lens : nullptr;
    c.query_tiles = s.query_tiles;
    c.qt = s.qt;
    c.splits = s.splits;
    c.prefix = i == 0;
    at += s.bytes;
    const int box = s.splits ? kPrefixTile : kAttendTile;
    CUtensorMap maps[2];
    for (int j = 0; j < 2; ++j) {
      const int st = encode_map(&maps[j], j ? view[i].v : view[i].k, view[i], format, p->num_kv_heads, s.caches, box);
      if (st != RA_OK) return st;
    }
    if (s.splits) {
      PrefixAttendParams a;
      memset(&a, 0, sizeof a);
      a.kmap = maps[0];
      a.vmap = maps[1];
      a.q = p->q;
      a.k_scale = view[i].k_scale;
      a.v_scale = view[i].v_scale;
      a.scale_hstride = view[i].shstride;
      a.part_o = part_o;
      a.part_ml = part_ml;
      a.status = static_cast<unsigned*>(p->status);
      a.n_tokens = view[i].n_tokens;
      a.queries = s.queries;
      a.query_tiles = s.query_tiles;
      a.hq = p->num_q_heads;
      a.hkv = p->num_kv_heads;
      a.group = cp.group;
      a.splits = s.splits;
      a.early = early;
      a.scale_log2e = p->sm_scale * kLog2e;
      const cudaError_t e = launch_prefix_attend(a, format, bf16, stream);
      if (e != cudaSuccess) return host_cuda_fail(e, "prefix_attend launch");
      continue;
    }
    CacheAttendParams a;
    memset(&a, 0, sizeof a);
    AttendSegment& g = a.seg;
    g.kmap = maps[0];
    g.vmap = maps[1];
    g.cache = view[i];
    g.lens = i ? p->seq_lens : nullptr;
    g.caches = s.caches;
    g.queries = s.queries;
    g.query_tiles = s.query_tiles;
    g.grid = s.grid;
    g.nstages = cache_attend_stages(format, s.nq);
    g.part_o = part_o;
    g.part_ml = part_ml;
    g.span = const_cast<int*>(c.span);
    a.q = p->q;
    a.status = static_cast<unsigned*>(p->status);
    a.hq = p->num_q_heads;
    a.hkv = p->num_kv_heads;
    a.group = cp.group;
    a.after = i == 1 && has[0];
    a.early = a.after || early;
    a.scale_log2e = p->sm_scale * kLog2e;
    const cudaError_t e = launch_cache_attend(a, format, bf16, s.nq, stream);
    if (e != cudaSuccess) return host_cuda_fail(e, "cache_attend launch");
  }
  const cudaError_t e = launch_cache_combine(cp, bf16, stream);
  return e == cudaSuccess ? RA_OK : host_cuda_fail(e, "cache_combine launch");
}

}  // extern "C"
