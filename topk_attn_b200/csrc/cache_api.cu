// Entry points of the C ABI for quantised caches and attention behind a shared prefix: argument
// validation and launches.  Nothing here allocates device memory or synchronises.
#include "topk_attn_b200.h"

#include <cstring>

#include <algorithm>

#include "api_host.cuh"
#include "cache_attend.cuh"

namespace {

using namespace ra;

constexpr float kLog2e = 1.4426950408889634f;

int invalid(const char* why) { return host_fail(RA_ERR_INVALID_ARGUMENT, why); }
int unsupported(const char* why) { return host_fail(RA_ERR_UNSUPPORTED, why); }

bool misaligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// Checks a cache description and turns it into the kernels' view of it.
int view_of(const ra_kv_cache& c, bool per_row, int caches, CacheView& v) {
  if (c.format < RA_CACHE_FP16 || c.format > RA_CACHE_INT4) return invalid("unknown cache format");
  if (!c.k || !c.v) return invalid("a cache pointer is null");
  if (misaligned(c.k, 16) || misaligned(c.v, 16)) return invalid("cache pointers must be 16-byte aligned");
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

int check_rows(const ra_kv_rows_params* p, QuantParams& q) {
  if (!p) return invalid("params is null");
  if (p->head_dim != kHeadDim) return unsupported("head_dim must be 128");
  if (p->caches < 1 || p->num_kv_heads < 1 || p->num_rows < 0) return invalid("sizes must be positive");
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

// splits of one segment's tokens: about eight CTAs per multiprocessor, 256 tokens each at least
int split_count(int batch, int hq, int n) {
  if (n <= 0) return 0;
  const long long rows = (long long)batch * hq;
  const long long want = std::max<long long>(1, 8 * 148 / rows);
  return (int)std::min<long long>(want, (n + 255) / 256);
}

}  // namespace

extern "C" {

int ra_kv_append_quantized(const ra_kv_rows_params* p) {
  QuantParams q;
  const int st = check_rows(p, q);
  if (st != RA_OK) return st;
  if (!p->positions && (p->position < 0 || (int64_t)p->position + p->num_rows > p->cache.num_tokens))
    return invalid("rows outside the cache");
  if (p->num_rows == 0) return RA_OK;
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
  const cudaError_t e = launch_kv_dequantize(q, p->cache.format, p->row_type == RA_TYPE_BF16,
                                             static_cast<cudaStream_t>(p->stream));
  return e == cudaSuccess ? RA_OK : host_cuda_fail(e, "kv_dequantize launch");
}

size_t ra_cache_attention_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                          int32_t prefix_tokens, int32_t cache_tokens) {
  if (batch < 1 || num_kv_heads < 1 || num_q_heads < 1 || prefix_tokens < 0 || cache_tokens < 0) return 0;
  const size_t rows = (size_t)batch * num_q_heads;
  const size_t parts = (size_t)split_count(batch, num_q_heads, prefix_tokens) +
                       (size_t)split_count(batch, num_q_heads, cache_tokens);
  return std::max<size_t>(256, rows * parts * kPartialFloats * sizeof(float));
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
  if ((long long)p->batch * p->num_q_heads > 65535) return unsupported("more than 65535 query rows");
  CacheAttendParams c[2];
  for (int i = 0; i < 2; ++i) {
    const ra_kv_cache& kv = i ? p->cache : p->prefix;
    memset(&c[i], 0, sizeof c[i]);
    if (!has[i]) continue;
    if (kv.format <= RA_CACHE_BF16 && kv.format != p->type) return invalid("the cache must have the type of q");
    const int st = view_of(kv, i == 1, p->batch, c[i].cache);
    if (st != RA_OK) return st;
    c[i].q = p->q;
    c[i].batch = p->batch;
    c[i].hq = p->num_q_heads;
    c[i].hkv = p->num_kv_heads;
    c[i].group = p->num_q_heads / p->num_kv_heads;
    c[i].seq_lens = i ? p->seq_lens : nullptr;
    c[i].status = static_cast<unsigned*>(p->status);
    c[i].splits = split_count(p->batch, p->num_q_heads, kv.num_tokens);
    c[i].split_len = (kv.num_tokens + c[i].splits - 1) / c[i].splits;
    c[i].scale_log2e = p->sm_scale * kLog2e;
  }
  const size_t need = ra_cache_attention_workspace_bytes(p->batch, p->num_q_heads, p->num_kv_heads,
                                                         p->prefix.num_tokens, p->cache.num_tokens);
  if (!p->workspace || p->workspace_bytes < need || misaligned(p->workspace, 256))
    return host_fail(RA_ERR_WORKSPACE,
                     "workspace missing, misaligned or smaller than ra_cache_attention_workspace_bytes()");
  cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
  const bool bf16 = p->type == RA_TYPE_BF16;
  const int rows = p->batch * p->num_q_heads;
  c[0].partials = static_cast<float*>(p->workspace);
  c[1].partials = c[0].partials + (size_t)c[0].splits * rows * kPartialFloats;
  for (int i = 0; i < 2; ++i) {
    if (!has[i]) continue;
    const cudaError_t e = launch_cache_attend(c[i], (i ? p->cache : p->prefix).format, bf16, stream);
    if (e != cudaSuccess) return host_cuda_fail(e, "cache_attend launch");
  }
  const cudaError_t e = launch_cache_combine(c[0].partials, c[0].splits, c[1].partials, c[1].splits, rows, p->out,
                                             bf16, stream);
  return e == cudaSuccess ? RA_OK : host_cuda_fail(e, "cache_combine launch");
}

}  // extern "C"
