// Torch binding `cache_ops_cpp` of the quantised-cache and cache-attention entry points: argument checks,
// scratch and the fill of the C ABI's structs, in C++ because a decode step calls them once for every
// layer and token and the same work in Python takes longer than the kernels.  ops.py documents the
// operators; the functions here return the C ABI's status for it to raise.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "topk_attn_b200.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

[[noreturn]] void refuse(const std::string& why) { throw py::value_error(why); }

// The status block of a device, shared by its streams and graphs: kernels only set bits in it.
std::mutex g_mu;
std::map<int, Tensor> g_status;

bool capturing(cudaStream_t stream) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  return cudaStreamIsCapturing(stream, &st) == cudaSuccess && st != cudaStreamCaptureStatusNone;
}

// The block outlives every graph whose kernels write it, also one captured before any eager call on the device:
// it is no part of the capture, so it comes from cudaMalloc in a thread whose capture mode lets that pass, and is
// zeroed on a stream of its own.
Tensor status_for(const torch::Device& dev) {
  std::lock_guard<std::mutex> g(g_mu);
  auto it = g_status.find(dev.index());
  if (it != g_status.end()) return it->second;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
  void* p = nullptr;
  cudaStream_t own = nullptr;
  cudaError_t e = cudaMalloc(&p, 256);
  if (e == cudaSuccess) e = cudaStreamCreateWithFlags(&own, cudaStreamNonBlocking);
  if (e == cudaSuccess) e = cudaMemsetAsync(p, 0, 256, own);
  if (e == cudaSuccess) e = cudaStreamSynchronize(own);
  if (own) cudaStreamDestroy(own);
  if (e != cudaSuccess && p) cudaFree(p);
  C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
  C10_CUDA_CHECK(e);
  return g_status[dev.index()] = torch::from_blob(p, {256}, torch::TensorOptions().dtype(torch::kUInt8).device(dev));
}

// Scratch for one call: the stream's buffer, or memory of the call's own inside a capture, because captured graphs
// may be replayed at the same time, on any streams.  The buffer grows to twice its size at least, and an outgrown
// one goes back to the stream's pool, whose next user on the stream runs behind the launches that still use it.
Tensor scratch_for(size_t bytes, const torch::Device& dev, cudaStream_t stream) {
  static std::map<std::pair<int, cudaStream_t>, Tensor> cache;
  const auto opt = torch::TensorOptions().dtype(torch::kUInt8).device(dev);
  if (capturing(stream)) return torch::empty({(int64_t)bytes}, opt);
  std::lock_guard<std::mutex> g(g_mu);
  Tensor& t = cache[std::make_pair((int)dev.index(), stream)];
  const size_t had = t.defined() ? (size_t)t.numel() : 0;
  if (had < bytes || !t.defined()) {
    t = Tensor();
    t = torch::empty({(int64_t)std::max<size_t>({bytes, 2 * had, 1 << 20})}, opt);
  }
  return t;
}

int row_type(const Tensor& t, const char* what) {
  if (t.scalar_type() == at::kHalf) return RA_TYPE_FP16;
  if (t.scalar_type() == at::kBFloat16) return RA_TYPE_BF16;
  refuse(std::string(what) + " must be fp16 or bf16");
}

struct Strides {
  int64_t b, t, h;
  bool operator==(const Strides& o) const { return b == o.b && t == o.t && h == o.h; }
};

// (batch, token, head) strides of rows [B,T,H,row] or [T,H,row]; dimensions of size one, whose stride
// means nothing, get the one a dense tensor would have.
Strides strides_of(const Tensor& x, int64_t row) {
  const int64_t d = x.dim();
  if (x.stride(d - 1) != 1) refuse("the last dimension must be contiguous");
  Strides s;
  s.h = x.size(d - 2) > 1 ? x.stride(d - 2) : row;
  s.t = x.size(d - 3) > 1 ? x.stride(d - 3) : std::max<int64_t>(x.size(d - 2) * s.h, row);
  s.b = d == 4 && x.size(0) > 1 ? x.stride(0) : std::max<int64_t>(x.size(d - 3), 1) * s.t;
  return s;
}

struct Cache {
  ra_kv_cache c;
  int caches = 0, heads = 0;
};

Cache cache_of(const Tensor& k, const Tensor& v, const OptTensor& ks, const OptTensor& vs, bool per_row,
               const torch::Device& dev) {
  Cache r;
  memset(&r.c, 0, sizeof r.c);
  if (k.dim() != (per_row ? 4 : 3) || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type())
    refuse(per_row ? "k and v must be [B,N,Hkv,128]" : "k and v must be [N,Hkv,128]");
  const bool quantized = ks.has_value();
  if (quantized) {
    if (k.scalar_type() == at::kChar) r.c.format = RA_CACHE_INT8;
    else if (k.scalar_type() == at::kFloat8_e4m3fn) r.c.format = RA_CACHE_FP8;
    else if (k.scalar_type() == at::kByte) r.c.format = RA_CACHE_INT4;
    else refuse("codes must be int8, float8_e4m3fn or uint8 (two int4)");
  } else {
    r.c.format = row_type(k, "a cache that is no QuantizedKV");
  }
  const bool int4 = r.c.format == RA_CACHE_INT4;
  const int64_t row = int4 ? 64 : 128, n = k.size(-3);
  if (k.size(-1) != row) refuse("rows of this cache must have " + std::to_string(row) + " elements");
  r.caches = per_row ? (int)k.size(0) : 1;
  r.heads = (int)k.size(-2);
  if (k.device() != dev || v.device() != dev) refuse("tensors must be on one CUDA device");
  if (n > INT32_MAX) refuse("a cache has at most 2^31 - 1 tokens");
  r.c.num_tokens = (int32_t)n;
  if (n == 0 || r.caches == 0) return r;
  const Strides s = strides_of(k, row);
  if (!(strides_of(v, row) == s)) refuse("k and v must have the same strides");
  r.c.k = k.data_ptr();
  r.c.v = v.data_ptr();
  r.c.batch_stride = s.b;
  r.c.token_stride = s.t;
  r.c.head_stride = s.h;
  if (quantized) {
    const int64_t w = int4 ? 4 : 1, d0 = per_row ? 1 : 0;
    int64_t hs[2], bs[2];
    for (int i = 0; i < 2; ++i) {
      const Tensor& t = i ? *vs : *ks;
      bool ok = t.scalar_type() == at::kFloat && t.device() == dev && t.dim() == d0 + 2 + (int4 ? 1 : 0) &&
                t.size(d0) == r.heads && t.size(d0 + 1) == n && (!per_row || t.size(0) == r.caches) &&
                (!int4 || t.size(d0 + 2) == 4);
      if (!ok) refuse("scales must be fp32 [B,Hkv,N] (shared [Hkv,N]; four to a row for int4)");
      if ((n > 1 && t.stride(d0 + 1) != w) || (int4 && t.stride(d0 + 2) != 1))
        refuse("a head's scales must be contiguous along the tokens");
      hs[i] = r.heads > 1 ? t.stride(d0) : n * w;
      bs[i] = per_row && r.caches > 1 ? t.stride(0) : r.heads * hs[i];
    }
    if (hs[0] != hs[1] || bs[0] != bs[1]) refuse("the scales of k and v must have the same strides");
    r.c.k_scale = ks->data_ptr<float>();
    r.c.v_scale = vs->data_ptr<float>();
    r.c.scale_head_stride = hs[0];
    r.c.scale_batch_stride = bs[0];
  }
  return r;
}

const int32_t* int32_vector(const Tensor& t, int64_t n, const torch::Device& dev, const char* name) {
  if (t.scalar_type() != at::kInt || t.device() != dev || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
    refuse(std::string(name) + " must be a contiguous int32 tensor of " + std::to_string(n) +
           " on the device of the others");
  return t.data_ptr<int32_t>();
}

// back: the cache's rows into k, v; otherwise k, v into the cache
int kv_rows(bool back, const Tensor& ck, const Tensor& cv, const Tensor& cks, const Tensor& cvs, const Tensor& k,
            const Tensor& v, const OptTensor& positions, int64_t position, const OptTensor& counts) {
  if (!k.is_cuda()) refuse("tensors must be CUDA tensors");
  const auto dev = k.device();
  const c10::cuda::CUDAGuard guard(dev);
  const bool per_row = ck.dim() == 4;
  const Cache c = cache_of(ck, cv, cks, cvs, per_row, dev);
  if (k.dim() != ck.dim() || k.size(-1) != 128 || k.size(-2) != c.heads || v.sizes() != k.sizes() ||
      (per_row && k.size(0) != c.caches))
    refuse("rows must be [B,T,Hkv,128] for per-row caches, [T,Hkv,128] for a shared one");
  if (v.scalar_type() != k.scalar_type() || v.device() != dev)
    refuse("rows must be of one type, on the device of the cache");
  if (k.size(-3) > INT32_MAX || position > INT32_MAX || position < INT32_MIN) refuse("sizes beyond 2^31 - 1");
  ra_kv_rows_params p;
  memset(&p, 0, sizeof p);
  p.cache = c.c;
  p.caches = c.caches;
  p.num_kv_heads = c.heads;
  p.head_dim = 128;
  p.row_type = row_type(k, "rows");
  p.num_rows = (int32_t)k.size(-3);
  if (p.num_rows == 0) return RA_OK;
  const Strides a = strides_of(k, 128), b = strides_of(v, 128);
  p.k_batch_stride = a.b; p.k_token_stride = a.t; p.k_head_stride = a.h;
  p.v_batch_stride = b.b; p.v_token_stride = b.t; p.v_head_stride = b.h;
  p.k_rows = k.data_ptr();
  p.v_rows = v.data_ptr();
  if (positions) p.positions = int32_vector(*positions, c.caches, dev, "position");
  p.position = (int32_t)position;
  if (counts) p.counts = int32_vector(*counts, c.caches, dev, "counts");
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  p.stream = stream;
  const Tensor status = status_for(dev);
  p.status = status.data_ptr();
  return back ? ra_kv_dequantize(&p) : ra_kv_append_quantized(&p);
}

// count tokens of every cache as new tensors: (status, k, v)
std::tuple<int, Tensor, Tensor> kv_read(const Tensor& ck, const Tensor& cv, const Tensor& cks, const Tensor& cvs,
                                        const OptTensor& positions, int64_t position, int64_t count, bool bf16) {
  if (!ck.is_cuda()) refuse("tensors must be CUDA tensors");
  if (ck.dim() != 3 && ck.dim() != 4) refuse("k and v must be [B,N,Hkv,128] or [N,Hkv,128]");
  if (count < 0) refuse("count must not be negative");
  std::vector<int64_t> shape(ck.sizes().begin(), ck.sizes().end());
  shape[shape.size() - 3] = count;
  shape.back() = 128;
  const auto opt = torch::TensorOptions().dtype(bf16 ? at::kBFloat16 : at::kHalf).device(ck.device());
  const c10::cuda::CUDAGuard guard(ck.device());
  Tensor k = torch::empty(shape, opt), v = torch::empty(shape, opt);
  const int st = count ? kv_rows(true, ck, cv, cks, cvs, k, v, positions, position, OptTensor()) : RA_OK;
  return {st, k, v};
}

std::pair<int, Tensor> cache_attention(const Tensor& q, const OptTensor& pk, const OptTensor& pv, const OptTensor& pks,
                                       const OptTensor& pvs, const OptTensor& k, const OptTensor& v,
                                       const OptTensor& ks, const OptTensor& vs, const OptTensor& seq_lens,
                                       double sm_scale, const OptTensor& out_given) {
  if (pk.has_value() != pv.has_value() || k.has_value() != v.has_value()) refuse("a cache needs both k and v");
  if (pks.has_value() != pvs.has_value() || ks.has_value() != vs.has_value()) refuse("a quantised cache needs both scales");
  if (!q.is_cuda()) refuse("tensors must be CUDA tensors");
  if (q.dim() != 3 || q.size(2) != 128 || !q.is_contiguous())
    refuse("q must be a contiguous fp16 or bf16 tensor [B,Hq,128]");
  if (!pk && !k) refuse("nothing to attend to: give a prefix, a cache or both");
  const auto dev = q.device();
  const c10::cuda::CUDAGuard guard(dev);
  ra_cache_attention_params p;
  memset(&p, 0, sizeof p);
  p.type = row_type(q, "q");
  if (q.size(0) > INT32_MAX || q.size(1) > INT32_MAX) refuse("sizes beyond 2^31 - 1");
  p.batch = (int32_t)q.size(0);
  p.num_q_heads = (int32_t)q.size(1);
  p.head_dim = 128;
  if (pk) {
    const Cache c = cache_of(*pk, *pv, pks, pvs, false, dev);
    p.prefix = c.c;
    p.num_kv_heads = c.heads;
  }
  if (k) {
    const Cache c = cache_of(*k, *v, ks, vs, true, dev);
    if (c.caches != p.batch) refuse("each row needs a cache: cache.size(0) must be the batch");
    if (pk && c.heads != p.num_kv_heads) refuse("prefix and cache must have the same kv heads");
    p.cache = c.c;
    p.num_kv_heads = c.heads;
  }
  if (seq_lens) {
    if (!k) refuse("seq_lens are the lengths of the rows' own caches");
    p.seq_lens = int32_vector(*seq_lens, p.batch, dev, "seq_lens");
  }
  Tensor out;
  if (out_given) {
    out = *out_given;
    if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || out.device() != dev || !out.is_contiguous())
      refuse("out must be contiguous, of the shape and type of q");
  } else {
    out = torch::empty_like(q);
  }
  p.q = q.data_ptr();
  p.out = out.data_ptr();
  p.sm_scale = (float)sm_scale;
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  p.stream = stream;
  const size_t need = ra_cache_attention_workspace_bytes(p.batch, p.num_q_heads, p.num_kv_heads, p.prefix.num_tokens,
                                                         p.cache.num_tokens);
  const Tensor ws = scratch_for(std::max<size_t>(need, 256), dev, stream), status = status_for(dev);
  p.workspace = ws.data_ptr();
  p.workspace_bytes = (size_t)ws.numel();
  p.status = status.data_ptr();
  return {ra_cache_attention(&p), out};
}

OptTensor status_block(int64_t device) {
  std::lock_guard<std::mutex> g(g_mu);
  auto it = g_status.find((int)device);
  return it == g_status.end() ? OptTensor() : OptTensor(it->second);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("kv_rows", &kv_rows, "Rows into a quantised cache, or back out of it; the C ABI's status");
  m.def("kv_read", &kv_read, "Tokens of a quantised cache as new tensors: (status, k, v)");
  m.def("cache_attention", &cache_attention, "Attention over a shared prefix and own caches: (status, out)");
  m.def("status_block", &status_block, "A device's status block, or None before the first call there");
}
