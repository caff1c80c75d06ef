// The batched-serving operators of `megakernel_extension`: prompt_attention,
// paged_attention and paged_append over the C ABI of libmkb200.so.
//
// Every argument that the host can see is checked (ValueError); lengths and page
// numbers live on the device and are checked there (see serving_status). A call
// launches on the caller's current stream, synchronises nothing and can be captured
// into a CUDA graph. The attention's workspace is kept per device and stream, so
// that calls on different streams never share one; a captured call gets its own, whose
// counters (5 KB) the graph clears. (A replayed decode call over one request of 33 keys takes
// 7.9 us, over 48 of 1-4,096 58.4; 27.9 and 87.2 where all of its 79 MB are cleared.)

#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime.h>

#include <cmath>
#include <map>
#include <mutex>
#include <optional>
#include <utility>

#include "mkb200.h"

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

int type_code(const Tensor& t, const char* name, bool fp32 = false) {
  switch (t.scalar_type()) {
    case torch::kBFloat16: return MKB_BF16;
    case torch::kHalf: return MKB_FP16;
    case torch::kFloat:
      if (fp32) return MKB_FP32;
      [[fallthrough]];
    default:
      TORCH_CHECK_VALUE(false, name, " must be bfloat16", fp32 ? ", float16 or float32" : " or float16", ", got ",
                        t.scalar_type());
  }
}

void check_on(const Tensor& t, const char* name, c10::Device dev) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK_VALUE(t.device() == dev, name, " must be on ", dev, ", is on ", t.device());
}

// 16-byte accesses along the last dimension; other dimensions of one element carry no stride
void check_layout(const Tensor& t, const char* name) {
  const int64_t d = t.dim();
  TORCH_CHECK_VALUE(t.stride(d - 1) == 1 || t.numel() == 0, name, " must be contiguous in its last dimension");
  const int64_t unit = 16 / t.element_size();
  for (int64_t i = 0; i + 1 < d; ++i)
    TORCH_CHECK_VALUE(t.size(i) <= 1 || t.stride(i) % unit == 0, name, " must have strides of whole 16 bytes, got ",
                      t.strides());
  TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name, " must be 16-byte aligned");
}

// keys at places of their own (dimension i not expanded)
void check_apart(const Tensor& t, const char* name, int64_t i) {
  TORCH_CHECK_VALUE(t.size(i) <= 1 || t.stride(i) != 0, name, " must not be expanded along dimension ", i);
}

int64_t stride_of(const Tensor& t, int64_t i) { return t.size(i) <= 1 ? 0 : t.stride(i); }

void check_type(const Tensor& t, const char* name, const Tensor& like, const char* like_name) {
  TORCH_CHECK_VALUE(t.scalar_type() == like.scalar_type(), name, " must have ", like_name, "'s type ",
                    like.scalar_type(), ", got ", t.scalar_type());
}

void check_int32(const Tensor& t, const char* name, c10::Device dev, int64_t dim) {
  check_on(t, name, dev);
  TORCH_CHECK_VALUE(t.scalar_type() == torch::kInt, name, " must be int32, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == dim, name, " must have ", dim, " dimension(s), got ", t.dim());
  TORCH_CHECK_VALUE(t.numel() == 0 || t.stride(dim - 1) == 1 || t.size(dim - 1) == 1, name,
                    " must be contiguous in its last dimension");
}

int as_int(int64_t v, const char* what) {
  TORCH_CHECK_VALUE(v >= 0 && v <= 0x7fffffff, what, " is out of range: ", v);
  return static_cast<int>(v);
}

// ---- per-device status word, per-stream workspace --------------------------------
struct Kept {
  std::mutex mu;
  std::map<int, Tensor> status;
  std::map<std::pair<int, unsigned long long>, Tensor> workspace;
};
Kept& kept() {
  static Kept* k = new Kept;  // outlives the interpreter: the tensors are not freed at exit
  return *k;
}

Tensor status_of(c10::Device dev) {
  std::lock_guard<std::mutex> lk(kept().mu);
  Tensor& t = kept().status[dev.index()];
  if (!t.defined()) {
    // once per device, in memory of its own and cleared on a stream of its own: the first call
    // may be one that is captured, and the word outlives the graph
    const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
    void* word = nullptr;
    cudaStream_t side = nullptr;
    C10_CUDA_CHECK(cudaMalloc(&word, sizeof(int)));
    C10_CUDA_CHECK(cudaStreamCreateWithFlags(&side, cudaStreamNonBlocking));
    C10_CUDA_CHECK(cudaMemsetAsync(word, 0, sizeof(int), side));
    C10_CUDA_CHECK(cudaStreamSynchronize(side));
    C10_CUDA_CHECK(cudaStreamDestroy(side));
    t = torch::from_blob(word, {1}, torch::TensorOptions().dtype(torch::kInt).device(dev));
  }
  return t;
}

Tensor workspace_of(c10::Device dev, cudaStream_t stream, size_t bytes) {
  const auto options = torch::TensorOptions().dtype(torch::kByte).device(dev);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  C10_CUDA_CHECK(cudaStreamIsCapturing(stream, &cap));
  auto fresh = [&] {
    const Tensor t = torch::empty({static_cast<int64_t>(bytes)}, options);
    C10_CUDA_CHECK(mkb_attn_workspace_reset(t.data_ptr(), bytes, stream));
    return t;
  };
  if (cap != cudaStreamCaptureStatusNone) return fresh();
  unsigned long long id = 0;
  C10_CUDA_CHECK(cudaStreamGetId(stream, &id));
  std::lock_guard<std::mutex> lk(kept().mu);
  Tensor& t = kept().workspace[{dev.index(), id}];
  if (!t.defined() || static_cast<size_t>(t.numel()) < bytes) t = fresh();  // the old one is freed in stream order
  return t;
}

// ---- the packed batch ---------------------------------------------------------------
struct Batch {
  int tokens, batch, q_len;
  const int* cu;
  int64_t token_stride, head_stride;
};

// x [tokens, heads, D] with cu_q, or [batch, heads, D] / [batch, n, heads, D] without
Batch batch_of(const Tensor& x, const char* name, const OptTensor& cu_q, int64_t requests, c10::Device dev) {
  Batch b{};
  const int64_t d = x.dim();
  if (cu_q.has_value()) {
    TORCH_CHECK_VALUE(d == 3, name, " must be [tokens, heads, dim] where cu_q is given, got ", x.sizes());
    check_int32(*cu_q, "cu_q", dev, 1);
    TORCH_CHECK_VALUE(cu_q->size(0) == requests + 1, "cu_q must have ", requests + 1, " entries, got ", cu_q->size(0));
    b.cu = cu_q->data_ptr<int>();
    b.tokens = as_int(x.size(0), "tokens");
    b.token_stride = stride_of(x, 0);
  } else {
    TORCH_CHECK_VALUE(d == 3 || d == 4, name, " must be [batch, heads, dim] or [batch, n, heads, dim], got ", x.sizes());
    TORCH_CHECK_VALUE(x.size(0) == requests, name, " must hold ", requests, " requests, got ", x.size(0));
    b.q_len = d == 4 ? as_int(x.size(1), "new tokens") : 1;
    b.tokens = as_int(x.size(0) * b.q_len, "tokens");
    b.token_stride = d == 4 && x.size(1) > 1 ? x.stride(1) : stride_of(x, 0);
    TORCH_CHECK_VALUE(d == 3 || x.size(0) <= 1 || x.size(1) <= 1 || x.stride(0) == x.size(1) * x.stride(1), name,
                      " must have its tokens evenly apart, got strides ", x.strides());
  }
  TORCH_CHECK_VALUE(b.tokens == 0 || requests > 0, name, " holds tokens of no request");
  b.batch = as_int(requests, "batch");
  b.head_stride = stride_of(x, d - 2);
  return b;
}

Tensor output_for(const OptTensor& out, const Tensor& q, c10::Device dev) {
  if (!out.has_value()) return torch::empty(q.sizes(), q.options());
  check_on(*out, "out", dev);
  check_type(*out, "out", q, "q");
  TORCH_CHECK_VALUE(out->sizes() == q.sizes(), "out must have q's shape ", q.sizes(), ", got ", out->sizes());
  check_layout(*out, "out");
  TORCH_CHECK_VALUE(out->dim() == 3 || out->size(0) <= 1 || out->size(1) <= 1 ||
                        out->stride(0) == out->size(1) * out->stride(1),
                    "out must have its tokens evenly apart, got strides ", out->strides());
  return *out;
}

void set_query(mkb_attn_args& a, const Tensor& q, const Tensor& out, const Batch& b, std::optional<double> scale) {
  const int64_t d = q.dim();
  for (int64_t i = 0; i + 1 < d; ++i) {
    check_apart(q, "q", i);
    check_apart(out, "out", i);
  }
  a.heads = as_int(q.size(d - 2), "heads");
  a.head_dim = as_int(q.size(d - 1), "head_dim");
  TORCH_CHECK_VALUE(a.head_dim == 64 || a.head_dim == 128, "the head dimension must be 64 or 128, got ", a.head_dim);
  a.tokens = b.tokens;
  a.batch = b.batch;
  a.q_len = b.q_len;
  a.cu_q = b.cu;
  a.q = q.data_ptr();
  a.q_stride[0] = b.token_stride;
  a.q_stride[1] = b.head_stride;
  a.out = out.data_ptr();
  a.out_stride[0] = d == 4 && out.size(1) > 1 ? out.stride(1) : stride_of(out, 0);
  a.out_stride[1] = stride_of(out, d - 2);
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(a.head_dim));
  TORCH_CHECK_VALUE(std::isfinite(static_cast<float>(s)) && static_cast<float>(s) > 0.f,
                    "scale must be positive and finite, got ", s);
  a.scale = static_cast<float>(s);
}

void check_heads(int heads, int64_t kv_heads, const Batch& b) {
  TORCH_CHECK_VALUE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, heads, " query heads are no multiple of ",
                    kv_heads, " KV heads");
  TORCH_CHECK_VALUE(heads / kv_heads <= 128, "at most 128 query heads may share a KV head, got ", heads / kv_heads);
  // (rows and their blocks, over all heads, are counted in 32 bits)
  TORCH_CHECK_VALUE(static_cast<int64_t>(b.tokens) + b.batch <= (int64_t{1} << 30) / heads, b.tokens, " tokens and ",
                    b.batch, " requests of ", heads, " heads are more than can be counted: at most ",
                    (int64_t{1} << 30) / heads);
}

struct Paging {
  int kv_heads, pages, page_size, width;
  int64_t table_stride;
  int64_t k_stride[3], v_stride[3];
};

Paging paging_of(const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table, const Tensor& kv_lens,
                 int64_t head_dim, c10::Device dev) {
  Paging p{};
  check_on(k_cache, "k_cache", dev);
  check_on(v_cache, "v_cache", dev);
  TORCH_CHECK_VALUE(k_cache.dim() == 4, "k_cache must be [pages, kv_heads, page_size, dim], got ", k_cache.sizes());
  TORCH_CHECK_VALUE(v_cache.sizes() == k_cache.sizes(), "v_cache must have k_cache's shape ", k_cache.sizes(), ", got ",
                    v_cache.sizes());
  TORCH_CHECK_VALUE(k_cache.size(3) == head_dim, "k_cache must have heads of ", head_dim, ", got ", k_cache.size(3));
  check_type(v_cache, "v_cache", k_cache, "k_cache");
  check_layout(k_cache, "k_cache");
  check_layout(v_cache, "v_cache");
  for (const int i : {0, 2}) {
    check_apart(k_cache, "k_cache", i);
    check_apart(v_cache, "v_cache", i);
  }
  p.pages = as_int(k_cache.size(0), "pages");
  p.kv_heads = as_int(k_cache.size(1), "kv_heads");
  p.page_size = as_int(k_cache.size(2), "page_size");
  TORCH_CHECK_VALUE(p.page_size >= 16 && (p.page_size & (p.page_size - 1)) == 0,
                    "page_size must be a power of two, 16 or more, got ", p.page_size);
  check_int32(block_table, "block_table", dev, 2);
  check_int32(kv_lens, "kv_lens", dev, 1);
  TORCH_CHECK_VALUE(kv_lens.size(0) == block_table.size(0), "kv_lens must have ", block_table.size(0),
                    " entries (one per row of block_table), got ", kv_lens.size(0));
  p.width = as_int(block_table.size(1), "block_table's width");
  p.table_stride = stride_of(block_table, 0);
  for (int i = 0; i < 3; ++i) {
    p.k_stride[i] = stride_of(k_cache, i);
    p.v_stride[i] = stride_of(v_cache, i);
  }
  return p;
}

}  // namespace

Tensor prompt_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_seqlens,
                        std::optional<double> scale, const OptTensor& out_) {
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a CUDA tensor");
  const c10::Device dev = q.device();
  mkb_attn_args a{};
  a.dtype = type_code(q, "q");
  TORCH_CHECK_VALUE(q.dim() == 3, "q must be [tokens, heads, dim], got ", q.sizes());
  check_on(k, "k", dev);
  check_on(v, "v", dev);
  check_type(k, "k", q, "q");
  check_type(v, "v", q, "q");
  TORCH_CHECK_VALUE(k.dim() == 3 && k.size(0) == q.size(0) && k.size(2) == q.size(2),
                    "k must be [tokens, kv_heads, dim] with q's tokens and dim, got ", k.sizes());
  TORCH_CHECK_VALUE(v.sizes() == k.sizes(), "v must have k's shape ", k.sizes(), ", got ", v.sizes());
  check_layout(q, "q");
  check_layout(k, "k");
  check_layout(v, "v");
  check_apart(k, "k", 0);
  check_apart(v, "v", 0);
  TORCH_CHECK_VALUE(cu_seqlens.dim() == 1 && cu_seqlens.size(0) >= 1, "cu_seqlens must be [prompts + 1]");
  const Batch b = batch_of(q, "q", cu_seqlens, cu_seqlens.size(0) - 1, dev);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor out = output_for(out_, q, dev);
  set_query(a, q, out, b, scale);
  a.kv_heads = as_int(k.size(1), "kv_heads");
  check_heads(a.heads, a.kv_heads, b);
  if (a.tokens == 0) return out;
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  for (int i = 0; i < 2; ++i) {
    a.k_stride[i] = stride_of(k, i);
    a.v_stride[i] = stride_of(v, i);
  }
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  const Tensor ws = workspace_of(dev, stream, mkb_attn_workspace_bytes(&a)), st = status_of(dev);
  a.workspace = ws.data_ptr();
  a.status = reinterpret_cast<uint32_t*>(st.data_ptr());
  C10_CUDA_CHECK(mkb_prompt_attention(&a, stream));
  return out;
}

Tensor paged_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table,
                       const Tensor& kv_lens, const OptTensor& cu_q, std::optional<double> scale,
                       const OptTensor& out_) {
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a CUDA tensor");
  const c10::Device dev = q.device();
  mkb_attn_args a{};
  a.dtype = type_code(q, "q");
  TORCH_CHECK_VALUE(q.dim() >= 3, "q must be [batch, heads, dim], [batch, n, heads, dim] or, with cu_q, ",
                    "[tokens, heads, dim], got ", q.sizes());
  check_layout(q, "q");
  const Paging p = paging_of(k_cache, v_cache, block_table, kv_lens, q.size(q.dim() - 1), dev);
  check_type(k_cache, "k_cache", q, "q");
  const Batch b = batch_of(q, "q", cu_q, kv_lens.size(0), dev);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor out = output_for(out_, q, dev);
  set_query(a, q, out, b, scale);
  a.kv_heads = p.kv_heads;
  check_heads(a.heads, a.kv_heads, b);
  if (a.tokens == 0) return out;
  a.k = k_cache.data_ptr();
  a.v = v_cache.data_ptr();
  for (int i = 0; i < 3; ++i) {
    a.k_stride[i] = p.k_stride[i];
    a.v_stride[i] = p.v_stride[i];
  }
  a.kv_lens = kv_lens.data_ptr<int>();
  a.block_table = block_table.data_ptr<int>();
  a.table_stride = p.table_stride;
  a.table_width = p.width;
  a.pages = p.pages;
  a.page_size = p.page_size;
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  const Tensor ws = workspace_of(dev, stream, mkb_attn_workspace_bytes(&a)), st = status_of(dev);
  a.workspace = ws.data_ptr();
  a.status = reinterpret_cast<uint32_t*>(st.data_ptr());
  C10_CUDA_CHECK(mkb_paged_attention(&a, stream));
  return out;
}

pybind11::object paged_append(const Tensor& qkv, const Tensor& k_cache, const Tensor& v_cache,
                              const Tensor& block_table, const Tensor& kv_lens, const Tensor& cos, const Tensor& sin,
                              const OptTensor& cu_q, const OptTensor& q_norm, const OptTensor& k_norm, double eps,
                              bool return_k) {
  TORCH_CHECK_VALUE(qkv.is_cuda(), "qkv must be a CUDA tensor");
  const c10::Device dev = qkv.device();
  mkb_append_args a{};
  a.source_dtype = type_code(qkv, "qkv", true);
  TORCH_CHECK_VALUE(qkv.dim() >= 3, "qkv must be [batch, heads + 2 kv_heads, dim], [batch, n, ...] or, with cu_q, ",
                    "[tokens, ...], got ", qkv.sizes());
  check_layout(qkv, "qkv");
  const int64_t d = qkv.dim(), dim = qkv.size(d - 1);
  TORCH_CHECK_VALUE(dim == 64 || dim == 128, "the head dimension must be 64 or 128, got ", dim);
  const Paging p = paging_of(k_cache, v_cache, block_table, kv_lens, dim, dev);
  check_apart(k_cache, "k_cache", 1);  // (attention may read one head for all; here each is written)
  check_apart(v_cache, "v_cache", 1);
  a.dtype = type_code(k_cache, "k_cache");
  const Batch b = batch_of(qkv, "qkv", cu_q, kv_lens.size(0), dev);
  const int64_t heads = qkv.size(d - 2) - 2 * static_cast<int64_t>(p.kv_heads);
  TORCH_CHECK_VALUE(heads >= 1 && p.kv_heads >= 1 && heads % p.kv_heads == 0, "qkv has ", qkv.size(d - 2),
                    " heads: with ", p.kv_heads, " KV heads that is no whole number of query heads for each");
  check_on(cos, "cos", dev);
  check_on(sin, "sin", dev);
  TORCH_CHECK_VALUE(cos.scalar_type() == torch::kFloat || cos.scalar_type() == k_cache.scalar_type(),
                    "cos must be float32 or of k_cache's type, got ", cos.scalar_type());
  check_type(sin, "sin", cos, "cos");
  TORCH_CHECK_VALUE(cos.dim() == 2 && cos.size(1) == dim && cos.is_contiguous(), "cos must be contiguous [positions, ",
                    dim, "], got ", cos.sizes());
  TORCH_CHECK_VALUE(sin.sizes() == cos.sizes() && sin.is_contiguous(), "sin must match cos");
  check_layout(cos, "cos");
  check_layout(sin, "sin");
  for (const auto& [w, name] : {std::pair<const OptTensor&, const char*>{q_norm, "q_norm"}, {k_norm, "k_norm"}}) {
    if (!w.has_value()) continue;
    check_on(*w, name, dev);
    check_type(*w, name, k_cache, "k_cache");
    TORCH_CHECK_VALUE(w->dim() == 1 && w->size(0) == dim, name, " must be [", dim, "], got ", w->sizes());
    check_layout(*w, name);
  }
  TORCH_CHECK_VALUE(std::isfinite(eps) && eps >= 0, "eps must not be negative, got ", eps);

  const c10::cuda::CUDAGuard guard(dev);
  auto shape = qkv.sizes().vec();
  shape[d - 2] = heads;
  const Tensor q = torch::empty(shape, k_cache.options());
  Tensor k;
  if (return_k) {
    shape[d - 2] = p.kv_heads;
    k = torch::empty(shape, k_cache.options());
  }
  if (b.tokens > 0) {
    a.heads = static_cast<int>(heads);
    a.kv_heads = p.kv_heads;
    a.head_dim = static_cast<int>(dim);
    a.tokens = b.tokens;
    a.batch = b.batch;
    a.q_len = b.q_len;
    a.cu_q = b.cu;
    a.qkv = qkv.data_ptr();
    a.qkv_stride[0] = b.token_stride;
    a.qkv_stride[1] = b.head_stride;
    a.q_norm = q_norm.has_value() ? q_norm->data_ptr() : nullptr;
    a.k_norm = k_norm.has_value() ? k_norm->data_ptr() : nullptr;
    a.eps = static_cast<float>(eps);
    a.cos_table = cos.data_ptr();
    a.sin_table = sin.data_ptr();
    a.rope_fp32 = cos.scalar_type() == torch::kFloat;
    a.rope_rows = as_int(cos.size(0), "positions");
    a.q_out = q.data_ptr();
    a.k_out = return_k ? k.data_ptr() : nullptr;
    a.k_cache = k_cache.data_ptr();
    a.v_cache = v_cache.data_ptr();
    for (int i = 0; i < 3; ++i) {
      a.k_stride[i] = p.k_stride[i];
      a.v_stride[i] = p.v_stride[i];
    }
    a.kv_lens = kv_lens.data_ptr<int>();
    a.block_table = block_table.data_ptr<int>();
    a.table_stride = p.table_stride;
    a.table_width = p.width;
    a.pages = p.pages;
    a.page_size = p.page_size;
    const Tensor st = status_of(dev);
    a.status = reinterpret_cast<uint32_t*>(st.data_ptr());
    C10_CUDA_CHECK(mkb_paged_append(&a, at::cuda::getCurrentCUDAStream().stream()));
  }
  if (!return_k) return pybind11::cast(q);
  return pybind11::cast(std::make_pair(q, k));
}

// First error that the operators met on a device since the last call, 0 if none.
int64_t serving_status(int64_t device) {
  const c10::Device dev(c10::kCUDA, static_cast<c10::DeviceIndex>(device));
  const c10::cuda::CUDAGuard guard(dev);
  C10_CUDA_CHECK(cudaDeviceSynchronize());
  const Tensor t = status_of(dev);
  const int64_t code = t.item<int>();
  if (code != 0) {
    t.zero_();
    C10_CUDA_CHECK(cudaDeviceSynchronize());
  }
  return code;
}

void register_serving(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("prompt_attention", &prompt_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("cu_seqlens"),
        py::arg("scale") = py::none(), py::arg("out") = py::none(), "causal attention of packed prompts");
  m.def("paged_attention", &paged_attention, py::arg("q"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("block_table"), py::arg("kv_lens"), py::arg("cu_q") = py::none(), py::arg("scale") = py::none(),
        py::arg("out") = py::none(), "attention of new tokens over a paged cache");
  m.def("paged_append", &paged_append, py::arg("qkv"), py::arg("k_cache"), py::arg("v_cache"), py::arg("block_table"),
        py::arg("kv_lens"), py::arg("cos"), py::arg("sin"), py::arg("cu_q") = py::none(),
        py::arg("q_norm") = py::none(), py::arg("k_norm") = py::none(), py::arg("eps") = 1e-6,
        py::arg("return_k") = false, "q/k norm, RoPE and the append to a paged cache");
  m.def("serving_status", &serving_status, "first error of the serving operators on a device since the last call");
}
