// Torch-extension binding of attention to stored keys and values: the checks,
// allocations and calls behind b200_gemm.kv_cache_write, cache_attn, cross_attn
// and cross_attn_backward (b200_gemm/attention.py documents them).  The work is
// done by the C ABI (include/b200_gemm.h).  In C++ because a serving step's
// kernels last 3 to 10 us: the same checks in Python took 28 to 55 us a call.
//
// Errors: TypeError for a wrong element type, ValueError for a wrong shape,
// stride or device, B200GemmError for what the C ABI returns.  With a stream,
// memory comes from that stream's pool, so that its use there is ordered;
// outputs are also marked as used on the stream that was current.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <utility>

#include "b200_gemm.h"

namespace {

namespace py = pybind11;
using torch::Tensor;
using OptTensor = std::optional<Tensor>;
using OptStream = std::optional<std::pair<int64_t, int64_t>>;  // torch.cuda.Stream's stream_id and device_index

constexpr int64_t kHeadDim = 128;

// Messages by std::to_string and concatenation: number formatting of
// std::ostringstream crashed in this extension (as TORCH_CHECK's would).
std::string str(const char* s) { return s; }
std::string str(int64_t v) { return std::to_string(v); }
std::string str(double v) { return std::to_string(v); }
std::string str(const torch::Device& d) { return d.str(); }
std::string str(at::ScalarType t) { return c10::toString(t); }
std::string str(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}
template <typename... Parts>
std::string text(const Parts&... parts) {
  return (std::string() + ... + str(parts));
}
template <typename... Parts>
[[noreturn]] void bad_value(const Parts&... parts) {
  throw std::invalid_argument(text(parts...));
}
template <typename... Parts>
[[noreturn]] void bad_type(const Parts&... parts) {
  throw py::type_error(text(parts...));
}

void check(int rc, const std::string& what) {
  if (rc == B200_OK) return;
  const py::object cls = py::module_::import("b200_gemm._lib").attr("B200GemmError");
  const py::object error = cls(rc, what);
  PyErr_SetObject(cls.ptr(), error.ptr());
  throw py::error_already_set();
}

// None arrives as an undefined tensor.
void need(const char* name, const Tensor& t) {
  if (!t.defined()) bad_type(name, " must be a torch.Tensor, not None");
}

// A [batch, tokens, heads, 128] bf16 CUDA tensor as a b200_attn_view.
b200_attn_view view_of(const char* name, const Tensor& t) {
  need(name, t);
  if (t.scalar_type() != torch::kBFloat16) bad_type(name, " must be bfloat16, got ", t.scalar_type());
  if (!t.is_cuda() || t.dim() != 4) bad_value(name, " must be a 4-D CUDA tensor [batch, tokens, heads, 128]");
  if (t.size(3) != kHeadDim) bad_value(name, " must have head_dim 128, got ", t.size(3));
  if (t.numel() > 0) {
    if (t.stride(3) != 1) bad_value(name, " must be contiguous in its last dimension, got strides ", t.strides());
    for (int i = 0; i < 3; ++i) {
      if (t.size(i) > 1 && (t.stride(i) < kHeadDim || t.stride(i) % 8 != 0))
        bad_value(name, "'s strides must be multiples of 8, at least 128 (expanded tensors are not taken), got ",
                  t.strides());
    }
  }
  return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

const int32_t* lens_of(const char* name, const Tensor& t, int64_t batch, const torch::Device& device) {
  need(name, t);
  if (t.scalar_type() != torch::kInt) bad_type(name, " must be int32, got ", t.scalar_type());
  if (t.device() != device || t.dim() != 1 || t.size(0) != batch || (batch > 1 && t.stride(0) != 1))
    bad_value(name, " must be a contiguous [", batch, "] tensor on ", device);
  return static_cast<const int32_t*>(t.data_ptr());
}
const int32_t* lens_of(const char* name, const OptTensor& t, int64_t batch, const torch::Device& device) {
  return t.has_value() ? lens_of(name, *t, batch, device) : nullptr;
}

b200_kv_cache cache_of(const Tensor& k, const Tensor& v, const Tensor& k_scale, const Tensor& v_scale,
                       const Tensor& table, int64_t batch, const torch::Device& device) {
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"k_cache", k}, {"v_cache", v}}) {
    need(name, t);
    if (t.scalar_type() != torch::kFloat8_e4m3fn) bad_type(name, " must be float8_e4m3fn, got ", t.scalar_type());
    if (t.dim() != 4 || t.size(3) != kHeadDim || !t.is_contiguous() ||
        (t.size(2) != 16 && t.size(2) != 32 && t.size(2) != 64 && t.size(2) != 128))
      bad_value(name, " must be contiguous [num_pages, kv_heads, page_size, 128] with page_size 16, 32, 64 or 128, got ",
                t.sizes());
  }
  if (!v.sizes().equals(k.sizes())) bad_value("k_cache and v_cache must have the same shape");
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"k_scale", k_scale}, {"v_scale", v_scale}}) {
    need(name, t);
    if (t.scalar_type() != torch::kFloat) bad_type(name, " must be float32, got ", t.scalar_type());
    if (t.dim() != 2 || t.size(0) != k.size(0) || t.size(1) != k.size(1) || !t.is_contiguous())
      bad_value(name, " must be contiguous [", k.size(0), ", ", k.size(1), "], got ", t.sizes());
  }
  need("block_table", table);
  if (table.scalar_type() != torch::kInt) bad_type("block_table must be int32, got ", table.scalar_type());
  if (table.dim() != 2 || table.size(0) != batch || (table.size(1) > 1 && table.stride(1) != 1))
    bad_value("block_table must be row-major [", batch, ", max_pages], got ", table.sizes());
  for (const Tensor* t : {&k, &v, &k_scale, &v_scale, &table}) {
    if (t->device() != device) bad_value("the cache, its scales and the block table must be on ", device);
  }
  const int64_t most = table.size(1), pitch = batch > 1 ? table.stride(0) : most;
  if (pitch < most) bad_value("block_table's rows overlap");
  return {k.data_ptr(),
          v.data_ptr(),
          static_cast<float*>(k_scale.data_ptr()),
          static_cast<float*>(v_scale.data_ptr()),
          k.size(0),
          k.size(2),
          k.size(1),
          static_cast<const int32_t*>(table.data_ptr()),
          pitch,
          most};
}

void check_groups(int64_t heads, int64_t kv_heads) {
  if ((heads > 0 && kv_heads == 0) || (kv_heads > 0 && heads % kv_heads != 0))
    bad_value("the number of query heads (", heads, ") must be a multiple of the key/value heads (", kv_heads, ")");
}

float scale_of(const std::optional<double>& scale) {
  if (!scale.has_value()) return 0.08838834764831845f;  // 128 ** -0.5
  const float s = static_cast<float>(*scale);
  if (!(s > 0.0f) || !std::isfinite(s)) bad_value("scale must be positive and finite, got ", *scale);
  return s;
}

void check_like(const char* name, const Tensor& t, const Tensor& q) {
  if (!t.sizes().equals(q.sizes()) || t.device() != q.device())
    bad_value(name, " must be ", q.sizes(), " on ", q.device(), ", got ", t.sizes(), " on ", t.device());
}

// An output tensor of the caller's: like q, but not q itself (warps that share
// rows of q finish at different times).
void check_out(const Tensor& out, const Tensor& q) {
  check_like("out", out, q);
  if (out.numel() > 0 && out.data_ptr() == q.data_ptr()) bad_value("out may not be q's memory");
}

// Makes the tensors' device current and picks the stream of a call.
struct Scope {
  c10::cuda::CUDAGuard device;
  c10::cuda::CUDAStream current, stream;

  Scope(const torch::Device& d, const OptStream& s)
      : device(d), current(c10::cuda::getCurrentCUDAStream(d.index())), stream(current) {
    if (!s.has_value()) return;
    if (s->second != d.index()) bad_value("stream is on device ", s->second, ", the tensors on ", d);
    stream = c10::cuda::CUDAStream::unpack3(s->first, static_cast<c10::DeviceIndex>(s->second), c10::DeviceType::CUDA);
  }
  Tensor empty(at::IntArrayRef shape, at::ScalarType type) const {
    const auto options = at::TensorOptions().dtype(type).device(c10::Device(c10::kCUDA, stream.device_index()));
    if (stream == current) return at::empty(shape, options);
    const c10::cuda::CUDAStreamGuard guard(stream);
    Tensor t = at::empty(shape, options);
    if (t.numel() > 0) t.record_stream(current);
    return t;
  }
  // The allocator's blocks are 512-byte aligned.
  Tensor workspace(size_t bytes) const { return empty({static_cast<int64_t>(bytes)}, torch::kByte); }
};

void kv_cache_write(const Tensor& k, const Tensor& v, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale,
                    const Tensor& v_scale, const Tensor& block_table, const Tensor& seq_lens, const OptTensor& new_lens,
                    const OptStream& stream) {
  const b200_attn_view kk = view_of("k", k), vv = view_of("v", v);
  check_like("v", v, k);
  const int64_t batch = k.size(0), new_max = k.size(1);
  const b200_kv_cache cache = cache_of(k_cache, v_cache, k_scale, v_scale, block_table, batch, k.device());
  if (k.size(2) != cache.kv_heads) bad_value("k and v must have the cache's ", cache.kv_heads, " heads, got ", k.size(2));
  const int32_t* lens = lens_of("seq_lens", seq_lens, batch, k.device());
  const int32_t* fresh = lens_of("new_lens", new_lens, batch, k.device());
  const Scope scope(k.device(), stream);
  const int rc = b200_kv_cache_write(&kk, &vv, &cache, lens, fresh, batch, new_max, kHeadDim, scope.stream.stream());
  if (rc != B200_OK) check(rc, text("kv_cache_write batch=", batch, " new_max=", new_max, " kv_heads=", cache.kv_heads));
}

Tensor cache_attn(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale,
                  const Tensor& v_scale, const Tensor& block_table, const Tensor& seq_lens, const OptTensor& new_lens,
                  const std::optional<double>& scale_in, const OptTensor& out, const OptStream& stream) {
  const b200_attn_view qq = view_of("q", q);
  const int64_t batch = q.size(0), q_len = q.size(1), heads = q.size(2);
  const b200_kv_cache cache = cache_of(k_cache, v_cache, k_scale, v_scale, block_table, batch, q.device());
  check_groups(heads, cache.kv_heads);
  const int32_t* lens = lens_of("seq_lens", seq_lens, batch, q.device());
  const int32_t* fresh = lens_of("new_lens", new_lens, batch, q.device());
  const float scale = scale_of(scale_in);
  if (out.has_value()) check_out(*out, q);
  const Scope scope(q.device(), stream);
  const Tensor o = out.has_value() ? *out : scope.empty(q.sizes(), torch::kBFloat16);
  const b200_attn_view oo = view_of("out", o);
  size_t bytes = 0;
  int rc = b200_cache_attn_workspace_bytes(batch, q_len, heads, &cache, &bytes);
  if (rc == B200_OK) {
    const Tensor ws = scope.workspace(bytes);
    rc = b200_cache_attn(&qq, &cache, lens, fresh, &oo, batch, q_len, heads, kHeadDim, scale, ws.data_ptr(), bytes,
                         scope.stream.stream());
  }
  if (rc != B200_OK)
    check(rc, text("cache_attn batch=", batch, " q_len=", q_len, " heads=", heads, " kv_heads=", cache.kv_heads));
  return o;
}

struct CrossShape {
  int64_t batch, q_len, kv_len, heads, kv_heads;
};
CrossShape cross_shape(const Tensor& q, const Tensor& k, const Tensor& v) {
  if (!k.sizes().equals(v.sizes()) || k.size(0) != q.size(0) || k.device() != q.device() || v.device() != q.device())
    bad_value("k and v must have the same shape, and q's batch and device");
  check_groups(q.size(2), k.size(2));
  return {q.size(0), q.size(1), k.size(1), q.size(2), k.size(2)};
}
std::string cross_text(const char* name, const CrossShape& s) {
  return text(name, " batch=", s.batch, " q_len=", s.q_len, " kv_len=", s.kv_len, " heads=", s.heads, " kv_heads=",
              s.kv_heads);
}

std::pair<Tensor, OptTensor> cross_attn(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& kv_lens,
                                        const std::optional<double>& scale_in, const OptTensor& out, bool with_lse,
                                        const OptStream& stream) {
  const b200_attn_view qq = view_of("q", q), kk = view_of("k", k), vv = view_of("v", v);
  const CrossShape s = cross_shape(q, k, v);
  const int32_t* lens = lens_of("kv_lens", kv_lens, s.batch, q.device());
  const float scale = scale_of(scale_in);
  if (out.has_value()) check_out(*out, q);
  const Scope scope(q.device(), stream);
  const Tensor o = out.has_value() ? *out : scope.empty(q.sizes(), torch::kBFloat16);
  const b200_attn_view oo = view_of("out", o);
  OptTensor lse;
  if (with_lse) lse = scope.empty({s.batch, s.heads, s.q_len}, torch::kFloat);
  size_t bytes = 0;
  int rc = b200_cross_attn_workspace_bytes(s.batch, s.q_len, s.kv_len, s.heads, s.kv_heads, &bytes);
  if (rc == B200_OK) {
    Tensor ws;
    if (bytes > 0) ws = scope.workspace(bytes);
    rc = b200_cross_attn_bf16(&qq, &kk, &vv, lens, &oo, with_lse ? static_cast<float*>(lse->data_ptr()) : nullptr, s.batch,
                              s.q_len, s.kv_len, s.heads, s.kv_heads, kHeadDim, scale, bytes > 0 ? ws.data_ptr() : nullptr,
                              bytes, scope.stream.stream());
  }
  if (rc != B200_OK) check(rc, cross_text("cross_attn", s));
  return {o, lse};
}

std::tuple<Tensor, Tensor, Tensor> cross_attn_backward(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v,
                                                       const Tensor& out, const Tensor& lse, const OptTensor& kv_lens,
                                                       const std::optional<double>& scale_in, const OptStream& stream) {
  const b200_attn_view qq = view_of("q", q), kk = view_of("k", k), vv = view_of("v", v), oo = view_of("out", out),
                       dd = view_of("dout", dout);
  const CrossShape s = cross_shape(q, k, v);
  check_like("out", out, q);
  check_like("dout", dout, q);
  need("lse", lse);
  if (lse.scalar_type() != torch::kFloat) bad_type("lse must be float32, got ", lse.scalar_type());
  if (lse.dim() != 3 || lse.size(0) != s.batch || lse.size(1) != s.heads || lse.size(2) != s.q_len ||
      lse.device() != q.device() || !lse.is_contiguous())
    bad_value("lse must be contiguous [", s.batch, ", ", s.heads, ", ", s.q_len, "] on ", q.device(), ", got ", lse.sizes());
  const int32_t* lens = lens_of("kv_lens", kv_lens, s.batch, q.device());
  const float scale = scale_of(scale_in);
  const Scope scope(q.device(), stream);
  const Tensor dq = scope.empty(q.sizes(), torch::kBFloat16), dk = scope.empty(k.sizes(), torch::kBFloat16),
               dv = scope.empty(v.sizes(), torch::kBFloat16);
  const b200_attn_view dqv = view_of("dq", dq), dkv = view_of("dk", dk), dvv = view_of("dv", dv);
  size_t bytes = 0;
  int rc = b200_cross_attn_bwd_workspace_bytes(s.batch, s.q_len, s.kv_len, s.heads, s.kv_heads, &bytes);
  if (rc == B200_OK) {
    const Tensor ws = scope.workspace(bytes);
    rc = b200_cross_attn_bwd_bf16(&qq, &kk, &vv, &oo, &dd, static_cast<const float*>(lse.data_ptr()), lens, &dqv, &dkv, &dvv,
                                  s.batch, s.q_len, s.kv_len, s.heads, s.kv_heads, kHeadDim, scale, ws.data_ptr(), bytes,
                                  scope.stream.stream());
  }
  if (rc != B200_OK) check(rc, cross_text("cross_attn_backward", s));
  return {dq, dk, dv};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("kv_cache_write", &kv_cache_write, "Append keys and values to the paged e4m3 cache");
  m.def("cache_attn", &cache_attn, "Attention of the newest tokens over the paged e4m3 cache");
  m.def("cross_attn", &cross_attn, "Cross attention: (out, lse or None)");
  m.def("cross_attn_backward", &cross_attn_backward, "Gradients of cross attention: (dq, dk, dv)");
}
