// Python binding of the serving calls: argument checks, outputs and scratch from torch's allocator, the
// current stream, one call into the C ABI.  They are made once per layer and token, where the host's time
// counts: through ctypes, with the checks in Python, a call cost 14 us (append) to 23 us (attend), most of
// it attribute lookups and argument conversion; here 4 to 9 us, of which the launches are the larger part.
//
// The C ABI's functions come as addresses from the Python side (bind), so that whichever build of the
// library _lib.py has loaded is the one that runs.
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include "../../include/triton_b200.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using c10::optional;

decltype(&b200_attention_varlen_fwd) varlen_fwd = nullptr;
decltype(&b200_kv_append) kv_append = nullptr;
decltype(&b200_attention_decode) decode = nullptr;
decltype(&b200_attention_decode_workspace) decode_workspace = nullptr;
decltype(&b200_last_error) last_error = nullptr;

void bind(const std::map<std::string, uintptr_t>& address) {
  varlen_fwd = reinterpret_cast<decltype(varlen_fwd)>(address.at("b200_attention_varlen_fwd"));
  kv_append = reinterpret_cast<decltype(kv_append)>(address.at("b200_kv_append"));
  decode = reinterpret_cast<decltype(decode)>(address.at("b200_attention_decode"));
  decode_workspace = reinterpret_cast<decltype(decode_workspace)>(address.at("b200_attention_decode_workspace"));
  last_error = reinterpret_cast<decltype(last_error)>(address.at("b200_last_error"));
}

// the exceptions of ops.py: AssertionError for arguments, RuntimeError for the rest
void require(bool ok, const char* what) {
  if (ok) return;
  PyErr_SetString(PyExc_AssertionError, what);
  throw py::error_already_set();
}
[[noreturn]] void refuse(const std::string& what) {
  PyErr_SetString(PyExc_RuntimeError, what.c_str());
  throw py::error_already_set();
}
void check(int code, const char* what) {
  if (code) refuse(std::string("triton_b200 error [") + what + "] code " + std::to_string(code) + ": " + last_error());
}
void no_grad(const char* what, std::initializer_list<const Tensor*> ts) {
  // (torch.no_grad ends the recording of backward passes only: a dual tensor keeps its tangent under it)
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
    for (const Tensor* t : ts)
      if (t->_fw_grad(0).defined()) refuse(std::string(what) + " has no forward-mode derivative");
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : ts)
    if (t->requires_grad())
      refuse(std::string(what) + " has no backward: call it under torch.no_grad(), or attention() for training");
}
c10::Device one_device(std::initializer_list<const Tensor*> ts) {
  const c10::Device dev = (*ts.begin())->device();
  for (const Tensor* t : ts) {
    if (!t->is_cuda()) refuse("triton_b200 ops take CUDA tensors; there is no CPU fallback");
    if (t->device() != dev) refuse("all tensors must be on the same device");
  }
  return dev;
}
b200_stream_t stream_of(c10::Device dev) {
  return reinterpret_cast<b200_stream_t>(c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}
// what a call has written counts as changed for autograd's saved tensors (inference tensors keep no count)
void changed(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
bool half_type(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kHalf ? B200_F16 : B200_BF16; }
int small(int64_t n) {
  require(n <= 0x7fffffff, "a dimension is too large");
  return static_cast<int>(n);
}
// a vector of n int32
void ints(const Tensor& t, int64_t n, const char* what) {
  require(t.dim() == 1 && t.scalar_type() == at::kInt && t.size(0) == n && t.is_contiguous(), what);
}
Tensor output(const optional<Tensor>& out, const Tensor& q, c10::Device dev) {
  if (!out) return at::empty(q.sizes(), at::TensorOptions().dtype(q.scalar_type()).device(dev));
  require(out->sizes() == q.sizes() && out->scalar_type() == q.scalar_type() && out->device() == dev, "out= must look like q");
  no_grad("out=", {&*out});
  // q itself may take the output: what writes a row has read it.  Anything else that shares memory is read by others.
  at::assert_no_internal_overlap(*out);
  at::assert_no_partial_overlap(*out, q);
  return *out;
}
py::object result(const Tensor& o, const Tensor& m, bool stats) {
  return stats ? py::object(py::make_tuple(o, m)) : py::cast(o);
}

py::object attention_varlen(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu, bool causal,
                            double sm_scale, const optional<Tensor>& out, bool stats) {
  require(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes(), "q [T, Hq, D], k and v [T, Hkv, D]");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2), Hkv = k.size(1);
  require(k.size(0) == T && k.size(2) == D, "q, k and v must have the same rows and head dim");
  require(Hkv > 0 && Hq % Hkv == 0, "the query heads must be a multiple of the k/v heads");
  require(D == 64 || D == 128 || D == 256, "unsupported head dim");
  require(half_type(q) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "fp16 or bf16, one type");
  require(cu.dim() == 1 && cu.size(0) >= 1, "cu_seqlens holds one offset more than there are sequences");
  ints(cu, cu.size(0), "cu_seqlens must be a contiguous int32 tensor");
  no_grad("attention_varlen", {&q, &k, &v});
  const c10::Device dev = one_device({&q, &k, &v, &cu});
  c10::cuda::CUDAGuard guard(dev);
  const Tensor o = output(out, q, dev);
  if (out) {
    at::assert_no_overlap(o, k);
    at::assert_no_overlap(o, v);
  }
  Tensor m;
  if (stats) m = at::empty({Hq, T}, at::TensorOptions().dtype(at::kFloat).device(dev));
  check(varlen_fwd(stream_of(dev), q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), o.mutable_data_ptr(),
                   stats ? m.mutable_data_ptr<float>() : nullptr, cu.const_data_ptr<int>(), small(cu.size(0) - 1), small(T),
                   small(Hq), small(Hkv), small(D), q.strides().data(), k.strides().data(), v.strides().data(),
                   o.strides().data(), static_cast<float>(sm_scale), causal, dtype_of(q), out ? 2 : 1),
        "attention_varlen");
  if (out) changed({&*out});
  return result(o, m, stats);
}

struct Cache {
  int pages, heads, page, D;
};
Cache check_cache(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                  const Tensor& table, const Tensor& lens) {
  require(k_cache.dim() == 4 && v_cache.sizes() == k_cache.sizes(), "caches are [pages, Hkv, page size, D]");
  require(k_cache.scalar_type() == at::kFloat8_e4m3fn && v_cache.scalar_type() == at::kFloat8_e4m3fn,
          "caches hold float8_e4m3fn values");
  require(k_cache.is_contiguous() && v_cache.is_contiguous(), "caches must be contiguous");
  const Cache c{small(k_cache.size(0)), small(k_cache.size(1)), small(k_cache.size(2)), small(k_cache.size(3))};
  require(c.page == 16 || c.page == 32 || c.page == 64 || c.page == 128, "pages hold 16, 32, 64 or 128 tokens");
  require(c.D == 64 || c.D == 128 || c.D == 256, "a cache has head dim 64, 128 or 256");
  for (const Tensor* s : {&k_scale, &v_scale})
    require(s->dim() == 2 && s->scalar_type() == at::kFloat && s->size(0) == c.pages && s->size(1) == c.heads && s->is_contiguous(),
            "scales must be contiguous fp32 tensors [pages, Hkv]");
  require(table.dim() == 2 && table.scalar_type() == at::kInt && (table.stride(1) == 1 || table.size(1) <= 1),
          "page_table must be an int32 tensor [batch, pages of the longest sequence] with contiguous rows");
  ints(lens, table.size(0), "seq_lens must be a contiguous int32 tensor [batch]");
  return c;
}

void kv_cache_append(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                     const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens, const optional<Tensor>& cu) {
  const Cache c = check_cache(k_cache, v_cache, k_scale, v_scale, table, lens);
  const int64_t batch = table.size(0);
  require(k.dim() == 3 && k.size(1) == c.heads && k.size(2) == c.D && v.sizes() == k.sizes(),
          "k and v must be [T, Hkv, D] of the cache's heads");
  require(half_type(k) && v.scalar_type() == k.scalar_type(), "fp16 or bf16, one type");
  if (cu) ints(*cu, batch + 1, "cu_seqlens must be a contiguous int32 tensor [batch + 1]");
  else require(k.size(0) == batch, "without cu_seqlens every sequence has one new row");
  no_grad("kv_cache_append", {&k, &v, &k_cache, &v_cache, &k_scale, &v_scale});
  const c10::Device dev = one_device({&k_cache, &v_cache, &k_scale, &v_scale, &k, &v, &table, &lens});
  if (cu) one_device({&k, &*cu});
  c10::cuda::CUDAGuard guard(dev);
  check(kv_append(stream_of(dev), k_cache.mutable_data_ptr(), v_cache.mutable_data_ptr(), k_scale.mutable_data_ptr<float>(),
                  v_scale.mutable_data_ptr<float>(), c.pages, c.page, table.const_data_ptr<int>(), table.stride(0),
                  small(table.size(1)), lens.const_data_ptr<int>(), k.const_data_ptr(), v.const_data_ptr(),
                  cu ? cu->const_data_ptr<int>() : nullptr, small(batch), small(k.size(0)), c.heads, c.D, k.strides().data(),
                  v.strides().data(), dtype_of(k)),
        "kv_cache_append");
  changed({&k_cache, &v_cache, &k_scale, &v_scale});
}

py::object attention_decode(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale,
                            const Tensor& v_scale, const Tensor& table, const Tensor& lens, double sm_scale,
                            const optional<Tensor>& out, bool stats) {
  const Cache c = check_cache(k_cache, v_cache, k_scale, v_scale, table, lens);
  const int batch = small(table.size(0)), width = small(table.size(1));
  require(q.dim() == 3 && q.size(0) == batch && q.size(2) == c.D, "q must be [batch, Hq, D] of the cache's head dim");
  const int Hq = small(q.size(1));
  require(c.heads > 0 && Hq % c.heads == 0, "the query heads must be a multiple of the cache's heads");
  require(half_type(q), "fp16 or bf16");
  no_grad("attention_decode", {&q, &k_cache, &v_cache, &k_scale, &v_scale});
  const c10::Device dev = one_device({&q, &k_cache, &v_cache, &k_scale, &v_scale, &table, &lens});
  c10::cuda::CUDAGuard guard(dev);
  const Tensor o = output(out, q, dev);
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(dev);
  Tensor m, ws;
  if (stats) m = at::empty({batch, Hq}, f32);
  const size_t bytes = decode_workspace(batch, Hq, c.heads, c.D, c.page, width);
  if (bytes) ws = at::empty({static_cast<int64_t>(bytes / sizeof(float))}, f32);
  check(decode(stream_of(dev), q.const_data_ptr(), k_cache.const_data_ptr(), v_cache.const_data_ptr(),
               k_scale.const_data_ptr<float>(), v_scale.const_data_ptr<float>(), c.pages, c.page, table.const_data_ptr<int>(),
               table.stride(0), width, lens.const_data_ptr<int>(), o.mutable_data_ptr(),
               stats ? m.mutable_data_ptr<float>() : nullptr, batch, Hq, c.heads, c.D, q.strides().data(), o.strides().data(),
               static_cast<float>(sm_scale), dtype_of(q), bytes ? ws.mutable_data_ptr() : nullptr),
        "attention_decode");
  if (out) changed({&*out});
  return result(o, m, stats);
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
  m.def("bind", &bind);
  m.def("attention_varlen", &attention_varlen);
  m.def("kv_cache_append", &kv_cache_append);
  m.def("attention_decode", &attention_decode);
}
