// Host side of the embedding and gradient-norm operators: argument checks, outputs, workspaces and the calls of
// libbpc.so's C entry points, as a Python module on torch tensors.  In C++ because these calls are short: reading a
// list of 176 gradients through Python costs about 0.4 us per tensor, more than the kernels take; here 0.02 us.
// The module does not link to libbpc.so: _lib.py hands it the entry points of the library it loaded.
#include <cstdint>
#include <string>
#include <vector>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/extension.h>

#include "bpc.h"

namespace py = pybind11;
using at::Tensor;

namespace {

struct Entry {
  decltype(&bpc_last_error) last_error = nullptr;
  decltype(&bpc_embed_lookup) embed_lookup = nullptr;
  decltype(&bpc_embed_wgrad) embed_wgrad = nullptr;
  decltype(&bpc_embed_wgrad_workspace_size) embed_wgrad_workspace_size = nullptr;
  decltype(&bpc_grad_norm) grad_norm = nullptr;
  decltype(&bpc_clip_grads) clip_grads = nullptr;
  decltype(&bpc_grad_norm_workspace_size) grad_norm_workspace_size = nullptr;
} entry;

template <typename F>
void take(F& f, const py::dict& table, const char* name) {
  f = reinterpret_cast<F>(table[name].cast<uintptr_t>());
}

// table: entry point name -> address
void bind(const py::dict& table) {
  take(entry.last_error, table, "bpc_last_error");
  take(entry.embed_lookup, table, "bpc_embed_lookup");
  take(entry.embed_wgrad, table, "bpc_embed_wgrad");
  take(entry.embed_wgrad_workspace_size, table, "bpc_embed_wgrad_workspace_size");
  take(entry.grad_norm, table, "bpc_grad_norm");
  take(entry.clip_grads, table, "bpc_clip_grads");
  take(entry.grad_norm_workspace_size, table, "bpc_grad_norm_workspace_size");
}

void check(int rc, const char* what) {
  if (rc == 0) return;
  char msg[1024];
  entry.last_error(msg, sizeof(msg));
  TORCH_CHECK(false, what, " failed (", rc, "): ", msg);
}

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return BPC_DTYPE_F32;
    case at::kBFloat16: return BPC_DTYPE_BF16;
    case at::kHalf: return BPC_DTYPE_F16;
    default: return -1;
  }
}

void check_cuda(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "codecoder_b200 ops run on CUDA tensors only (no CPU path)");
}

void check_pair(const Tensor& a, const Tensor& b) {
  check_cuda(a);
  check_cuda(b);
  TORCH_CHECK_VALUE(a.device() == b.device(), "tensors are on different devices");
}

bpc_stream_t stream_of(const Tensor& t) {
  return reinterpret_cast<bpc_stream_t>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

// What a function of this file returns is not differentiable by itself: nothing of it is recorded.
Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, const Tensor& like) {
  return at::empty(shape, at::TensorOptions().dtype(dtype).device(like.device()));
}

int32_t check_embedding(const Tensor& ids, const Tensor& floats, at::ScalarType out) {
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong,
                   "token ids must be int32 or int64, got ", ids.scalar_type());
  TORCH_CHECK_TYPE(dtype_code(floats.scalar_type()) >= 0 && dtype_code(out) >= 0,
                   "embeddings are fp32, bf16 or fp16, got ", floats.scalar_type(), " -> ", out);
  return ids.scalar_type() == at::kLong ? 8 : 4;
}

// A (rows, C) tensor with contiguous channels and its row stride; copies only where the layout asks for it
int64_t row_stride(Tensor& t) {
  const int64_t rows = t.size(0), C = t.size(1);
  if ((C > 1 && t.stride(1) != 1) || (rows > 1 && t.stride(0) < C)) t = t.contiguous();
  return rows > 1 ? t.stride(0) : C;
}

Tensor embed_lookup(const Tensor& ids_in, const Tensor& weight_in, double scale, std::optional<at::ScalarType> dtype) {
  at::NoGradGuard no_grad;
  check_pair(weight_in, ids_in);
  const at::ScalarType out = dtype.value_or(weight_in.scalar_type());
  const int32_t id_bytes = check_embedding(ids_in, weight_in, out);
  TORCH_CHECK_VALUE(weight_in.dim() == 2, "embed_lookup: weight must be (V, C)");
  const c10::cuda::CUDAGuard guard(weight_in.device());
  Tensor weight = weight_in.resolve_neg(), ids = ids_in.contiguous();      // resolve_neg: a lazily negated view is copied
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(weight.size(1));
  Tensor y = empty(shape, out, weight);
  if (y.numel() == 0) return y;
  TORCH_CHECK_VALUE(weight.size(0) <= 0x7ffffffe && weight.size(1) <= (1 << 20), "embed_lookup: weight is too large");
  const int64_t ld = row_stride(weight);
  check(entry.embed_lookup(ids.const_data_ptr(), id_bytes, weight.const_data_ptr(), y.data_ptr(), ids.numel(),
                           static_cast<int32_t>(weight.size(0)), static_cast<int32_t>(weight.size(1)), ld,
                           static_cast<float>(scale), dtype_code(weight.scalar_type()), dtype_code(out), stream_of(weight)),
        "bpc_embed_lookup");
  return y;
}

Tensor embed_wgrad(const Tensor& gy_in, const Tensor& ids_in, int64_t n_tokens, double scale, at::ScalarType dtype) {
  at::NoGradGuard no_grad;
  check_pair(gy_in, ids_in);
  const int32_t id_bytes = check_embedding(ids_in, gy_in, dtype);
  TORCH_CHECK_VALUE(gy_in.dim() == ids_in.dim() + 1 && gy_in.sizes().slice(0, ids_in.dim()) == ids_in.sizes(),
                    "embed_wgrad: gy must be ids' shape with the channels added");
  const int64_t n = ids_in.numel(), C = gy_in.size(-1);
  TORCH_CHECK_VALUE(n_tokens >= 1 && n_tokens <= 0x7ffffffe && C <= (1 << 20),
                    "embed_wgrad: 1 <= n_tokens < 2^31 - 1 tokens, at most 2^20 channels");
  const c10::cuda::CUDAGuard guard(gy_in.device());
  Tensor dw = empty({n_tokens, C}, dtype, gy_in);
  if (C == 0) return dw;
  Tensor ids = ids_in.contiguous(), gy = gy_in.resolve_neg().reshape({n, C});
  const int64_t ld = row_stride(gy);
  const int32_t V = static_cast<int32_t>(n_tokens), Ci = static_cast<int32_t>(C);
  Tensor ws = empty({static_cast<int64_t>(entry.embed_wgrad_workspace_size(n, V, Ci))}, at::kByte, gy);
  check(entry.embed_wgrad(gy.const_data_ptr(), ids.const_data_ptr(), id_bytes, dw.data_ptr(), ws.data_ptr(), ws.numel(), n,
                          V, Ci, ld, static_cast<float>(scale), dtype_code(gy.scalar_type()), dtype_code(dtype), stream_of(gy)),
        "bpc_embed_wgrad");
  return dw;
}

// The tensors of a Python list, borrowed from it (the GIL is held meanwhile): a vector of tensors would count every
// reference up and down.
const Tensor& tensor_at(const py::list& list, size_t k, const char* what) {
  PyObject* o = PyList_GET_ITEM(list.ptr(), static_cast<Py_ssize_t>(k));
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, " takes a list of tensors, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

// Host arrays of a list of dense tensors on one GPU
struct TensorArrays {
  std::vector<void*> at;
  std::vector<int64_t> numel;
  std::vector<int32_t> dtype;
};

TensorArrays arrays_of(const py::list& list, const char* what) {
  const size_t n = list.size();
  TORCH_CHECK_VALUE(n > 0, what, " needs at least one tensor");
  const Tensor& first = tensor_at(list, 0, what);
  check_cuda(first);
  const at::Device device = first.device();
  TensorArrays a;
  a.at.resize(n);
  a.numel.resize(n);
  a.dtype.resize(n);
  for (size_t k = 0; k < n; ++k) {
    const Tensor& t = tensor_at(list, k, what);
    TORCH_CHECK_VALUE(t.device() == device, what, ": tensors are on different devices");
    const int32_t code = dtype_code(t.scalar_type());
    TORCH_CHECK_TYPE(t.layout() == at::kStrided && code >= 0, what, " takes dense fp32, bf16 and fp16 tensors, got ",
                     t.layout(), " ", t.scalar_type());
    TORCH_CHECK_VALUE(t.is_non_overlapping_and_dense(), what,
                      ": a tensor with gaps or overlaps between its elements (strides ", t.strides(), ")");
    a.numel[k] = t.numel();
    a.dtype[k] = code;
  }
  return a;
}

// The addresses of tensors that are read, or written.  One that is to be written and shares its memory until then (copy on
// write) gets its own here, so the written ones come first: what is read is then where it stays.
void take_addresses(TensorArrays& a, const py::list& list, bool written) {
  for (size_t k = 0; k < a.at.size(); ++k) {
    const Tensor& t = THPVariable_Unpack(PyList_GET_ITEM(list.ptr(), static_cast<Py_ssize_t>(k)));
    a.at[k] = written ? t.mutable_data_ptr() : const_cast<void*>(t.const_data_ptr());
  }
}

Tensor norm_workspace(const Tensor& like, size_t n) {
  return empty({static_cast<int64_t>(entry.grad_norm_workspace_size(static_cast<int32_t>(n)))}, at::kByte, like);
}

Tensor grad_norm(const py::list& ts) {
  TensorArrays a = arrays_of(ts, "grad_norm");
  const Tensor& first = tensor_at(ts, 0, "grad_norm");
  const c10::cuda::CUDAGuard guard(first.device());
  take_addresses(a, ts, false);
  Tensor norm = empty({}, at::kFloat, first), ws = norm_workspace(first, a.at.size());
  check(entry.grad_norm(a.at.data(), a.numel.data(), a.dtype.data(), static_cast<int32_t>(a.at.size()),
                        static_cast<float*>(norm.data_ptr()), ws.data_ptr(), ws.numel(), stream_of(first)),
        "bpc_grad_norm");
  return norm;
}

Tensor clip_grads(const py::list& ts, double max_norm, const std::optional<py::list>& out) {
  TensorArrays a = arrays_of(ts, "clip_grads");
  const py::list& outs = out ? *out : ts;
  const Tensor& first = tensor_at(ts, 0, "clip_grads");
  TensorArrays other;
  if (out) {
    TORCH_CHECK_VALUE(outs.size() == ts.size(), "clip_grads: out must hold one tensor of the same shape per gradient");
    other = arrays_of(outs, "clip_grads");
    TORCH_CHECK_VALUE(tensor_at(outs, 0, "clip_grads").device() == first.device(),
                      "clip_grads: tensors are on different devices");
    for (size_t k = 0; k < a.at.size(); ++k) {
      const Tensor &o = tensor_at(outs, k, "clip_grads"), &t = tensor_at(ts, k, "clip_grads");
      TORCH_CHECK_VALUE(o.sizes() == t.sizes(), "clip_grads: out must hold one tensor of the same shape per gradient");
      TORCH_CHECK_VALUE((o.is_contiguous() && t.is_contiguous()) || o.strides() == t.strides(),
                        "clip_grads: out must have the gradients' strides");
      TORCH_CHECK_VALUE(o.is_neg() == t.is_neg(), "clip_grads: a lazily negated view into one that is not, or the reverse");
    }
  }
  TensorArrays& b = out ? other : a;
  const c10::cuda::CUDAGuard guard(first.device());
  take_addresses(b, outs, true);
  if (out) take_addresses(a, ts, false);
  Tensor norm = empty({}, at::kFloat, first), ws = norm_workspace(first, a.at.size());
  check(entry.clip_grads(a.at.data(), b.at.data(), a.numel.data(), a.dtype.data(), b.dtype.data(),
                         static_cast<int32_t>(a.at.size()), max_norm, static_cast<float*>(norm.data_ptr()), ws.data_ptr(),
                         ws.numel(), stream_of(first)),
        "bpc_clip_grads");
  for (size_t k = 0; k < a.at.size(); ++k) {         // written behind autograd's back: count a new version
    const Tensor& t = tensor_at(outs, k, "clip_grads");
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  return norm;
}

}  // namespace

// What the build reads back, to compile again for another torch or Python, and to refuse loading there until then
__attribute__((used)) const char built_for[] = "torch_ops built for [" BUILT_FOR "]";

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  const auto release = py::call_guard<py::gil_scoped_release>();
  m.def("embed_lookup", &embed_lookup, release);
  m.def("embed_wgrad", &embed_wgrad, release);
  m.def("grad_norm", &grad_norm);
  m.def("clip_grads", &clip_grads);
}
