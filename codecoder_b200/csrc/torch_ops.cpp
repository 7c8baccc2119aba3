// Host side of the embedding, gradient-norm, group-norm and linear-attention operators: argument checks, outputs, workspaces
// and the calls of libbpc.so's C entry points, as a Python module on torch tensors.  In C++ because these calls are short:
// reading a list of 176 gradients through Python costs about 0.4 us per tensor, more than the kernels take; here 0.02 us.
// The module does not link to libbpc.so: _lib.py hands it the entry points of the library it loaded.
#include <cstdint>
#include <string>
#include <vector>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
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
  decltype(&bpc_group_norm_fwd) group_norm_fwd = nullptr;
  decltype(&bpc_group_norm_bwd) group_norm_bwd = nullptr;
  decltype(&bpc_group_norm_workspace_size) group_norm_workspace_size = nullptr;
  decltype(&bpc_linear_attention_fwd) linear_attention_fwd = nullptr;
  decltype(&bpc_linear_attention_bwd) linear_attention_bwd = nullptr;
  decltype(&bpc_linear_attention_step) linear_attention_step = nullptr;
  decltype(&bpc_linear_attention_workspace_size) linear_attention_workspace_size = nullptr;
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
  take(entry.group_norm_fwd, table, "bpc_group_norm_fwd");
  take(entry.group_norm_bwd, table, "bpc_group_norm_bwd");
  take(entry.group_norm_workspace_size, table, "bpc_group_norm_workspace_size");
  take(entry.linear_attention_fwd, table, "bpc_linear_attention_fwd");
  take(entry.linear_attention_bwd, table, "bpc_linear_attention_bwd");
  take(entry.linear_attention_step, table, "bpc_linear_attention_step");
  take(entry.linear_attention_workspace_size, table, "bpc_linear_attention_workspace_size");
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

// What would be lost without a word: the kernels have no forward-mode derivative, and a trace would keep their result as a
// constant.  Undefined tensors carry nothing.
void check_followed(const char* what, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " cannot be traced: its result would be a constant of the trace");
}

// x (B, ..., C) as (B, N, C) with contiguous channels; copies only where the layout asks for it
Tensor samples_of(const Tensor& x_in) {
  Tensor x = x_in.resolve_neg();
  const int64_t C = x.size(-1), N = x.numel() / (x.size(0) * C);
  x = x.reshape({x.size(0), N, C});
  return C > 1 && x.stride(2) != 1 ? x.contiguous() : x;
}

void check_norm(const Tensor& x, int64_t groups, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                at::ScalarType out) {
  check_cuda(x);
  const at::ScalarType in = x.scalar_type();
  TORCH_CHECK_TYPE(dtype_code(in) >= 0 && dtype_code(out) >= 0 && (in == out || in == at::kFloat),
                   "group_norm takes fp32, bf16 and fp16 features, and narrows fp32 ones only, got ", in, " -> ", out);
  TORCH_CHECK_VALUE(x.dim() >= 2, "group_norm: x must be (samples, ..., channels)");
  const int64_t C = x.size(-1);
  TORCH_CHECK_VALUE(C >= 1 && C <= (1 << 20) && groups >= 1 && C % groups == 0,
                    "group_norm: the channels (1 to 2^20) must divide into the groups, got ", C, " and ", groups);
  for (const auto& p : {weight, bias})
    if (p) {
      check_pair(x, *p);
      TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == C, "group_norm: weight and bias must be (channels)");
      TORCH_CHECK_TYPE(at::isFloatingType(p->scalar_type()), "group_norm: weight and bias must be floating point");
    }
}

// A per-channel vector as contiguous fp32; an undefined tensor where there is none
Tensor channel_vector(const std::optional<Tensor>& p) {
  return p ? p->to(at::kFloat).resolve_neg().contiguous() : Tensor();
}
const float* f32_or_null(const Tensor& t) { return t.defined() ? static_cast<const float*>(t.const_data_ptr()) : nullptr; }

Tensor norm_workspace(const Tensor& x, int64_t groups, bool backward) {
  return empty({static_cast<int64_t>(entry.group_norm_workspace_size(x.size(0), x.size(1), static_cast<int32_t>(x.size(2)),
                                                                     static_cast<int32_t>(groups), dtype_code(x.scalar_type()), backward))},
               at::kByte, x);
}

// y, and where `want_stats` is set the groups' statistics (samples, groups, 2)
std::tuple<Tensor, Tensor> group_norm_fwd(const Tensor& x_in, int64_t groups, const std::optional<Tensor>& weight,
                                                  const std::optional<Tensor>& bias, double eps, int64_t activation,
                                                  std::optional<at::ScalarType> dtype, bool want_stats) {
  at::NoGradGuard no_grad;
  const at::ScalarType out = dtype.value_or(x_in.scalar_type());
  check_norm(x_in, groups, weight, bias, out);
  const c10::cuda::CUDAGuard guard(x_in.device());
  Tensor y = empty(x_in.sizes(), out, x_in), stats;
  if (want_stats) stats = empty({x_in.size(0), groups, 2}, at::kFloat, x_in);
  if (y.numel() == 0) return {y, stats};
  Tensor x = samples_of(x_in), w = channel_vector(weight), b = channel_vector(bias), ws = norm_workspace(x, groups, false);
  check(entry.group_norm_fwd(x.const_data_ptr(), y.data_ptr(), want_stats ? static_cast<float*>(stats.data_ptr()) : nullptr,
                             f32_or_null(w), f32_or_null(b), x.size(0), x.size(1), static_cast<int32_t>(x.size(2)),
                             static_cast<int32_t>(groups), x.stride(0), x.stride(1), static_cast<float>(eps),
                             static_cast<int32_t>(activation), dtype_code(x.scalar_type()), dtype_code(out), ws.data_ptr(),
                             ws.numel(), stream_of(x)),
        "bpc_group_norm_fwd");
  return {y, stats};
}

// dx, dw, db; undefined where `want` says that one is not asked for
std::tuple<Tensor, Tensor, Tensor> group_norm_bwd(const Tensor& gy_in, const Tensor& x_in, const Tensor& stats,
                                                  int64_t groups, const std::optional<Tensor>& weight,
                                                  const std::optional<Tensor>& bias, int64_t activation, bool want_dx,
                                                  bool want_dw, bool want_db) {
  at::NoGradGuard no_grad;
  check_pair(x_in, gy_in);
  check_norm(x_in, groups, weight, bias, gy_in.scalar_type());
  TORCH_CHECK_VALUE(gy_in.sizes() == x_in.sizes(), "group_norm: gy must have x's shape");
  const c10::cuda::CUDAGuard guard(x_in.device());
  const int64_t C = x_in.size(-1);
  Tensor dx, dw, db;
  if (want_dx) dx = empty(x_in.sizes(), x_in.scalar_type(), x_in);
  if (want_dw) dw = empty({C}, at::kFloat, x_in);
  if (want_db) db = empty({C}, at::kFloat, x_in);
  if (x_in.numel() == 0) {
    if (want_dw) dw.zero_();
    if (want_db) db.zero_();
    return {dx, dw, db};
  }
  Tensor x = samples_of(x_in), gy = samples_of(gy_in), w = channel_vector(weight), b = channel_vector(bias);
  Tensor ws = norm_workspace(x, groups, true);
  check(entry.group_norm_bwd(gy.const_data_ptr(), x.const_data_ptr(), f32_or_null(stats), f32_or_null(w), f32_or_null(b),
                             want_dx ? dx.data_ptr() : nullptr,
                             want_dw ? static_cast<float*>(dw.data_ptr()) : nullptr,
                             want_db ? static_cast<float*>(db.data_ptr()) : nullptr, x.size(0), x.size(1),
                             static_cast<int32_t>(C), static_cast<int32_t>(groups), gy.stride(0), gy.stride(1), x.stride(0),
                             x.stride(1), static_cast<int32_t>(activation), dtype_code(x.scalar_type()),
                             dtype_code(gy.scalar_type()), ws.data_ptr(), ws.numel(), stream_of(x)),
        "bpc_group_norm_bwd");
  return {dx, dw, db};
}

// Head rows with contiguous elements
Tensor head_rows(const Tensor& t_in) {
  Tensor t = t_in.resolve_neg();
  return t.size(-1) > 1 && t.stride(-1) != 1 ? t.contiguous() : t;
}

int32_t check_heads(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, int64_t dims, const char* what) {
  check_cuda(q);
  for (const Tensor* t : {&k, &v, &log_decay}) check_pair(q, *t);
  const int32_t code = dtype_code(q.scalar_type());
  TORCH_CHECK_TYPE((code == BPC_DTYPE_F32 || code == BPC_DTYPE_BF16) && k.scalar_type() == q.scalar_type() &&
                       v.scalar_type() == q.scalar_type(),
                   what, " takes fp32 or bf16 q, k and v of one type, got ", q.scalar_type(), ", ", k.scalar_type(), ", ",
                   v.scalar_type());
  TORCH_CHECK_TYPE(log_decay.scalar_type() == at::kFloat, what, ": log_decay must be fp32, got ", log_decay.scalar_type());
  TORCH_CHECK_VALUE(q.dim() == dims && k.sizes() == q.sizes() && v.dim() == dims &&
                        v.sizes().slice(0, dims - 1) == q.sizes().slice(0, dims - 1),
                    what, ": q and k of one shape, v the same but for the head size (", dims, " dimensions), got ", q.sizes(),
                    ", ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_VALUE(q.size(-1) >= 1 && q.size(-1) <= 128 && v.size(-1) >= 1 && v.size(-1) <= 128, what,
                    ": head sizes must be 1 to 128, got ", q.size(-1), " and ", v.size(-1));
  TORCH_CHECK_VALUE(log_decay.dim() == 1 && log_decay.size(0) == q.size(-2), what, ": log_decay must be (heads)");
  return code;
}

// A (batch, heads, dk, dv) fp32 state as a contiguous, 16-byte aligned tensor
Tensor check_state(const Tensor& s, const Tensor& q, const Tensor& v, const char* what) {
  check_pair(q, s);
  TORCH_CHECK_TYPE(s.scalar_type() == at::kFloat, what, ": states are fp32, got ", s.scalar_type());
  TORCH_CHECK_VALUE(s.sizes() == at::IntArrayRef({q.size(0), q.size(-2), q.size(-1), v.size(-1)}), what,
                    ": a state must be (batch, heads, dk, dv), got ", s.sizes());
  Tensor t = s.resolve_neg().contiguous();
  return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 ? t.clone() : t;
}

Tensor check_lengths(const std::optional<Tensor>& lengths, const Tensor& q, const char* what) {
  if (!lengths) return Tensor();
  check_pair(q, *lengths);
  TORCH_CHECK_TYPE(lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong, what,
                   ": lengths must be int32 or int64, got ", lengths->scalar_type());
  TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == q.size(0), what, ": lengths must be (batch)");
  return lengths->contiguous();
}
int32_t length_bytes(const Tensor& t) { return t.defined() ? static_cast<int32_t>(t.element_size()) : 0; }
const void* data_or_null(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

void strides_of(const Tensor& t, int64_t*& at) {
  for (int64_t d = 0; d + 1 < t.dim(); ++d) *at++ = t.stride(d);
}

Tensor attention_workspace(const Tensor& q, const Tensor& v, int32_t code, bool backward) {
  return empty({static_cast<int64_t>(entry.linear_attention_workspace_size(
                   q.size(0), q.size(1), static_cast<int32_t>(q.size(2)), static_cast<int32_t>(q.size(3)),
                   static_cast<int32_t>(v.size(3)), code, backward))},
               at::kByte, q);
}

// o, where `want_state` is set the state after each sequence's last position, and the workspace
std::tuple<Tensor, Tensor, Tensor> linear_attention_fwd(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                                                const Tensor& log_decay, double scale, const std::optional<Tensor>& state_in,
                                                const std::optional<Tensor>& lengths_in, bool want_state) {
  at::NoGradGuard no_grad;
  const char* what = "linear_attention";
  const int32_t code = check_heads(q_in, k_in, v_in, log_decay, 4, what);
  const c10::cuda::CUDAGuard guard(q_in.device());
  Tensor state = state_in ? check_state(*state_in, q_in, v_in, what) : Tensor(), lengths = check_lengths(lengths_in, q_in, what);
  Tensor q = head_rows(q_in), k = head_rows(k_in), v = head_rows(v_in), decay = log_decay.resolve_neg().contiguous();
  Tensor o = empty(v.sizes(), v.scalar_type(), v), new_state;
  if (want_state) new_state = empty({q.size(0), q.size(2), q.size(3), v.size(3)}, at::kFloat, q);
  if (q.size(0) == 0 || q.size(2) == 0) return {o, new_state, Tensor()};
  Tensor ws = attention_workspace(q, v, code, false);
  int64_t strides[9], *at = strides;
  for (const Tensor* t : {&q, &k, &v}) strides_of(*t, at);
  check(entry.linear_attention_fwd(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), o.data_ptr(),
                                   f32_or_null(decay), f32_or_null(state),
                                   want_state ? static_cast<float*>(new_state.data_ptr()) : nullptr, data_or_null(lengths),
                                   length_bytes(lengths), q.size(0), q.size(1), static_cast<int32_t>(q.size(2)),
                                   static_cast<int32_t>(q.size(3)), static_cast<int32_t>(v.size(3)), strides,
                                   static_cast<float>(scale), code, ws.data_ptr(), ws.numel(), stream_of(q)),
        "bpc_linear_attention_fwd");
  return {o, new_state, ws};
}

// dq, dk, dv, and where `want_dstate` is set the gradient of the first state
std::tuple<Tensor, Tensor, Tensor, Tensor> linear_attention_bwd(
    const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& go_in, const Tensor& log_decay, double scale,
    const std::optional<Tensor>& state_in, const std::optional<Tensor>& grad_state_in, const Tensor& fwd_workspace,
    const std::optional<Tensor>& lengths_in, bool want_dstate) {
  at::NoGradGuard no_grad;
  const char* what = "linear_attention";
  const int32_t code = check_heads(q_in, k_in, v_in, log_decay, 4, what);
  check_pair(q_in, go_in);
  TORCH_CHECK_VALUE(go_in.sizes() == v_in.sizes() && go_in.scalar_type() == v_in.scalar_type(),
                    "linear_attention: go must be like v");
  const c10::cuda::CUDAGuard guard(q_in.device());
  Tensor state = state_in ? check_state(*state_in, q_in, v_in, what) : Tensor();
  Tensor grad_state = grad_state_in ? check_state(*grad_state_in, q_in, v_in, what) : Tensor();
  Tensor lengths = check_lengths(lengths_in, q_in, what), decay = log_decay.resolve_neg().contiguous();
  Tensor q = head_rows(q_in), k = head_rows(k_in), v = head_rows(v_in), go = head_rows(go_in);
  Tensor dq = empty(q.sizes(), q.scalar_type(), q), dk = at::empty_like(dq), dv = empty(v.sizes(), v.scalar_type(), v), dstate;
  if (want_dstate) dstate = empty({q.size(0), q.size(2), q.size(3), v.size(3)}, at::kFloat, q);
  if (q.size(0) == 0 || q.size(2) == 0) return {dq, dk, dv, dstate};
  Tensor ws = attention_workspace(q, v, code, true);
  int64_t strides[12], *at = strides;
  for (const Tensor* t : {&q, &k, &v, &go}) strides_of(*t, at);
  check(entry.linear_attention_bwd(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), go.const_data_ptr(),
                                   f32_or_null(decay), f32_or_null(state), f32_or_null(grad_state), data_or_null(fwd_workspace),
                                   data_or_null(lengths), length_bytes(lengths), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                   want_dstate ? static_cast<float*>(dstate.data_ptr()) : nullptr, q.size(0), q.size(1),
                                   static_cast<int32_t>(q.size(2)), static_cast<int32_t>(q.size(3)),
                                   static_cast<int32_t>(v.size(3)), strides, static_cast<float>(scale), code, ws.data_ptr(),
                                   ws.numel(), stream_of(q)),
        "bpc_linear_attention_bwd");
  return {dq, dk, dv, dstate};
}

// o; new_state (the state itself where none is given) is written
Tensor linear_attention_step(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& log_decay,
                             const Tensor& state, double scale, const std::optional<Tensor>& new_state) {
  at::NoGradGuard no_grad;
  const char* what = "linear_attention_step";
  check_followed(what, {&q_in, &k_in, &v_in, &log_decay, &state, new_state ? &*new_state : &state});
  const int32_t code = check_heads(q_in, k_in, v_in, log_decay, 3, what);
  const Tensor& to = new_state ? *new_state : state;
  for (const Tensor* s : {&state, &to}) {
    check_pair(q_in, *s);
    TORCH_CHECK_TYPE(s->scalar_type() == at::kFloat, what, ": states are fp32, got ", s->scalar_type());
    TORCH_CHECK_VALUE(s->sizes() == at::IntArrayRef({q_in.size(0), q_in.size(1), q_in.size(2), v_in.size(2)}), what,
                      ": a state must be (batch, heads, dk, dv), got ", s->sizes());
    TORCH_CHECK_VALUE(s->is_contiguous() && !s->is_neg(), what, ": states must be contiguous");
    TORCH_CHECK_VALUE(!s->requires_grad(), what, ": a state that requires a gradient (it is updated without one)");
  }
  const c10::cuda::CUDAGuard guard(q_in.device());
  Tensor q = head_rows(q_in), k = head_rows(k_in), v = head_rows(v_in), decay = log_decay.resolve_neg().contiguous();
  Tensor o = empty(v.sizes(), v.scalar_type(), v);
  if (o.numel() == 0) return o;
  int64_t strides[6], *at = strides;
  for (const Tensor* t : {&q, &k, &v}) strides_of(*t, at);
  float* written = static_cast<float*>(to.mutable_data_ptr());      // first: a state that shares its memory until written moves
  check(entry.linear_attention_step(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), o.data_ptr(),
                                    f32_or_null(decay), f32_or_null(state), written, q.size(0),
                                    static_cast<int32_t>(q.size(1)), static_cast<int32_t>(q.size(2)),
                                    static_cast<int32_t>(v.size(2)), strides, static_cast<float>(scale), code, stream_of(q)),
        "bpc_linear_attention_step");
  if (!to.is_inference()) to.unsafeGetTensorImpl()->bump_version();       // written behind autograd's back
  return o;
}

// ---- autograd: in C++ too, a forward and backward pass of small tensors through Python costs some 40 us more ----------------

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients that are not differentiable themselves: where a graph of them is asked for, its use is an error
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in;
  for (const Tensor& t : grads) in.push_back(t.defined() ? t.detach().set_requires_grad(true) : t);
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that is differentiable once", static_cast<int64_t>(in.size()));
  return (*error)(std::move(in));
}

bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const std::optional<Tensor>& t) { return t && t->requires_grad(); }

std::optional<Tensor> if_defined(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

struct GroupNorm : torch::autograd::Function<GroupNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, int64_t groups, const std::optional<Tensor>& weight,
                        const std::optional<Tensor>& bias, double eps, int64_t activation, std::optional<at::ScalarType> dtype) {
    auto [y, stats] = group_norm_fwd(x, groups, weight, bias, eps, activation, dtype, true);
    ctx->save_for_backward({x, stats, weight.value_or(Tensor()), bias.value_or(Tensor())});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["activation"] = activation;
    ctx->set_materialize_grads(false);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gy) {
    variable_list out(7);
    if (!gy[0].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &weight = saved[2], &bias = saved[3];
    size_t at = 0;                       // edges are counted over the tensors that were given
    const bool dx = ctx->needs_input_grad(at++), dw = weight.defined() && ctx->needs_input_grad(at++);
    const bool db = bias.defined() && ctx->needs_input_grad(at++);
    auto [gx, gw, gb] = group_norm_bwd(gy[0], saved[0], saved[1], ctx->saved_data["groups"].toInt(), if_defined(weight),
                                       if_defined(bias), ctx->saved_data["activation"].toInt(), dx, dw, db);
    const variable_list g = once({gx, dw ? gw.to(weight.scalar_type()) : gw, db ? gb.to(bias.scalar_type()) : gb});
    out[0] = g[0], out[2] = g[1], out[3] = g[2];
    return out;
  }
};

Tensor group_norm(const Tensor& x, int64_t groups, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                  double eps, int64_t activation, std::optional<at::ScalarType> dtype) {
  const Tensor none;
  check_followed("group_norm", {&x, weight ? &*weight : &none, bias ? &*bias : &none});
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias)))
    return GroupNorm::apply(x, groups, weight, bias, eps, activation, dtype);
  return std::get<0>(group_norm_fwd(x, groups, weight, bias, eps, activation, dtype, false));
}

struct LinearAttention : torch::autograd::Function<LinearAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                               double scale, const std::optional<Tensor>& state, const std::optional<Tensor>& lengths,
                               bool want_state) {
    auto [o, new_state, ws] = linear_attention_fwd(q, k, v, log_decay, scale, state, lengths, want_state);
    ctx->save_for_backward({q, k, v, log_decay, state.value_or(Tensor()), lengths.value_or(Tensor()), ws});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return want_state ? variable_list{o, new_state} : variable_list{o};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(8);
    const Tensor grad_state = g.size() > 1 ? g[1] : Tensor();
    if (!g[0].defined() && !grad_state.defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &state = saved[4];
    const Tensor go = g[0].defined() ? g[0] : at::zeros_like(v);
    auto [dq, dk, dv, dstate] = linear_attention_bwd(q, k, v, go, saved[3], ctx->saved_data["scale"].toDouble(), if_defined(state),
                                                     if_defined(grad_state), saved[6], if_defined(saved[5]),
                                                     state.defined() && ctx->needs_input_grad(4));
    const variable_list grads = once({dq, dk, dv, dstate});
    for (int i = 0; i < 3; ++i) out[i] = grads[i];
    out[5] = grads[3];
    return out;
  }
};

// o, and with want_state the state after each sequence's last position
std::tuple<Tensor, Tensor> linear_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, double scale,
                                            const std::optional<Tensor>& state, const std::optional<Tensor>& lengths,
                                            bool want_state) {
  const Tensor none;
  check_followed("linear_attention", {&q, &k, &v, &log_decay, state ? &*state : &none});
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(v) || wants_grad(state))) {
    const variable_list r = LinearAttention::apply(q, k, v, log_decay, scale, state, lengths, want_state);
    return {r[0], want_state ? r[1] : Tensor()};
  }
  auto [o, new_state, ws] = linear_attention_fwd(q, k, v, log_decay, scale, state, lengths, want_state);
  return {o, new_state};
}

}  // namespace

// What the build reads back, to compile again for another torch or Python, and to refuse loading there until then
__attribute__((used)) const char built_for[] = "torch_ops built for [" BUILT_FOR "]";

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  const auto release = py::call_guard<py::gil_scoped_release>();
  m.def("embed_lookup", &embed_lookup, release);
  m.def("embed_wgrad", &embed_wgrad, release);
  m.def("group_norm", &group_norm, release);
  m.def("linear_attention", &linear_attention, release);
  m.def("linear_attention_step", &linear_attention_step, release);
  m.def("grad_norm", &grad_norm);
  m.def("clip_grads", &clip_grads);
}
