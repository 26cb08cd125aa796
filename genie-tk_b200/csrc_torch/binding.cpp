// Python binding of the training operators: checks, allocations and the call of the C ABI
// (include/genie_tk_b200.h) in one step, for calls that cost less than the interpreter's work
// around them (a list of some hundred gradients, a LayerNorm over a few rows).
//
// The entry points of libgenie_tk_b200.so are handed over by address (`bind`), so the module
// always runs on the library that genie_tk._lib loaded. Memory comes from PyTorch's caching
// allocator on the current stream, and the kernels run on the tensors' device and its current
// stream. Workspaces are allocated per call: two streams or two captured graphs never share one.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <numeric>
#include <optional>
#include <string>
#include <vector>

#include "../../include/genie_tk_b200.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

struct Api {
  decltype(&gtk_last_error_string) last_error = nullptr;
  decltype(&gtk_layernorm_forward) layernorm_forward = nullptr;
  decltype(&gtk_layernorm_backward) layernorm_backward = nullptr;
  decltype(&gtk_layernorm_backward_workspace_bytes) layernorm_backward_workspace_bytes = nullptr;
  decltype(&gtk_grad_norm_workspace_bytes) grad_norm_workspace_bytes = nullptr;
  decltype(&gtk_grad_norm) grad_norm = nullptr;
  decltype(&gtk_clip_grad_norm) clip_grad_norm = nullptr;
  decltype(&gtk_embedding_forward) embedding_forward = nullptr;
  decltype(&gtk_embedding_backward) embedding_backward = nullptr;
  decltype(&gtk_embedding_backward_workspace_bytes) embedding_backward_workspace_bytes = nullptr;
} api;

template <typename F>
void bind_one(const py::dict& addresses, const char* name, F* out) {
  if (!addresses.contains(name)) throw py::key_error(name);
  *out = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

void bind(const py::dict& d) {
  bind_one(d, "gtk_last_error_string", &api.last_error);
  bind_one(d, "gtk_layernorm_forward", &api.layernorm_forward);
  bind_one(d, "gtk_layernorm_backward", &api.layernorm_backward);
  bind_one(d, "gtk_layernorm_backward_workspace_bytes", &api.layernorm_backward_workspace_bytes);
  bind_one(d, "gtk_grad_norm_workspace_bytes", &api.grad_norm_workspace_bytes);
  bind_one(d, "gtk_grad_norm", &api.grad_norm);
  bind_one(d, "gtk_clip_grad_norm", &api.clip_grad_norm);
  bind_one(d, "gtk_embedding_forward", &api.embedding_forward);
  bind_one(d, "gtk_embedding_backward", &api.embedding_backward);
  bind_one(d, "gtk_embedding_backward_workspace_bytes", &api.embedding_backward_workspace_bytes);
}

const std::string kPrefix = "genie_tk (B200): ";

[[noreturn]] void type_error(const std::string& m) { throw py::type_error(kPrefix + m); }
[[noreturn]] void value_error(const std::string& m) { throw py::value_error(kPrefix + m); }

void check(int rc, const char* what) {
  if (rc) {
    const char* m = api.last_error();
    throw std::runtime_error(std::string(what) + " failed (" + std::to_string(rc) + "): " + (m ? m : ""));
  }
}

// The dtype code of a tensor's elements, or -1.
int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat:
      return GTK_F32;
    case at::kBFloat16:
      return GTK_BF16;
    case at::kHalf:
      return GTK_F16;
    default:
      return -1;
  }
}

std::string name_of(at::ScalarType t) { return c10::toString(t); }

int dtype_code(const Tensor& t, const char* name) {
  const int c = code_of(t.scalar_type());
  if (c < 0)
    type_error(std::string(name) + " must be float32, bfloat16 or float16, got " + name_of(t.scalar_type()));
  return c;
}

// The operators have no forward-mode formula: a tangent that they would lose is an error. Tensors have
// tangents while a level of forward mode is open only.
bool forward_mode() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }

void refuse_tangent(const Tensor& t, const char* name) {
  if (!t.defined() || !t._fw_grad(0).defined()) return;
  PyErr_SetString(PyExc_NotImplementedError,
                  (kPrefix + name + " has a tangent, and this operator no forward-mode derivative").c_str());
  throw py::error_already_set();
}

void refuse_tangents(std::initializer_list<std::pair<const Tensor*, const char*>> tensors) {
  if (!forward_mode()) return;
  for (const auto& t : tensors)
    if (t.first) refuse_tangent(*t.first, t.second);
}

const Tensor* given(const OptTensor& t) { return t ? &*t : nullptr; }

void require_cuda(const Tensor& t, const char* name) {
  if (!t.is_cuda())
    throw std::runtime_error(kPrefix + name + " must be a CUDA tensor; this package has no CPU path");
  if (t.layout() != at::kStrided || t.is_neg()) type_error(std::string(name) + " must be a dense tensor");
}

void same_device(const Tensor& t, c10::Device d, const char* name) {
  if (!t.is_cuda() || t.device() != d)
    throw std::runtime_error(kPrefix + name + " must be a CUDA tensor on device " + std::to_string(d.index()));
  if (t.layout() != at::kStrided || t.is_neg()) type_error(std::string(name) + " must be a dense tensor");
}

std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

Tensor contiguous(const Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }

void* stream_of(c10::Device d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

Tensor scratch(size_t bytes, const Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ---- LayerNorm ------------------------------------------------------------------------------

// The rows of x [*, D]: contiguous, or strided leading axes that merge into at most three
// (`used`), else a contiguous copy of x.
Tensor row_view(const Tensor& x, gtk_rows* rows, bool* used) {
  *used = false;
  if (x.is_contiguous()) return x;
  const int64_t last = x.dim() - 1;
  if (x.stride(last) != 1 && x.size(last) != 1) return x.contiguous();
  int64_t size[3], stride[3];
  int n = 0;
  for (int64_t i = 0; i < last; ++i) {
    if (x.size(i) == 1) continue;
    if (n && stride[n - 1] == x.stride(i) * x.size(i)) {
      size[n - 1] *= x.size(i);
      stride[n - 1] = x.stride(i);
      continue;
    }
    if (n == 3) return x.contiguous();
    size[n] = x.size(i);
    stride[n++] = x.stride(i);
  }
  for (int i = 0; i < 3; ++i) {
    const int k = i - (3 - n);
    rows->size[i] = k < 0 ? 1 : size[k];
    rows->stride[i] = k < 0 ? 0 : stride[k];
  }
  *used = true;
  return x;
}

// A parameter of LayerNorm, contiguous; sets *code to its dtype code (-1 while there is none).
Tensor parameter(const OptTensor& p, const Tensor& x, const char* name, int* code) {
  if (!p || !p->defined()) return Tensor();
  same_device(*p, x.device(), name);
  const int64_t D = x.size(-1);
  if (p->numel() != D)
    value_error(std::string(name) + " must have " + std::to_string(D) + " elements, got " + shape_of(*p));
  const int c = code_of(p->scalar_type());
  if (c < 0 || (c != GTK_F32 && p->scalar_type() != x.scalar_type()) || (*code >= 0 && c != *code))
    type_error("LayerNorm parameters must both be float32 or " + name_of(x.scalar_type()) + ", got " +
               name_of(p->scalar_type()));
  *code = c;
  return contiguous(*p);
}

py::tuple layernorm_forward(const Tensor& x_in, const OptTensor& weight, const OptTensor& bias, double eps) {
  require_cuda(x_in, "x");
  if (x_in.dim() < 1 || x_in.size(-1) < 1) value_error("x must have a last axis of at least one element");
  const int xt = dtype_code(x_in, "x");
  refuse_tangents({{&x_in, "x"}, {given(weight), "weight"}, {given(bias), "bias"}});
  at::NoGradGuard no_grad;
  c10::cuda::CUDAGuard guard(x_in.device());
  int wt = -1;
  const Tensor w = parameter(weight, x_in, "weight", &wt), b = parameter(bias, x_in, "bias", &wt);
  const int64_t D = x_in.size(-1);
  Tensor y = at::empty(x_in.sizes(), x_in.options());
  const auto lead = x_in.sizes().slice(0, x_in.dim() - 1);
  Tensor mean = at::empty(lead, x_in.options().dtype(at::kFloat));
  Tensor rstd = at::empty(lead, mean.options());
  const int64_t n = mean.numel();
  if (n) {
    gtk_rows rows;
    bool used;
    const Tensor x = row_view(x_in, &rows, &used);
    check(api.layernorm_forward(x.data_ptr(), used ? &rows : nullptr, xt, ptr(w), ptr(b), wt < 0 ? xt : wt,
                                y.data_ptr(), static_cast<float*>(mean.data_ptr()),
                                static_cast<float*>(rstd.data_ptr()), n, D, static_cast<float>(eps),
                                stream_of(x.device())),
          "gtk_layernorm_forward");
  }
  return py::make_tuple(std::move(y), std::move(mean), std::move(rstd));
}

// Whether t has x's leading axes (and perhaps a last one of one), or all rows in one axis.
bool one_per_row(const Tensor& t, const Tensor& x) {
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  const bool keepdim = t.dim() == x.dim() && t.size(-1) == 1;
  return (keepdim ? t.sizes().slice(0, x.dim() - 1) : t.sizes()) == lead ||
         (t.dim() == 1 && t.numel() == c10::multiply_integers(lead));
}

py::tuple layernorm_backward(const Tensor& dy_in, const Tensor& x_in, const OptTensor& weight, const Tensor& mean_in,
                             const Tensor& rstd_in, bool need_weight, bool need_bias) {
  require_cuda(x_in, "x");
  const int xt = dtype_code(x_in, "x");
  same_device(dy_in, x_in.device(), "dy");
  same_device(mean_in, x_in.device(), "mean");
  same_device(rstd_in, x_in.device(), "rstd");
  if (dy_in.sizes() != x_in.sizes() || dy_in.scalar_type() != x_in.scalar_type())
    value_error("dy must have x's shape and type, got " + shape_of(dy_in) + " " + name_of(dy_in.scalar_type()));
  if (x_in.dim() < 1 || x_in.size(-1) < 1) value_error("x must have a last axis of at least one element");
  const int64_t D = x_in.size(-1), n = mean_in.numel();
  if (n * D != x_in.numel() || !one_per_row(mean_in, x_in) || !one_per_row(rstd_in, x_in))
    value_error("mean and rstd must have one element for each row of x, in x's leading axes or in one, got " +
                shape_of(mean_in) + " and " + shape_of(rstd_in));
  if (mean_in.scalar_type() != at::kFloat || rstd_in.scalar_type() != at::kFloat)
    type_error("mean and rstd must be float32");
  refuse_tangents({{&dy_in, "dy"}, {&x_in, "x"}, {given(weight), "weight"}, {&mean_in, "mean"}, {&rstd_in, "rstd"}});
  at::NoGradGuard no_grad;
  c10::cuda::CUDAGuard guard(x_in.device());
  int wt = -1;
  const Tensor w = parameter(weight, x_in, "weight", &wt);
  if (wt < 0) wt = xt;
  const auto options = x_in.options().dtype(w.defined() ? w.scalar_type() : x_in.scalar_type());
  Tensor dx = at::empty(x_in.sizes(), x_in.options()), dw, db;
  if (need_weight) dw = n ? at::empty({D}, options) : at::zeros({D}, options);
  if (need_bias) db = n ? at::empty({D}, options) : at::zeros({D}, options);
  if (n) {
    const size_t bytes = need_weight || need_bias ? api.layernorm_backward_workspace_bytes(n, D) : 0;
    Tensor ws;
    if (bytes) ws = scratch(bytes, x_in);
    const Tensor mean = contiguous(mean_in), rstd = contiguous(rstd_in);
    gtk_rows xr, dr;
    bool xu, du;
    const Tensor x = row_view(x_in, &xr, &xu), dy = row_view(dy_in, &dr, &du);
    check(api.layernorm_backward(dy.data_ptr(), du ? &dr : nullptr, x.data_ptr(), xu ? &xr : nullptr, xt, ptr(w), wt,
                                 static_cast<const float*>(mean.data_ptr()),
                                 static_cast<const float*>(rstd.data_ptr()), dx.data_ptr(), ptr(dw), ptr(db), ptr(ws),
                                 bytes, n, D, stream_of(x.device())),
          "gtk_layernorm_backward");
  }
  return py::make_tuple(dx, need_weight ? py::cast(dw) : py::none(), need_bias ? py::cast(db) : py::none());
}

// ---- The global gradient norm -----------------------------------------------------------------

struct Gradients {
  py::object list, out_list;  // hold the items until the call has been queued (a sequence may have made them for it)
  std::vector<const void*> in;
  std::vector<void*> out;
  std::vector<int64_t> numel;
  std::vector<int> in_type, out_type;
  std::vector<Tensor> keep;                           // copies of strided gradients
  std::vector<std::pair<Tensor, Tensor>> write_back;  // (gradient, its clipped copy)
  // Tensors to be written, and how many of them had their versions counted as the list was read (a loop
  // of its own behind the call costs 2.5 us for 464 of them). A refused call has written none.
  PyObject** counted = nullptr;
  Py_ssize_t n_counted = 0;
  Gradients() = default;
  Gradients(const Gradients&) = delete;
  ~Gradients() {
    for (Py_ssize_t i = 0; i < n_counted; ++i) {
      c10::TensorImpl* t = THPVariable_Unpack(counted[i]).unsafeGetTensorImpl();
      if (t->is_inference()) continue;
      c10::VariableVersion v = t->version_counter();  // shares the tensor's counter
      v.set_version(v.current_version() - 1);
    }
  }
  void done() { n_counted = 0; }
};

// Dense, and holding its values as they are (not a lazily negated view).
bool dense(const c10::TensorImpl* t) {
  return t->layout() == at::kStrided && !t->key_set().has(c10::DispatchKey::Negative);
}

// Item i of a list of tensors. (Reads the TensorImpl directly from here on: a list may hold
// hundreds of gradients, and every call on a Tensor counts: 1 us of 27 for 464 of them where this is
// not inlined.)
__attribute__((always_inline)) inline c10::TensorImpl* tensor_at(PyObject* o, const char* name, Py_ssize_t i) {
  if (!THPVariable_Check(o)) type_error(std::string(name) + "[" + std::to_string(i) + "] is not a tensor");
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.defined()) type_error(std::string(name) + "[" + std::to_string(i) + "] is not a tensor");
  return t.unsafeGetTensorImpl();
}

Tensor handle(c10::TensorImpl* t) {
  return Tensor(c10::intrusive_ptr<c10::TensorImpl, c10::UndefinedTensorImpl>::reclaim_copy(t));
}

// Has the tensors that are a few places ahead in the list brought near: their objects, and of
// nearer ones what the objects point to.
void prefetch(PyObject** items, Py_ssize_t i, Py_ssize_t n) {
  if (i + 12 < n) __builtin_prefetch(items[i + 12]);
  if (i + 8 < n) __builtin_prefetch(reinterpret_cast<char*>(items[i + 8]) + 64);
  if (i + 6 < n && THPVariable_CheckExact(items[i + 6])) {
    const char* t = reinterpret_cast<const char*>(THPVariable_Unpack(items[i + 6]).unsafeGetTensorImpl());
    __builtin_prefetch(t);
    __builtin_prefetch(t + 64);
    __builtin_prefetch(t + 128);
  }
}

// The memory that a strided tensor stands for: runs of `run` bytes, at every combination of the axes'
// steps. The axes' strides ascend.
struct Memory {
  struct Axis {
    int64_t size, stride;  // in bytes
  };
  int64_t at, run;
  std::vector<Axis> axes;
  std::vector<int64_t> span;  // [k]: bytes that the first k axes reach over
  Py_ssize_t index;           // in its list
  bool output;
  int64_t end() const { return at + span.back(); }
};

Memory memory_of(const c10::TensorImpl* t, Py_ssize_t index, bool output) {
  const int64_t bytes = static_cast<int64_t>(t->itemsize());
  Memory m{reinterpret_cast<int64_t>(t->data()), bytes, {}, {}, index, output};
  std::vector<Memory::Axis> axes;
  for (int64_t i = 0; i < t->dim(); ++i)
    if (t->size(i) != 1 && t->stride(i) != 0) axes.push_back({t->size(i), t->stride(i) * bytes});
  std::sort(axes.begin(), axes.end(), [](auto& a, auto& b) { return a.stride < b.stride; });
  for (const auto& a : axes) {
    if (m.axes.empty() && a.stride == m.run)
      m.run *= a.size;
    else if (!m.axes.empty() && a.stride == m.axes.back().stride * m.axes.back().size)
      m.axes.back().size *= a.size;
    else
      m.axes.push_back(a);
  }
  m.span.push_back(m.run);
  for (const auto& a : m.axes) m.span.push_back(m.span.back() + (a.size - 1) * a.stride);
  return m;
}

int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }

// Whether the first ka axes of `a`, from address `at_a` on, share a byte with the first kb axes of `b`.
// `steps` bounds how often one is taken apart; without an answer by then, yes.
bool meet(const Memory& a, int64_t at_a, size_t ka, const Memory& b, int64_t at_b, size_t kb, int64_t* steps) {
  if (at_a + a.span[ka] <= at_b || at_b + b.span[kb] <= at_a) return false;
  if (ka == 0 && kb == 0) return true;
  // all runs begin at at_a or at_b plus multiples of g (columns of one matrix: its rows): the runs of
  // the one lie in the gaps of the other, or may meet
  int64_t g = 0;
  for (size_t k = 0; k < ka; ++k) g = std::gcd(g, a.axes[k].stride);
  for (size_t k = 0; k < kb; ++k) g = std::gcd(g, b.axes[k].stride);
  const int64_t r = (at_b - at_a) - floor_div(at_b - at_a, g) * g;
  if (r >= a.run && r + b.run <= g) return false;
  if (--*steps < 0) return true;
  // the parts of the wider one that reach into the other
  if (ka == 0 || (kb && b.span[kb] > a.span[ka])) return meet(b, at_b, kb, a, at_a, ka, steps);
  const auto& axis = a.axes[ka - 1];
  const int64_t first = std::max<int64_t>(0, floor_div(at_b - at_a - a.span[ka - 1], axis.stride) + 1);
  const int64_t last = std::min(axis.size - 1, floor_div(at_b + b.span[kb] - at_a - 1, axis.stride));
  for (int64_t i = first; i <= last; ++i)
    if (meet(a, at_a + i * axis.stride, ka - 1, b, at_b, kb, steps)) return true;
  return false;
}

constexpr int64_t kMeetSteps = int64_t(1) << 20;  // of a call: some 10 ms

// Whether a tensor (without strides of zero) holds an element of memory more than once.
bool repeats(const Memory& m, int64_t* steps) {
  for (size_t k = 0; k < m.axes.size(); ++k)
    for (int64_t d = 1; d < m.axes[k].size && d * m.axes[k].stride < m.span[k]; ++d)
      if (meet(m, m.at, k, m, m.at + d * m.axes[k].stride, k, steps)) return true;
  return false;
}

// Refuses overlaps that the library cannot see, as it gets copies of the strided gradients: in place, of
// any two gradients; with outputs, of a `copied` gradient and any output.
__attribute__((noinline)) void check_memory(PyObject** items, PyObject** out_items, Py_ssize_t n,
                                            const std::vector<Py_ssize_t>& copied, int64_t* steps) {
  std::vector<Memory> all;
  auto add = [&](c10::TensorImpl* t, Py_ssize_t i, bool output) {
    if (t->numel()) all.push_back(memory_of(t, i, output));
  };
  if (out_items) {
    for (Py_ssize_t i : copied) add(tensor_at(items[i], "grads", i), i, false);
    for (Py_ssize_t i = 0; i < n; ++i) add(tensor_at(out_items[i], "out", i), i, true);
  } else {
    for (Py_ssize_t i = 0; i < n; ++i) add(tensor_at(items[i], "grads", i), i, false);
  }
  std::sort(all.begin(), all.end(), [](auto& a, auto& b) { return a.at < b.at; });
  for (size_t i = 0; i < all.size(); ++i)
    for (size_t j = i + 1; j < all.size() && all[j].at < all[i].end(); ++j) {
      const Memory &a = all[i], &b = all[j];
      if (out_items && a.output == b.output) continue;
      if (meet(a, a.at, a.axes.size(), b, b.at, b.axes.size(), steps))
        throw std::runtime_error(kPrefix + (a.output ? "out[" : "grads[") + std::to_string(a.index) + "] and " +
                                 (b.output ? "out[" : "grads[") + std::to_string(b.index) +
                                 "] overlap (the same tensor twice?)");
    }
}

// A contiguous copy of gradient i, whose clipped values are copied back behind the call.
__attribute__((noinline)) c10::TensorImpl* copy_strided(c10::TensorImpl* t, Py_ssize_t i, bool clip, int64_t* steps,
                                                        Gradients* g) {
  if (clip && t->numel() &&
      (at::has_internal_overlap(t) == at::MemOverlap::Yes || repeats(memory_of(t, i, false), steps)))
    value_error("grads[" + std::to_string(i) + "] holds an element more than once and cannot be clipped in place");
  g->keep.push_back(handle(t).contiguous());
  if (clip) g->write_back.emplace_back(handle(t), g->keep.back());
  return g->keep.back().unsafeGetTensorImpl();
}

// Checks the lists, fills the arrays and makes the gradients' device current. `outs` NULL: in place
// (`clip`) or the norm alone. What will be written is asked for as mutable, so that a lazy clone gets
// memory of its own.
c10::Device collect(const py::sequence& grads, const py::object* outs, bool clip, Gradients* g,
                    c10::cuda::OptionalCUDAGuard* guard) {
  g->list = py::reinterpret_steal<py::object>(PySequence_Fast(grads.ptr(), "grads must be a sequence"));
  if (!g->list) throw py::error_already_set();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(g->list.ptr());
  if (n == 0) value_error("the list of gradients is empty");
  PyObject** items = PySequence_Fast_ITEMS(g->list.ptr());
  PyObject** out_items = nullptr;
  if (outs) {
    g->out_list = py::reinterpret_steal<py::object>(PySequence_Fast(outs->ptr(), "out must be a sequence"));
    if (!g->out_list) throw py::error_already_set();
    if (PySequence_Fast_GET_SIZE(g->out_list.ptr()) != n) value_error("out must have one tensor for each gradient");
    out_items = PySequence_Fast_ITEMS(g->out_list.ptr());
  }
  g->in.resize(n);
  g->numel.resize(n);
  g->in_type.resize(n);
  g->counted = outs ? out_items : items;
  if (outs) {
    g->out.resize(n);
    g->out_type.resize(n);
  }
  require_cuda(handle(tensor_at(items[0], "grads", 0)), "grads[0]");
  const c10::Device device = tensor_at(items[0], "grads", 0)->device();
  guard->set_device(device);
  std::vector<Py_ssize_t> copied;
  int64_t steps = kMeetSteps;
  Py_ssize_t i = 0;
  try {
    for (; i < n; ++i) {
      prefetch(items, i, n);
      c10::TensorImpl *t = tensor_at(items[i], "grads", i), *written = t;
      if (t->device() != device)
        throw std::runtime_error(kPrefix + "all gradients must be CUDA tensors on one device");
      if (!dense(t)) type_error("gradients must be dense tensors");
      const at::ScalarType st = c10::typeMetaToScalarType(t->dtype());
      const int code = code_of(st);
      if (code < 0) type_error("gradients must be float32, bfloat16 or float16, got " + name_of(st));
      const bool plain = t->is_contiguous();
      if (outs) {
        prefetch(out_items, i, n);
        c10::TensorImpl* o = tensor_at(out_items[i], "out", i);
        if (o->device() != device || !dense(o))
          throw std::runtime_error(kPrefix + "out must hold dense CUDA tensors on the gradients' device");
        if (o->sizes() != t->sizes()) value_error("out[" + std::to_string(i) + "] must have its gradient's shape");
        const at::ScalarType ot = c10::typeMetaToScalarType(o->dtype());
        if (ot != at::kFloat && ot != st)
          type_error("out must be float32 or the gradient's type, got " + name_of(ot));
        const bool alike = (plain && o->is_contiguous()) ||
                           (t->is_non_overlapping_and_dense() && t->strides() == o->strides());
        if (!alike) {
          if (!o->is_contiguous()) value_error("out[" + std::to_string(i) + "] must be contiguous");
          copied.push_back(i);
          g->keep.push_back(handle(t).contiguous());
          t = g->keep.back().unsafeGetTensorImpl();
        }
        g->out[i] = o->mutable_data();
        g->out_type[i] = code_of(ot);
        written = o;
      } else if (!plain && !t->is_non_overlapping_and_dense()) {
        copied.push_back(i);
        t = copy_strided(t, i, clip, &steps, g);
      }
      g->in[i] = clip && !outs ? t->mutable_data() : t->data();
      g->numel[i] = t->numel();
      g->in_type[i] = code;
      if (clip && !written->is_inference()) written->bump_version();
    }
  } catch (...) {
    if (clip) g->n_counted = i;
    throw;
  }
  if (clip) g->n_counted = n;
  if (forward_mode())
    for (Py_ssize_t k = 0; k < n; ++k) {
      refuse_tangent(THPVariable_Unpack(items[k]), "a gradient");
      if (outs) refuse_tangent(THPVariable_Unpack(out_items[k]), "an output");
    }
  if (clip && !copied.empty()) check_memory(items, out_items, n, copied, &steps);
  return device;
}

int norm_kind(double norm_type) {
  if (norm_type == 2.0) return GTK_NORM_2;
  if (norm_type == std::numeric_limits<double>::infinity()) return GTK_NORM_INF;
  value_error("norm_type must be 2.0 or inf, got " + std::to_string(norm_type));
}

Tensor grad_norm(const py::sequence& grads, double norm_type) {
  const int kind = norm_kind(norm_type);
  at::NoGradGuard no_grad;
  Gradients g;
  c10::cuda::OptionalCUDAGuard guard;
  const c10::Device device = collect(grads, nullptr, false, &g, &guard);
  Tensor norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(device));
  const size_t bytes = api.grad_norm_workspace_bytes(g.in.size());
  Tensor ws = scratch(bytes, norm);
  check(api.grad_norm(g.in.data(), g.numel.data(), g.in_type.data(), g.in.size(), kind,
                      static_cast<float*>(norm.data_ptr()), ws.data_ptr(), bytes, stream_of(device)),
        "gtk_grad_norm");
  return norm;
}

Tensor clip_grad_norm(const py::sequence& grads, double max_norm, double norm_type, const py::object& out) {
  const int kind = norm_kind(norm_type);
  if (!(max_norm >= 0.0)) value_error("max_norm must be a number >= 0, got " + std::to_string(max_norm));
  at::NoGradGuard no_grad;
  Gradients g;
  const bool in_place = out.is_none();
  c10::cuda::OptionalCUDAGuard guard;
  const c10::Device device = collect(grads, in_place ? nullptr : &out, true, &g, &guard);
  Tensor norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(device));
  const size_t bytes = api.grad_norm_workspace_bytes(g.in.size());
  Tensor ws = scratch(bytes, norm);
  const int rc = api.clip_grad_norm(g.in.data(), in_place ? nullptr : g.out.data(), g.numel.data(), g.in_type.data(),
                                    in_place ? nullptr : g.out_type.data(), g.in.size(), kind, max_norm,
                                    static_cast<float*>(norm.data_ptr()), ws.data_ptr(), bytes, stream_of(device));
  if (rc == GTK_OK || rc == GTK_ERR_CUDA) g.done();  // a launch that fails may follow one that writes
  check(rc, "gtk_clip_grad_norm");
  for (auto& p : g.write_back) p.first.copy_(p.second);
  return norm;
}

// ---- Embedding ----------------------------------------------------------------------------------

int index_bits(const Tensor& tokens) {
  if (tokens.scalar_type() == at::kLong) return 64;
  if (tokens.scalar_type() == at::kInt) return 32;
  type_error("tokens must be int32 or int64, got " + name_of(tokens.scalar_type()));
}

Tensor embedding_forward(const Tensor& tokens_in, const Tensor& weight_in, double scale, uintptr_t status) {
  require_cuda(weight_in, "weight");
  same_device(tokens_in, weight_in.device(), "tokens");
  const int bits = index_bits(tokens_in);
  const int dt = dtype_code(weight_in, "weight");
  if (weight_in.dim() != 2 || weight_in.size(0) < 1)
    value_error("weight must be [vocabulary, width], got " + shape_of(weight_in));
  refuse_tangents({{&weight_in, "weight"}});
  at::NoGradGuard no_grad;
  c10::cuda::CUDAGuard guard(weight_in.device());
  std::vector<int64_t> shape = tokens_in.sizes().vec();
  shape.push_back(weight_in.size(1));
  Tensor y = at::empty(shape, weight_in.options());
  if (y.numel()) {
    const Tensor tokens = contiguous(tokens_in), weight = contiguous(weight_in);
    check(api.embedding_forward(tokens.data_ptr(), bits, weight.data_ptr(), dt, y.data_ptr(), tokens.numel(),
                                weight.size(0), weight.size(1), static_cast<float>(scale),
                                reinterpret_cast<uint32_t*>(status), stream_of(weight.device())),
          "gtk_embedding_forward");
  }
  return y;
}

Tensor embedding_backward(const Tensor& dy_in, const Tensor& tokens_in, int64_t vocab, double scale,
                          std::optional<int64_t> padding, std::optional<at::ScalarType> dtype, uintptr_t status) {
  require_cuda(dy_in, "dy");
  same_device(tokens_in, dy_in.device(), "tokens");
  const int bits = index_bits(tokens_in);
  const int gt = dtype_code(dy_in, "dy");
  if (dy_in.dim() != tokens_in.dim() + 1 || dy_in.sizes().slice(0, tokens_in.dim()) != tokens_in.sizes())
    value_error("dy must be [*tokens.shape, width], got " + shape_of(dy_in) + " for tokens " + shape_of(tokens_in));
  if (vocab < 1) value_error("the vocabulary must have at least one token");
  const at::ScalarType wd = dtype.value_or(dy_in.scalar_type());
  if (wd != at::kFloat && wd != dy_in.scalar_type())
    type_error("the table's gradient must be float32 or dy's type, got " + name_of(wd));
  if (padding && (*padding < 0 || *padding >= vocab))
    value_error("padding_idx must be a token of the vocabulary, got " + std::to_string(*padding));
  refuse_tangents({{&dy_in, "dy"}});
  at::NoGradGuard no_grad;
  c10::cuda::CUDAGuard guard(dy_in.device());
  const int64_t D = dy_in.size(-1), n = tokens_in.numel();
  const auto options = dy_in.options().dtype(wd);
  if (n == 0 || D == 0) return at::zeros({vocab, D}, options);
  Tensor dw = at::empty({vocab, D}, options);
  const Tensor tokens = contiguous(tokens_in);
  Tensor dy = contiguous(dy_in);
  if (reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16) dy = dy.clone();  // a view that begins off a vector
  const size_t bytes = api.embedding_backward_workspace_bytes(n, vocab, D, gt);
  Tensor ws = scratch(bytes, dy);
  check(api.embedding_backward(dy.data_ptr(), gt, tokens.data_ptr(), bits, dw.data_ptr(), code_of(wd), n, vocab, D,
                               static_cast<float>(scale), padding.value_or(-1), ws.data_ptr(), bytes,
                               reinterpret_cast<uint32_t*>(status), stream_of(dy.device())),
        "gtk_embedding_backward");
  return dw;
}

}  // namespace

PYBIND11_MODULE(_gtk_torch, m) {
  m.doc() = "PyTorch binding of the training operators of libgenie_tk_b200.so";
  m.def("bind", &bind);
  m.def("layernorm_forward", &layernorm_forward);
  m.def("layernorm_backward", &layernorm_backward);
  m.def("grad_norm", &grad_norm);
  m.def("clip_grad_norm", &clip_grad_norm);
  m.def("embedding_forward", &embedding_forward);
  m.def("embedding_backward", &embedding_backward);
}
