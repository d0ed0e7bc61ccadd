// expert_calls.cpp - calls of the INT8 products, routing and the exchange of tokens from Python in compiled code.
//
// As for the FP4 operators (fp4_calls.cpp): these functions make the calls whose arguments need nothing special (plain CUDA
// tensors on the current device, rows that lie together, matching shapes and types) and return None for any others, which
// then take the Python path with its messages and copies. Both paths make the same library calls, through entry points
// bound by address. A call that is differentiated gets a node of compiled code too, since a node of Python costs more than
// the kernels: routing 777 tokens and its gradient took 153 us in a program with it, 21 of them on the device.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstring>
#include <memory>
#include <utility>
#include <vector>

#include "../../include/piper_int8.h"
#include "../../include/piper_routing.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entry {
  decltype(&piper_int8_linear_workspace) linear_workspace;
  decltype(&piper_int8_grad_input_workspace) grad_workspace;
  decltype(&piper_int8_linear) linear;
  decltype(&piper_int8_grad_input) grad_input;
  decltype(&piper_int8_last_error) int8_error;
  decltype(&piper_routing_workspace) route_workspace;
  decltype(&piper_routing_route) route;
  decltype(&piper_routing_route_grad) route_grad;
  decltype(&piper_routing_dispatch) dispatch;
  decltype(&piper_routing_combine) combine;
  decltype(&piper_routing_combine_grad) combine_grad;
  decltype(&piper_routing_last_error) routing_error;
} g_entry;
constexpr int kEntries = 12;

PyObject *g_qdata, *g_scale, *g_block, *g_zero, *g_pre, *g_cb, *g_scb, *g_data;

// A Python reference that is given back.
struct Ref {
  PyObject* o = nullptr;
  Ref() = default;
  Ref(const Ref&) = delete;
  ~Ref() { Py_XDECREF(o); }
};

struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

bool attribute(PyObject* from, PyObject* name, Ref& to) {
  if (_PyObject_LookupAttr(from, name, &to.o) < 0) PyErr_Clear();
  return to.o != nullptr;
}

// Without a forward-mode tangent, which the Python path refuses, and with memory of its own as it reads.
const Tensor* plain_tensor(PyObject* o) {
  if (o == nullptr || !THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided && t.has_storage() && !t.is_neg() && !t._fw_grad(/*level=*/0).defined() ? &t : nullptr;
}

// The same numbers in both headers.
static_assert(int{PIPER_INT8_BF16} == int{PIPER_ROUTING_BF16} && int{PIPER_INT8_F16} == int{PIPER_ROUTING_F16} &&
              int{PIPER_INT8_F32} == int{PIPER_ROUTING_F32});
int dtype_of(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? PIPER_INT8_BF16
         : t.scalar_type() == at::kHalf   ? PIPER_INT8_F16
         : t.scalar_type() == at::kFloat  ? PIPER_INT8_F32
                                          : -1;
}

// Rows of `cols` values one after another at a stride that does not overlap.
bool rows_of(const Tensor& x, int64_t cols, int64_t& rows, int64_t& stride) {
  const int64_t dims = x.dim();
  if (dims < 1 || x.size(dims - 1) != cols || x.numel() == 0) return false;
  rows = x.numel() / cols;
  stride = cols;
  if (x.is_contiguous()) return true;
  if (dims != 2 || x.stride(1) != 1 || (x.stride(0) < cols && rows > 1)) return false;
  stride = x.stride(0);
  return true;
}

// The same, by a copy where it is needed: gradients come in any layout.
Tensor with_rows(const Tensor& x, int64_t cols, int64_t& rows, int64_t& stride) {
  const Tensor plain = x.resolve_neg();
  if (rows_of(plain, cols, rows, stride)) return plain;
  const Tensor copy = plain.contiguous();
  rows = copy.numel() / cols;
  stride = cols;
  return copy;
}

void* stream_of(c10::DeviceIndex device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

std::vector<int64_t> shape_with_last(const Tensor& x, int64_t last) {
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = last;
  return shape;
}

// A tensor that a node does not look at: one that gets no gradient, or none.
struct Aside {
  Tensor tensor;
};

// A backward pass has no derivative of its own: one that is asked for raises when it is reached.
variable_list once_differentiable(const variable_list& grads, variable_list&& outputs) {
  bool wanted = at::GradMode::is_enabled();
  if (wanted) {
    wanted = false;
    for (const Tensor& g : grads) wanted = wanted || (g.defined() && g.requires_grad());
  }
  if (!wanted) return std::move(outputs);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", static_cast<int64_t>(outputs.size()));
  variable_list leaves;
  for (const Tensor& t : outputs) leaves.push_back(t.defined() ? t.detach().requires_grad_() : t);
  return (*error)(std::move(leaves));
}

void check_int8(int rc) {
  TORCH_CHECK_VALUE(rc != PIPER_INT8_EINVAL, g_entry.int8_error());
  TORCH_CHECK(rc == PIPER_INT8_OK, "piper int8 failed (status ", rc, "): ", g_entry.int8_error());
}

void check_routing(int rc) {
  TORCH_CHECK_VALUE(rc != PIPER_ROUTING_EINVAL, g_entry.routing_error());
  TORCH_CHECK(rc == PIPER_ROUTING_OK, "piper routing failed (status ", rc, "): ", g_entry.routing_error());
}

// ----------------------------------------------------------------------------------- products
// A weight's tensors as they are now: what one product and its backward pass work with.
struct Weight {
  Tensor codes, scale, zero;
  piper_int8_matrix m{};
  std::vector<std::pair<Tensor, int64_t>> versions;

  // dims 2: a weight, 3: a stack of experts.
  bool read(PyObject* w, int dims) {
    Ref q, s, z, block, pre;
    m.per_row = 1;
    if (attribute(w, g_cb, q)) {
      if (!attribute(w, g_scb, s) || dims != 2) return false;
      m.over_127 = 1;
    } else {
      Ref other;
      if (!attribute(w, g_qdata, q) || !attribute(w, g_scale, s) || !attribute(w, g_block, block) || attribute(w, g_data, other)) return false;
      if (attribute(w, g_pre, pre) && pre.o != Py_None) return false;
      attribute(w, g_zero, z);
      if (!PyTuple_CheckExact(block.o) || PyTuple_GET_SIZE(block.o) != 2) return false;
    }
    const Tensor *qt = plain_tensor(q.o), *st = plain_tensor(s.o);
    const bool has_zero = z.o != nullptr && z.o != Py_None;
    const Tensor* zt = has_zero ? plain_tensor(z.o) : nullptr;
    if (qt == nullptr || st == nullptr || qt->scalar_type() != at::kChar || qt->dim() != dims || !qt->is_contiguous() || qt->numel() == 0 ||
        (has_zero && zt == nullptr))
      return false;
    m.batch = dims == 3 ? qt->size(0) : 1;
    m.rows = qt->size(dims - 2);
    m.cols = qt->size(dims - 1);
    if (block.o != nullptr) {
      const long first = PyLong_AsLong(PyTuple_GET_ITEM(block.o, 0)), last = PyLong_AsLong(PyTuple_GET_ITEM(block.o, 1));
      if (PyErr_Occurred()) PyErr_Clear();
      m.per_row = first == 1;
      if (last != m.cols || (m.per_row == 0 && (first != m.rows || dims == 3))) return false;
    }
    const int64_t values = m.per_row != 0 ? m.batch * m.rows : 1;
    m.scale_dtype = dtype_of(*st);
    if (m.scale_dtype < 0 || st->numel() != values || !st->is_contiguous() || st->get_device() != qt->get_device()) return false;
    if (has_zero && (zt->scalar_type() != at::kChar || zt->numel() != values || !zt->is_contiguous() || zt->get_device() != qt->get_device()))
      return false;
    codes = *qt;
    scale = *st;
    if (has_zero) zero = *zt;
    m.codes = codes.const_data_ptr();
    m.scale = scale.const_data_ptr();
    m.zero = has_zero ? zero.const_data_ptr() : nullptr;
    return codes.get_device() == c10::cuda::current_device();
  }

  void mark() {
    for (const Tensor* t : {&codes, &scale, &zero})
      if (t->defined() && !t->is_inference()) versions.emplace_back(*t, t->_version());
  }

  void check() const {
    for (const auto& [t, version] : versions)
      TORCH_CHECK(t._version() == version, "a tensor of an INT8 weight has been modified by an inplace operation since its product, "
                                           "whose gradient needs it as it was.");
  }
};

Tensor product(const Weight& w, const Tensor& x, int64_t stride, int64_t tokens, const Tensor& ends, bool grad) {
  const int dtype = dtype_of(x);
  size_t need = 0;
  check_int8(grad ? g_entry.grad_workspace(&w.m, tokens, dtype, &need) : g_entry.linear_workspace(&w.m, tokens, ends.defined(), &need));
  Tensor y = at::empty(shape_with_last(x, grad ? w.m.cols : w.m.rows), x.options().requires_grad(false));
  Tensor workspace;
  if (need > 0) workspace = at::empty({static_cast<int64_t>(need)}, x.options().dtype(at::kByte).requires_grad(false));
  const auto call = grad ? g_entry.grad_input : g_entry.linear;
  check_int8(call(&w.m, x.const_data_ptr(), stride, tokens, ends.defined() ? ends.const_data_ptr<int32_t>() : nullptr, y.mutable_data_ptr(),
                  dtype, need > 0 ? workspace.mutable_data_ptr() : nullptr, need, stream_of(static_cast<c10::DeviceIndex>(x.get_device()))));
  return y;
}

struct Int8Product : torch::autograd::Function<Int8Product> {
  struct Held : torch::CustomClassHolder {
    explicit Held(std::shared_ptr<Weight> w) : weight(std::move(w)) {}
    std::shared_ptr<Weight> weight;
  };

  static Tensor forward(AutogradContext* ctx, const Tensor& x, std::shared_ptr<Weight> w, int64_t stride, int64_t tokens, const Aside& ends) {
    at::AutoDispatchBelowADInplaceOrView below;
    w->mark();
    ctx->saved_data["weight"] = c10::IValue::make_capsule(c10::make_intrusive<Held>(w));
    ctx->save_for_backward({ends.tensor});
    return product(*w, x, stride, tokens, ends.tensor, false);
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const auto held = c10::static_intrusive_pointer_cast<Held>(ctx->saved_data["weight"].toCapsule());
    const Weight& w = *held->weight;
    w.check();
    variable_list out(5);
    Tensor dx;
    {
      const at::NoGradGuard no_grad;
      const c10::cuda::CUDAGuard device(grads[0].device());
      int64_t tokens, stride;
      const Tensor g = with_rows(grads[0], w.m.rows, tokens, stride);
      dx = product(w, g, stride, tokens, saved[0], true);
    }
    out[0] = once_differentiable(grads, {std::move(dx)})[0];
    return out;
  }
};

bool ends_of(PyObject* o, const Weight& w, Tensor& ends) {
  if (o == Py_None) return true;
  const Tensor* t = plain_tensor(o);
  if (t == nullptr || t->scalar_type() != at::kInt || t->dim() != 1 || t->numel() != w.m.batch || !t->is_contiguous() ||
      t->get_device() != w.codes.get_device())
    return false;
  ends = *t;
  return true;
}

// int8(x, weight, ends or None, gradient) -> y or dx
PyObject* int8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) Py_RETURN_NONE;
  const Tensor* x = plain_tensor(args[0]);
  const bool grad = args[3] == Py_True;
  const auto w = std::make_shared<Weight>();
  Tensor ends;
  int64_t tokens, stride;
  if (x == nullptr || dtype_of(*x) < 0 || !w->read(args[1], args[2] == Py_None ? 2 : 3) || x->get_device() != w->codes.get_device() ||
      !rows_of(*x, grad ? w->m.rows : w->m.cols, tokens, stride) || !ends_of(args[2], *w, ends) || (ends.defined() && x->dim() != 2))
    Py_RETURN_NONE;
  Tensor y;
  {
    NoGil nogil;
    if (!grad && x->requires_grad() && at::GradMode::is_enabled()) y = Int8Product::apply(*x, w, stride, tokens, Aside{ends});
    else y = product(*w, *x, stride, tokens, ends, grad);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------ routing
// at::empty on the current device, without what the dispatcher costs (64 x 8 routed 6.5 us of host time, 8.4 with it).
Tensor results(at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_generic(sizes, c10::cuda::CUDACachingAllocator::get(), c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}

variable_list route_of(const piper_routing_config& c, const Tensor& logits, int64_t stride, const Tensor& bias, const Tensor& mask) {
  // each with memory of its own: parts of one allocation (5.5 us) cannot be saved together, and each keeps and saves all of it
  Tensor weights = results({c.tokens, c.top_k}, at::kFloat), experts = results({c.tokens, c.top_k}, at::kInt);
  Tensor rows = results({c.tokens, c.top_k}, at::kInt), source = results({c.tokens * c.top_k}, at::kInt), ends = results({c.experts}, at::kInt);
  size_t need = 0;
  check_routing(g_entry.route_workspace(&c, &need));
  Tensor workspace;
  if (need > 0) workspace = at::empty({static_cast<int64_t>(need)}, logits.options().requires_grad(false).dtype(at::kByte));
  check_routing(g_entry.route(&c, logits.const_data_ptr(), stride, dtype_of(logits), bias.defined() ? bias.const_data_ptr<float>() : nullptr,
                              mask.defined() ? static_cast<const uint8_t*>(mask.const_data_ptr()) : nullptr, weights.mutable_data_ptr<float>(),
                              experts.mutable_data_ptr<int32_t>(), ends.mutable_data_ptr<int32_t>(), rows.mutable_data_ptr<int32_t>(),
                              source.mutable_data_ptr<int32_t>(), need > 0 ? workspace.mutable_data_ptr() : nullptr, need,
                              stream_of(static_cast<c10::DeviceIndex>(logits.get_device()))));
  return {weights, experts, ends, rows, source};
}

// The rules of a routing, kept for its backward pass as numbers.
std::vector<int64_t> numbers_of(const piper_routing_config& c) {
  return {c.tokens, c.experts, c.top_k, c.scoring, c.groups, c.top_groups, c.group_score, c.renormalize};
}

piper_routing_config config_of(const std::vector<int64_t>& v, double scale) {
  const auto i = [&](int at) { return static_cast<int32_t>(v[at]); };
  return {v[0], i(1), i(2), i(3), i(4), i(5), i(6), i(7), static_cast<float>(scale)};
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const piper_routing_config& c, int64_t stride, const Aside& bias,
                               const Aside& mask) {
    at::AutoDispatchBelowADInplaceOrView below;
    variable_list out = route_of(c, logits, stride, bias.tensor, mask.tensor);
    ctx->saved_data["config"] = numbers_of(c);
    ctx->saved_data["scale"] = static_cast<double>(c.scale);
    ctx->save_for_backward({logits, out[1]});
    ctx->mark_non_differentiable({out[1], out[2], out[3], out[4]});
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(5);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const piper_routing_config c = config_of(ctx->saved_data["config"].toIntVector(), ctx->saved_data["scale"].toDouble());
    Tensor dlogits;
    {
      const at::NoGradGuard no_grad;
      const c10::cuda::CUDAGuard device(grads[0].device());
      int64_t tokens, stride;
      const Tensor logits = with_rows(saved[0], c.experts, tokens, stride);
      const Tensor g = grads[0].resolve_neg().contiguous();
      dlogits = at::empty({c.tokens, c.experts}, logits.options().requires_grad(false));
      check_routing(g_entry.route_grad(&c, logits.const_data_ptr(), stride, dtype_of(logits), saved[1].const_data_ptr<int32_t>(),
                                       g.const_data_ptr<float>(), dlogits.mutable_data_ptr(),
                                       stream_of(static_cast<c10::DeviceIndex>(logits.get_device()))));
    }
    out[0] = once_differentiable({grads[0]}, {std::move(dlogits)})[0];
    return out;
  }
};

PyObject* tuple_of(variable_list&& tensors) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
  if (out == nullptr) return nullptr;
  for (size_t i = 0; i < tensors.size(); ++i) PyTuple_SET_ITEM(out, static_cast<Py_ssize_t>(i), THPVariable_Wrap(std::move(tensors[i])));
  return out;
}

// route(logits, top_k, scoring, bias or None, groups, top_groups, group_score, renormalize, scale, mask or None)
//   -> (weights, experts, ends, rows, source)
PyObject* route(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10) Py_RETURN_NONE;
  const Tensor* logits = plain_tensor(args[0]);
  if (logits == nullptr || logits->dim() != 2 || dtype_of(*logits) < 0 || logits->get_device() != c10::cuda::current_device()) Py_RETURN_NONE;
  piper_routing_config c{};
  int64_t tokens, stride;
  if (!rows_of(*logits, logits->size(1), tokens, stride) || logits->size(1) > PIPER_ROUTING_MAX_EXPERTS) Py_RETURN_NONE;
  for (const int i : {1, 2, 4, 5, 6})
    if (!PyLong_CheckExact(args[i])) Py_RETURN_NONE;
  c.tokens = tokens;
  c.experts = static_cast<int32_t>(logits->size(1));
  const auto number = [&](int i) { return static_cast<int32_t>(std::min<long>(std::max<long>(PyLong_AsLong(args[i]), -1), 1 << 20)); };
  c.top_k = number(1);
  c.scoring = number(2);
  c.groups = number(4);
  c.top_groups = number(5);
  c.group_score = number(6);
  c.renormalize = PyObject_IsTrue(args[7]) == 1;
  const double scale = PyFloat_AsDouble(args[8]);
  if (PyErr_Occurred() || c.top_k < 1 || c.top_k > PIPER_ROUTING_MAX_TOP_K || c.groups < 1 || c.groups > PIPER_ROUTING_MAX_GROUPS) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  c.scale = static_cast<float>(scale);
  Tensor bias, mask;
  if (args[3] != Py_None) {
    const Tensor* t = plain_tensor(args[3]);
    if (t == nullptr || t->scalar_type() != at::kFloat || t->dim() != 1 || t->numel() != c.experts || !t->is_contiguous() ||
        t->get_device() != logits->get_device())
      Py_RETURN_NONE;
    bias = t->detach();
  }
  if (args[9] != Py_None) {
    const Tensor* t = plain_tensor(args[9]);
    if (t == nullptr || t->scalar_type() != at::kBool || t->dim() != 1 || t->numel() != tokens || !t->is_contiguous() ||
        t->get_device() != logits->get_device())
      Py_RETURN_NONE;
    mask = *t;
  }
  variable_list out;
  {
    NoGil nogil;
    if (logits->requires_grad() && at::GradMode::is_enabled()) out = Route::apply(*logits, c, stride, Aside{bias}, Aside{mask});
    else out = route_of(c, *logits, stride, bias, mask);
  }
  return tuple_of(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ----------------------------------------------------------------------------------- exchange
piper_routing_exchange exchange_of(const Tensor& rows, const Tensor& ends, const Tensor& t) {
  return {rows.size(0), static_cast<int32_t>(rows.size(1)), static_cast<int32_t>(t.size(1)), dtype_of(t), rows.const_data_ptr<int32_t>(),
          ends.const_data_ptr<int32_t>() + (ends.size(0) - 1)};
}

Tensor sent(const Tensor& x, int64_t stride, const Tensor& rows, const Tensor& ends) {
  Tensor out = at::empty({rows.numel(), x.size(1)}, x.options().requires_grad(false));
  const piper_routing_exchange e = exchange_of(rows, ends, x);
  check_routing(g_entry.dispatch(&e, x.const_data_ptr(), stride, out.mutable_data_ptr(), stream_of(static_cast<c10::DeviceIndex>(x.get_device()))));
  return out;
}

Tensor combined(const Tensor& y, int64_t stride, const Tensor& weights, const Tensor& rows, const Tensor& ends) {
  Tensor out = at::empty({rows.size(0), y.size(1)}, y.options().requires_grad(false));
  const piper_routing_exchange e = exchange_of(rows, ends, y);
  check_routing(g_entry.combine(&e, y.const_data_ptr(), stride, weights.defined() ? weights.const_data_ptr<float>() : nullptr,
                                out.mutable_data_ptr(), stream_of(static_cast<c10::DeviceIndex>(y.get_device()))));
  return out;
}

struct Dispatch : torch::autograd::Function<Dispatch> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, int64_t stride, const Tensor& rows, const Tensor& ends) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({rows, ends});
    return sent(x, stride, rows, ends);
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    variable_list out(4);
    Tensor dx;
    {
      const at::NoGradGuard no_grad;
      const c10::cuda::CUDAGuard device(grads[0].device());
      int64_t rows, stride;
      const Tensor g = with_rows(grads[0], grads[0].size(1), rows, stride);
      dx = combined(g, stride, Tensor(), saved[0], saved[1]);
    }
    out[0] = once_differentiable(grads, {std::move(dx)})[0];
    return out;
  }
};

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, int64_t stride, const Tensor& weights, const Tensor& rows, const Tensor& ends) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({y, weights, rows, ends});
    return combined(y, stride, weights, rows, ends);
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    variable_list out(5);
    Tensor dy, dweights;
    {
      const at::NoGradGuard no_grad;
      const c10::cuda::CUDAGuard device(grads[0].device());
      int64_t n, y_stride, g_stride;
      const Tensor y = with_rows(saved[0], saved[0].size(1), n, y_stride), g = with_rows(grads[0], grads[0].size(1), n, g_stride);
      dy = at::empty(y.sizes(), y.options().requires_grad(false));
      dweights = at::empty(saved[1].sizes(), saved[1].options().requires_grad(false));
      const piper_routing_exchange e = exchange_of(saved[2], saved[3], y);
      check_routing(g_entry.combine_grad(&e, y.const_data_ptr(), y_stride, saved[1].const_data_ptr<float>(), g.const_data_ptr(), g_stride,
                                         dy.mutable_data_ptr(), dweights.mutable_data_ptr<float>(),
                                         stream_of(static_cast<c10::DeviceIndex>(y.get_device()))));
    }
    variable_list both = once_differentiable(grads, {std::move(dy), std::move(dweights)});
    out[0] = both[0];
    out[2] = both[1];
    return out;
  }
};

// A routing's rows and ends, and rows of values on their device: one for a token (`per_token`) or for each place.
bool exchange_args(const Tensor* t, const Tensor* rows, const Tensor* ends, bool per_token, int64_t& stride) {
  if (t == nullptr || rows == nullptr || ends == nullptr || t->dim() != 2 || dtype_of(*t) < 0 || rows->scalar_type() != at::kInt ||
      ends->scalar_type() != at::kInt || rows->dim() != 2 || ends->dim() != 1 || !rows->is_contiguous() || !ends->is_contiguous() ||
      ends->numel() == 0 || rows->numel() == 0 || t->size(1) > (1 << 24) || rows->size(1) > PIPER_ROUTING_MAX_TOP_K)
    return false;
  const auto device = t->get_device();
  int64_t n;
  return rows->get_device() == device && ends->get_device() == device && device == c10::cuda::current_device() &&
         t->size(0) == (per_token ? rows->size(0) : rows->numel()) && rows_of(*t, t->size(1), n, stride);
}

// dispatch(x, rows, ends) -> rows sorted by expert
PyObject* dispatch(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) Py_RETURN_NONE;
  const Tensor *x = plain_tensor(args[0]), *rows = plain_tensor(args[1]), *ends = plain_tensor(args[2]);
  int64_t stride;
  if (!exchange_args(x, rows, ends, true, stride)) Py_RETURN_NONE;
  Tensor out;
  {
    NoGil nogil;
    out = x->requires_grad() && at::GradMode::is_enabled() ? Dispatch::apply(*x, stride, *rows, *ends) : sent(*x, stride, *rows, *ends);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// combine(y, weights, rows, ends) -> tokens
PyObject* combine(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) Py_RETURN_NONE;
  const Tensor *y = plain_tensor(args[0]), *w = plain_tensor(args[1]), *rows = plain_tensor(args[2]), *ends = plain_tensor(args[3]);
  int64_t stride;
  if (!exchange_args(y, rows, ends, false, stride) || w == nullptr || w->scalar_type() != at::kFloat || !w->is_contiguous() ||
      w->sizes() != rows->sizes() || w->get_device() != y->get_device())
    Py_RETURN_NONE;
  Tensor out;
  {
    NoGil nogil;
    out = (y->requires_grad() || w->requires_grad()) && at::GradMode::is_enabled() ? Combine::apply(*y, stride, *w, *rows, *ends)
                                                                                   : combined(*y, stride, *w, *rows, *ends);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// bind(twelve addresses): the libraries' entry points, in Entry's order
PyObject* bind(PyObject*, PyObject* args) {
  if (PyTuple_GET_SIZE(args) != kEntries) {
    PyErr_SetString(PyExc_ValueError, "bind takes the entry points in their order");
    return nullptr;
  }
  void* at[kEntries];
  for (int i = 0; i < kEntries; ++i) at[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(args, i));
  if (PyErr_Occurred()) return nullptr;
  static_assert(sizeof(Entry) == sizeof(at));
  std::memcpy(&g_entry, at, sizeof(at));
  Py_RETURN_NONE;
}

#define FAST(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {{"bind", bind, METH_VARARGS, nullptr}, FAST(int8), FAST(route), FAST(dispatch), FAST(combine),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_expert_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__expert_calls() {
  const struct {
    PyObject** to;
    const char* name;
  } names[] = {{&g_qdata, "qdata"}, {&g_scale, "scale"}, {&g_block, "block_size"}, {&g_zero, "zero_point"}, {&g_pre, "act_pre_scale"},
               {&g_cb, "CB"}, {&g_scb, "SCB"}, {&g_data, "_data"}};
  for (const auto& n : names)
    if ((*n.to = PyUnicode_InternFromString(n.name)) == nullptr) return nullptr;
  return PyModule_Create(&g_module);
}
