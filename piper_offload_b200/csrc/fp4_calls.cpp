// fp4_calls.cpp - the FP4 operators' calls from Python without the cost of checking and passing everything there.
//
// A call whose kernels take 5 to 10 us spends 14 to 20 us in Python: attribute
// reads, allocations and argument conversions. These functions do the same for
// arguments that need nothing special (plain CUDA tensors on the current
// device, rows that lie together, matching shapes and types) and return None
// for any others, which then take the Python path with its messages and
// copies. Both paths make the same library calls; the entry points are bound
// by address, so that they are those of the one loaded library.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/piper_fp4.h"

namespace {

struct Entry {
  decltype(&piper_fp4_quantize) quantize;
  decltype(&piper_fp4_dequantize) dequantize;
  decltype(&piper_fp4_linear_workspace) linear_workspace;
  decltype(&piper_fp4_grad_input_workspace) grad_workspace;
  decltype(&piper_fp4_linear) linear;
  decltype(&piper_fp4_grad_input) grad_input;
} g_entry;

PyObject *g_qdata, *g_scale, *g_second, *g_swizzled, *g_elem, *g_block, *g_kwargs, *g_mode, *g_value, *g_dtype;
PyObject* g_fp4_type;  // torch.float4_e2m1fn_x2

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

// Without a forward-mode tangent, which the Python path refuses.
const at::Tensor* plain_tensor(PyObject* o) {
  if (o == nullptr || !THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided && !t._fw_grad(/*level=*/0).defined() ? &t : nullptr;
}

int dtype_of(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? PIPER_FP4_BF16 : t.scalar_type() == at::kFloat ? PIPER_FP4_F32 : -1;
}

// FLOOR without a mode, -1 for one that is not known.
int scaling_mode(PyObject* weight) {
  Ref kwargs, mode, value;
  if (!attribute(weight, g_kwargs, kwargs) || !attribute(kwargs.o, g_mode, mode) || mode.o == Py_None) return PIPER_FP4_FLOOR;
  PyObject* name = attribute(mode.o, g_value, value) ? value.o : mode.o;
  if (!PyUnicode_Check(name)) return -1;
  const char* names[] = {"floor", "rceil", "ceil", "even"};
  for (int i = 0; i < 4; ++i)
    if (PyUnicode_CompareWithASCIIString(name, names[i]) == 0) return i;
  return -1;
}

// A packed weight (dims 2) or stack of experts (dims 3); the references keep its tensors for the call.
struct Weight {
  Ref codes, scale, second;
  piper_fp4_matrix m{};
  int mode = 0;
  c10::DeviceIndex device = -1;

  bool read(PyObject* w, int dims) {
    Ref swizzled, elem, block;
    if (!attribute(w, g_qdata, codes) || !attribute(w, g_scale, scale) || !attribute(w, g_swizzled, swizzled) ||
        !attribute(w, g_block, block))
      return false;
    const at::Tensor *q = plain_tensor(codes.o), *s = plain_tensor(scale.o);
    if (q == nullptr || s == nullptr || q->scalar_type() != at::kByte || q->dim() != dims || s->dim() != dims ||
        !q->is_contiguous() || !s->is_contiguous() || q->get_device() != s->get_device() || q->numel() == 0 ||
        (swizzled.o != Py_True && swizzled.o != Py_False))
      return false;
    m.batch = dims == 3 ? q->size(0) : 1;
    m.rows = q->size(dims - 2);
    m.cols = q->size(dims - 1) * 2;
    m.swizzled = swizzled.o == Py_True;
    int values;
    if (attribute(w, g_elem, elem)) {
      if (elem.o != g_fp4_type || (s->scalar_type() != at::kByte && s->scalar_type() != at::kFloat8_e8m0fnu)) return false;
      mode = scaling_mode(w);
      if (mode < 0) return false;
      m.format = PIPER_FP4_MX;
      values = 32;
    } else {
      if (s->scalar_type() != at::kFloat8_e4m3fn || !attribute(w, g_second, second)) return false;
      if (second.o != Py_None) {
        const at::Tensor* g = plain_tensor(second.o);
        if (g == nullptr || g->scalar_type() != at::kFloat || g->numel() != m.batch || g->get_device() != q->get_device() ||
            !g->is_contiguous())
          return false;
        m.second = static_cast<float*>(g->data_ptr());
      }
      m.format = PIPER_FP4_NV;
      values = 16;
    }
    const long size = PyLong_AsLong(block.o);
    if (size == -1 && PyErr_Occurred()) PyErr_Clear();
    if (size != values || m.cols % values != 0) return false;
    const int64_t blocks = m.cols / values;
    const int64_t rows = m.swizzled ? (m.rows + 127) / 128 * 32 : m.rows, cols = m.swizzled ? (blocks + 3) / 4 * 16 : blocks;
    if (s->size(dims - 2) != rows || s->size(dims - 1) != cols || (dims == 3 && s->size(0) != m.batch)) return false;
    m.codes = q->data_ptr();
    m.scale = s->data_ptr();
    device = static_cast<c10::DeviceIndex>(q->get_device());
    return device == c10::cuda::current_device();
  }
};

// Rows of `cols` values one after another at a stride that does not overlap.
bool rows_of(const at::Tensor& x, int64_t cols, int64_t& tokens, int64_t& stride) {
  const int64_t dims = x.dim();
  if (dims < 1 || x.size(dims - 1) != cols || x.numel() == 0) return false;
  tokens = x.numel() / cols;
  stride = cols;
  if (x.is_contiguous()) return true;
  if (dims != 2 || x.stride(1) != 1 || (x.stride(0) < cols && tokens > 1)) return false;
  stride = x.stride(0);
  return true;
}

void* stream_of(c10::DeviceIndex device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

bool ends_of(PyObject* o, const Weight& w, const int32_t*& ends) {
  ends = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = plain_tensor(o);
  if (t == nullptr || t->scalar_type() != at::kInt || t->dim() != 1 || t->numel() != w.m.batch || !t->is_contiguous() ||
      t->get_device() != w.device)
    return false;
  ends = static_cast<const int32_t*>(t->data_ptr());
  return true;
}

std::vector<int64_t> shape_with_last(const at::Tensor& x, int64_t last) {
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = last;
  return shape;
}

#define FP4_DECLINE Py_RETURN_NONE

// linear(x, weight, ends or None, act scale or None) -> y
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) FP4_DECLINE;
  const at::Tensor* x = plain_tensor(args[0]);
  Weight w;
  if (x == nullptr || !w.read(args[1], args[2] == Py_None ? 2 : 3) || x->get_device() != w.device) FP4_DECLINE;
  const int dtype = dtype_of(*x);
  int64_t tokens, stride;
  const int32_t* ends;
  if (dtype < 0 || !rows_of(*x, w.m.cols, tokens, stride) || !ends_of(args[2], w, ends) || (ends != nullptr && x->dim() != 2)) FP4_DECLINE;
  const float* act = nullptr;
  if (args[3] != Py_None) {
    const at::Tensor* t = plain_tensor(args[3]);
    if (t == nullptr || t->scalar_type() != at::kFloat || t->numel() != 1 || t->get_device() != w.device || w.m.format != PIPER_FP4_NV) FP4_DECLINE;
    act = static_cast<const float*>(t->data_ptr());
  }
  at::Tensor y;
  int rc;
  {
    NoGil nogil;
    size_t need = 0;
    rc = g_entry.linear_workspace(&w.m, tokens, &need);
    if (rc == PIPER_FP4_OK) {
      y = at::empty(shape_with_last(*x, w.m.rows), x->options());
      at::Tensor workspace;
      if (need > 0) workspace = at::empty({static_cast<int64_t>(need)}, x->options().dtype(at::kByte));
      rc = g_entry.linear(&w.m, x->data_ptr(), stride, tokens, ends, act, w.mode, y.data_ptr(), dtype,
                          need > 0 ? workspace.data_ptr() : nullptr, need, stream_of(w.device));
    }
  }
  if (rc != PIPER_FP4_OK) FP4_DECLINE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// grad_input(grad, weight, ends or None) -> dx
PyObject* grad_input(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) FP4_DECLINE;
  const at::Tensor* g = plain_tensor(args[0]);
  Weight w;
  if (g == nullptr || !w.read(args[1], args[2] == Py_None ? 2 : 3) || g->get_device() != w.device) FP4_DECLINE;
  const int dtype = dtype_of(*g);
  int64_t tokens, stride;
  const int32_t* ends;
  if (dtype < 0 || !rows_of(*g, w.m.rows, tokens, stride) || !ends_of(args[2], w, ends) || (ends != nullptr && g->dim() != 2)) FP4_DECLINE;
  at::Tensor dx;
  int rc;
  {
    NoGil nogil;
    size_t need = 0;
    rc = g_entry.grad_workspace(&w.m, g->data_ptr(), stride, tokens, dtype, &need);
    if (rc == PIPER_FP4_OK) {
      dx = at::empty(shape_with_last(*g, w.m.cols), g->options());
      at::Tensor workspace;
      if (need > 0) workspace = at::empty({static_cast<int64_t>(need)}, g->options().dtype(at::kByte));
      rc = g_entry.grad_input(&w.m, g->data_ptr(), stride, tokens, ends, dx.data_ptr(), dtype,
                              need > 0 ? workspace.data_ptr() : nullptr, need, stream_of(w.device));
    }
  }
  if (rc != PIPER_FP4_OK) FP4_DECLINE;
  return THPVariable_Wrap(std::move(dx));
  END_HANDLE_TH_ERRORS
}

// dequantize(weight, dims, dtype or None) -> values
PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) FP4_DECLINE;
  Weight w;
  Ref own;
  PyObject* type = args[2];
  if (type == Py_None) type = attribute(args[0], g_dtype, own) ? own.o : nullptr;
  if (type == nullptr || !THPDtype_Check(type) || !w.read(args[0], static_cast<int>(PyLong_AsLong(args[1])))) FP4_DECLINE;
  const at::ScalarType scalar = reinterpret_cast<THPDtype*>(type)->scalar_type;
  if (scalar != at::kBFloat16 && scalar != at::kFloat) FP4_DECLINE;
  const at::Tensor& q = THPVariable_Unpack(w.codes.o);
  at::Tensor y;
  int rc;
  {
    NoGil nogil;
    y = at::empty(shape_with_last(q, w.m.cols), q.options().dtype(scalar));
    rc = g_entry.dequantize(&w.m, y.data_ptr(), dtype_of(y), stream_of(w.device));
  }
  if (rc != PIPER_FP4_OK) FP4_DECLINE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// quantize(x, format, scale mode, swizzled, second mode) -> (codes, scale, second or None); no given second level
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) FP4_DECLINE;
  const at::Tensor* x = plain_tensor(args[0]);
  if (x == nullptr || (x->dim() != 2 && x->dim() != 3) || x->get_device() != c10::cuda::current_device()) FP4_DECLINE;
  const int dtype = dtype_of(*x);
  piper_fp4_matrix m{};
  m.format = static_cast<int32_t>(PyLong_AsLong(args[1]));
  const int mode = static_cast<int>(PyLong_AsLong(args[2])), second_mode = static_cast<int>(PyLong_AsLong(args[4]));
  m.swizzled = PyObject_IsTrue(args[3]) == 1;
  const int values = m.format == PIPER_FP4_MX ? 32 : 16;
  m.batch = x->dim() == 3 ? x->size(0) : 1;
  m.rows = x->size(x->dim() - 2);
  m.cols = x->size(x->dim() - 1);
  int64_t rows, stride;
  if (dtype < 0 || m.cols % values != 0 || !rows_of(*x, m.cols, rows, stride) || second_mode == PIPER_FP4_SECOND_GIVEN) FP4_DECLINE;
  const int64_t blocks = m.cols / values;
  at::Tensor codes, scale, second, maxima;
  int rc;
  {
    NoGil nogil;
    const at::TensorOptions bytes = x->options().dtype(at::kByte);
    const at::TensorOptions scales = x->options().dtype(m.format == PIPER_FP4_MX ? at::kByte : at::kFloat8_e4m3fn);
    const int64_t srows = m.swizzled ? (m.rows + 127) / 128 * 32 : m.rows, scols = m.swizzled ? (blocks + 3) / 4 * 16 : blocks;
    if (x->dim() == 3) {
      codes = at::empty({m.batch, m.rows, m.cols / 2}, bytes);
      scale = at::empty({m.batch, srows, scols}, scales);
    } else {
      codes = at::empty({m.rows, m.cols / 2}, bytes);
      scale = at::empty({srows, scols}, scales);
    }
    m.codes = codes.data_ptr();
    m.scale = scale.data_ptr();
    if (second_mode == PIPER_FP4_SECOND_COMPUTE) {
      second = at::empty({m.batch}, x->options().dtype(at::kFloat));
      m.second = static_cast<float*>(second.data_ptr());
      if (m.rows * m.cols > PIPER_FP4_SMALL_MATRIX) maxima = at::empty({m.batch}, x->options().dtype(at::kInt));
    }
    rc = g_entry.quantize(&m, x->data_ptr(), stride, dtype, mode, second_mode,
                          maxima.defined() ? static_cast<uint32_t*>(maxima.data_ptr()) : nullptr,
                          stream_of(static_cast<c10::DeviceIndex>(x->get_device())));
  }
  if (rc != PIPER_FP4_OK) FP4_DECLINE;
  PyObject* out = PyTuple_New(3);
  if (out == nullptr) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(codes)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(scale)));
  PyTuple_SET_ITEM(out, 2, second.defined() ? THPVariable_Wrap(std::move(second)) : Py_NewRef(Py_None));
  return out;
  END_HANDLE_TH_ERRORS
}

// bind(torch.float4_e2m1fn_x2, six addresses): the library's entry points, in Entry's order
PyObject* bind(PyObject*, PyObject* args) {
  PyObject* type;
  unsigned long long at[6];
  if (!PyArg_ParseTuple(args, "OKKKKKK", &type, &at[0], &at[1], &at[2], &at[3], &at[4], &at[5])) return nullptr;
  Py_XSETREF(g_fp4_type, Py_NewRef(type));
  g_entry.quantize = reinterpret_cast<decltype(g_entry.quantize)>(at[0]);
  g_entry.dequantize = reinterpret_cast<decltype(g_entry.dequantize)>(at[1]);
  g_entry.linear_workspace = reinterpret_cast<decltype(g_entry.linear_workspace)>(at[2]);
  g_entry.grad_workspace = reinterpret_cast<decltype(g_entry.grad_workspace)>(at[3]);
  g_entry.linear = reinterpret_cast<decltype(g_entry.linear)>(at[4]);
  g_entry.grad_input = reinterpret_cast<decltype(g_entry.grad_input)>(at[5]);
  Py_RETURN_NONE;
}

#define FAST(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {{"bind", bind, METH_VARARGS, nullptr}, FAST(linear), FAST(grad_input), FAST(dequantize), FAST(quantize),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_fp4_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fp4_calls() {
  const struct {
    PyObject** to;
    const char* name;
  } names[] = {{&g_qdata, "qdata"}, {&g_scale, "scale"}, {&g_second, "per_tensor_scale"}, {&g_swizzled, "is_swizzled_scales"},
               {&g_elem, "elem_dtype"}, {&g_block, "block_size"}, {&g_kwargs, "act_quant_kwargs"}, {&g_mode, "scaling_mode"},
               {&g_value, "value"}, {&g_dtype, "orig_dtype"}};
  for (const auto& n : names)
    if ((*n.to = PyUnicode_InternFromString(n.name)) == nullptr) return nullptr;
  return PyModule_Create(&g_module);
}
