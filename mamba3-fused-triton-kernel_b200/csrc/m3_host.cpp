// Host-side fast path of the language-model operators: the ordinary call of
// linear_w4, process_logits and next_tokens, from PyTorch tensors to the C
// entry point, without Python in between (the Python marshalling of
// src/kernels costs more than these kernels run for small batches).
//
// Every function takes the positional arguments of its Python counterpart
// and returns None for any call that it does not take as it stands: another
// type, layout, device or size, or one to be refused.  The Python path then
// checks, converts or raises; nothing is decided here that it would decide
// otherwise.
#include <Python.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "mamba3_b200_lm.h"

namespace {

using W4Fn = int (*)(const m3_w4_args *, m3_stream_t);
using LogitsFn = int (*)(const m3_logits_args *, m3_stream_t);
W4Fn linear_w4_fn = nullptr;
LogitsFn process_fn = nullptr, next_fn = nullptr;

bool is_tensor(PyObject *o) { return THPVariable_CheckExact(o); }
const at::Tensor &tensor(PyObject *o) { return THPVariable_Unpack(o); }

int dtype_code(at::ScalarType t) { return t == at::kFloat ? M3_F32 : t == at::kBFloat16 ? M3_BF16 : -1; }

bool on(const at::Tensor &t, int dev) { return t.is_cuda() && t.get_device() == dev; }

// it asks for a gradient, also a forward-mode one: the Python path refuses it
bool wants_gradient(const at::Tensor &t) {
  return (t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined();
}

m3_stream_t stream_of(int dev) {
  return reinterpret_cast<m3_stream_t>(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream());
}

// (x, codes, scales, zeros, group_size) -> y of x's type, or None
PyObject *linear_w4(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5 || !linear_w4_fn || !is_tensor(a[0]) || !is_tensor(a[1]) || !is_tensor(a[2]) || !PyLong_CheckExact(a[4]))
    Py_RETURN_NONE;
  const at::Tensor &x = tensor(a[0]), &codes = tensor(a[1]), &scales = tensor(a[2]);
  const long group = PyLong_AsLong(a[4]);
  if (group != 32 && group != 64 && group != 128) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (!x.is_cuda() || x.dim() != 2 || codes.dim() != 4 || scales.dim() != 2) Py_RETURN_NONE;
  const int dev = x.get_device(), xd = dtype_code(x.scalar_type()), sd = dtype_code(scales.scalar_type());
  const int64_t M = x.size(0), K = x.size(1), N = scales.size(0), groups = scales.size(1);
  if (xd < 0 || sd < 0 || M <= 0 || K <= 0 || N <= 0 || M > INT32_MAX || K > INT32_MAX || N > INT32_MAX ||
      !x.is_contiguous() || wants_gradient(x) || wants_gradient(scales) ||
      codes.scalar_type() != at::kInt || !codes.is_contiguous() || codes.size(0) != (N + 15) / 16 ||
      codes.size(1) != (K + 127) / 128 || codes.size(2) != 16 || codes.size(3) != 16 ||
      groups != (K + group - 1) / group || !scales.is_contiguous() || !on(codes, dev) || !on(scales, dev) ||
      c10::cuda::current_device() != dev)
    Py_RETURN_NONE;
  m3_w4_args w = {};
  if (a[3] != Py_None) {
    if (!is_tensor(a[3])) Py_RETURN_NONE;
    const at::Tensor &zeros = tensor(a[3]);
    if (zeros.scalar_type() != at::kByte || zeros.dim() != 2 || zeros.size(0) != N || zeros.size(1) != groups ||
        !zeros.is_contiguous() || !on(zeros, dev))
      Py_RETURN_NONE;
    w.zeros = static_cast<const uint8_t *>(zeros.data_ptr());
    w.zero_stride = groups;
  }
  at::Tensor y = at::empty({M, N}, x.options().requires_grad(false));
  w.M = (int32_t)M, w.N = (int32_t)N, w.K = (int32_t)K, w.group = (int32_t)group;
  w.x = x.data_ptr(), w.ldx = K, w.x_dtype = xd;
  w.codes = static_cast<const int32_t *>(codes.data_ptr());
  w.scales = scales.data_ptr(), w.scale_stride = groups, w.s_dtype = sd;
  w.y = y.data_ptr(), w.ldy = N, w.y_dtype = xd;
  if (linear_w4_fn(&w, stream_of(dev)) != M3_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// a (B,) fp32 tensor, a number, or None
bool per_row(PyObject *o, int64_t B, int dev, const float **ptr, float *value, float neutral) {
  *ptr = nullptr, *value = neutral;
  if (o == Py_None) return true;
  if (PyFloat_CheckExact(o)) {
    *value = (float)PyFloat_AS_DOUBLE(o);
    return true;
  }
  if (!is_tensor(o)) return false;
  const at::Tensor &t = tensor(o);
  if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != B || !t.is_contiguous() || !on(t, dev) ||
      wants_gradient(t))
    return false;
  *ptr = static_cast<const float *>(t.data_ptr());
  return true;
}

// a (B,) int32 or int64 tensor, or None
bool row_ints(PyObject *o, int64_t B, int dev, const void **ptr, int32_t *i64) {
  *ptr = nullptr, *i64 = 0;
  if (o == Py_None) return true;
  if (!is_tensor(o)) return false;
  const at::Tensor &t = tensor(o);
  if ((t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) || t.dim() != 1 || t.size(0) != B ||
      !t.is_contiguous() || !on(t, dev))
    return false;
  *ptr = t.data_ptr(), *i64 = t.scalar_type() == at::kLong;
  return true;
}

// a (width or more,) or (B, width or more) tensor of type `dt`, or None
bool shared_rows(PyObject *o, at::ScalarType dt, int64_t B, int64_t width, int dev, const void **ptr, int64_t *stride) {
  *ptr = nullptr, *stride = 0;
  if (o == Py_None) return true;
  if (!is_tensor(o)) return false;
  const at::Tensor &t = tensor(o);
  const int64_t d = t.dim();
  if (t.scalar_type() != dt || (d != 1 && d != 2) || t.size(d - 1) < width || t.stride(d - 1) != 1 ||
      (d == 2 && t.size(0) != B) || !on(t, dev) || wants_gradient(t))
    return false;
  *ptr = t.data_ptr(), *stride = d == 2 && B > 1 ? t.stride(0) : 0;
  return true;
}

// The nine arguments that both logit operators share.
bool adjust_args(PyObject *const *a, m3_logits_args *g, int *dev_out) {
  if (!is_tensor(a[0])) return false;
  const at::Tensor &logits = tensor(a[0]);
  if (!logits.is_cuda() || logits.dim() != 2) return false;
  const int dev = logits.get_device();
  const int64_t B = logits.size(0), V = logits.size(1);
  g->dtype = dtype_code(logits.scalar_type());
  if (g->dtype < 0 || B <= 0 || V <= 0 || B > INT32_MAX || V > (1 << 30) || logits.stride(1) != 1 ||
      wants_gradient(logits) || c10::cuda::current_device() != dev)
    return false;
  g->B = (int32_t)B, g->V = (int32_t)V, g->logits = logits.data_ptr(), g->ld = logits.stride(0);
  if (a[1] != Py_None) {
    if (!is_tensor(a[1])) return false;
    const at::Tensor &t = tensor(a[1]);
    if ((t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) || t.dim() != 2 || t.size(0) != B ||
        t.size(1) > INT32_MAX || (t.stride(1) != 1 && t.size(1) > 1) || !on(t, dev))
      return false;
    g->tokens = t.data_ptr(), g->T = (int32_t)t.size(1), g->tokens_stride = t.stride(0);
    g->tokens_i64 = t.scalar_type() == at::kLong;
  } else if (a[2] != Py_None || a[3] != Py_None) {
    return false;
  }
  const void *bias = nullptr, *allowed = nullptr;
  if (!row_ints(a[2], B, dev, &g->lengths, &g->lengths_i64) ||
      !row_ints(a[3], B, dev, &g->prompt_lengths, &g->prompt_i64) ||
      !per_row(a[4], B, dev, &g->repetition, &g->repetition_value, 1.f) || !(g->repetition_value > 0.f) ||
      !per_row(a[5], B, dev, &g->presence, &g->presence_value, 0.f) ||
      !per_row(a[6], B, dev, &g->frequency, &g->frequency_value, 0.f) ||
      !shared_rows(a[7], at::kFloat, B, V, dev, &bias, &g->bias_stride) ||
      !shared_rows(a[8], at::kInt, B, (V + 31) / 32, dev, &allowed, &g->allowed_stride))
    return false;
  g->bias = static_cast<const float *>(bias), g->allowed = static_cast<const int32_t *>(allowed);
  *dev_out = dev;
  return true;
}

// the nine arguments -> the adjusted logits, or None
PyObject *process_logits(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  m3_logits_args g = {};
  int dev = -1;
  if (n != 9 || !process_fn || !adjust_args(a, &g, &dev)) Py_RETURN_NONE;
  at::Tensor out = at::empty({g.B, g.V}, tensor(a[0]).options().requires_grad(false));
  g.out = out.data_ptr(), g.out_ld = g.V, g.out_dtype = g.dtype;
  if (process_fn(&g, stream_of(dev)) != M3_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// the nine arguments, temperature, seeds, positions -> (ids, logprobs), or None
PyObject *next_tokens(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  m3_logits_args g = {};
  int dev = -1;
  if (n != 12 || !next_fn || !adjust_args(a, &g, &dev)) Py_RETURN_NONE;
  if (a[9] != Py_None) {
    const void *seeds = nullptr, *positions = nullptr;
    int32_t s64 = 0, p64 = 0;
    g.sample = 1;
    if (!per_row(a[9], g.B, dev, &g.temperature, &g.temperature_value, 0.f) || a[10] == Py_None ||
        !row_ints(a[10], g.B, dev, &seeds, &s64) || !s64 || !row_ints(a[11], g.B, dev, &positions, &p64) ||
        (positions && !p64))
      Py_RETURN_NONE;
    g.seeds = static_cast<const int64_t *>(seeds), g.positions = static_cast<const int64_t *>(positions);
  }
  const auto options = tensor(a[0]).options().requires_grad(false);
  at::Tensor ids = at::empty({g.B}, options.dtype(at::kLong)), logprobs = at::empty({g.B}, options.dtype(at::kFloat));
  g.ids = static_cast<int64_t *>(ids.data_ptr()), g.logprobs = static_cast<float *>(logprobs.data_ptr());
  if (next_fn(&g, stream_of(dev)) != M3_OK) Py_RETURN_NONE;
  PyObject *i = THPVariable_Wrap(std::move(ids)), *p = THPVariable_Wrap(std::move(logprobs));
  PyObject *both = i && p ? PyTuple_Pack(2, i, p) : nullptr;
  Py_XDECREF(i);
  Py_XDECREF(p);
  return both;
  END_HANDLE_TH_ERRORS
}

// (linear_w4, process_logits, next_tokens): addresses of the C entry points
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "bind takes three addresses");
    return nullptr;
  }
  void *p[3];
  for (int i = 0; i < 3; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null address");
      return nullptr;
    }
  }
  linear_w4_fn = reinterpret_cast<W4Fn>(p[0]);
  process_fn = reinterpret_cast<LogitsFn>(p[1]);
  next_fn = reinterpret_cast<LogitsFn>(p[2]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
    {"linear_w4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_w4)), METH_FASTCALL, nullptr},
    {"process_logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(process_logits)), METH_FASTCALL,
     nullptr},
    {"next_tokens", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(next_tokens)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "m3_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: the PyTorch whose object layouts are compiled in here
PyMODINIT_FUNC PyInit_m3_host() {
  PyObject *m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", M3_TORCH_VERSION) < 0) Py_CLEAR(m);
  return m;
}
