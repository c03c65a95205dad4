// The eager calls of the few-bits operators, from Python to libftk without ctypes (module kernels._calls).
//
// Each function takes the tensors of its Python counterpart, checks that the call is the plain case the counterpart
// documents (types, shapes, devices, strides), allocates the output and launches. Whatever is not that case -- a wrong
// type, a view that needs a copy, another device than the current one, no rows -- gives None, nothing launched, and
// the Python function does the rest: it names what is wrong, or makes the copy. A small call's host time is most of
// what it takes: 4096 x 1024 at one row is issued in 4.8 us, 12 less than through ctypes; the kernel runs 3.7.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPFunctions.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/ftk.h"

namespace {

// The tensor behind a Python object that is exactly a tensor or a parameter (no subclass with calls of its own).
const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool on(const at::Tensor& t, int device, at::ScalarType type) {
  return t.scalar_type() == type && t.is_cuda() && t.get_device() == device && t.layout() == at::kStrided;
}
bool plain(const at::Tensor& t, int device, at::ScalarType type) { return on(t, device, type) && t.is_contiguous(); }
bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }

void* stream_of(int device) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device).stream(); }

at::Tensor empty(at::IntArrayRef sizes, int device, at::ScalarType type) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, (c10::DeviceIndex)device)));
}

bool integer(PyObject* o, long long& v) {
  if (!PyLong_CheckExact(o)) return false;
  v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
bool number(PyObject* o, double& v) {
  if (!PyFloat_CheckExact(o)) return false;
  v = PyFloat_AS_DOUBLE(o);
  return true;
}

// w4(x, handle, device, outputs, norm_weight or None, eps, residual or None)
PyObject* w4(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  long long address, device, outputs;
  double eps;
  if (n != 7 || !integer(args[1], address) || !integer(args[2], device) || !integer(args[3], outputs) ||
      !number(args[5], eps))
    Py_RETURN_NONE;
  const at::Tensor* x = tensor(args[0]);
  if (!x || !on(*x, (int)device, at::kBFloat16) || c10::hip::current_device() != device) Py_RETURN_NONE;
  const auto* w = reinterpret_cast<const ftk_w4*>(address);
  const int64_t dims = x->dim(), K = w->K;
  if (dims < 1 || x->size(dims - 1) != K) Py_RETURN_NONE;
  int64_t rows = 1, stride = K;
  if (dims == 2) {
    rows = x->size(0);
    stride = x->stride(0);
    if (x->stride(1) != 1 || (stride < K && rows > 1)) Py_RETURN_NONE;
  } else {
    if (!x->is_contiguous()) Py_RETURN_NONE;
    rows = x->numel() / K;
  }
  if (rows < 1 || rows > FTK_MAX_ROWS) Py_RETURN_NONE;
  const void* gain = nullptr;
  if (args[4] != Py_None) {
    const at::Tensor* t = tensor(args[4]);
    if (!t || !plain(*t, (int)device, at::kBFloat16) || t->dim() != 1 || t->size(0) != K) Py_RETURN_NONE;
    gain = t->data_ptr();
  }
  at::DimVector shape(x->sizes());
  shape[dims - 1] = outputs;
  const void* residual = nullptr;
  if (args[6] != Py_None) {
    const at::Tensor* t = tensor(args[6]);
    if (!t || !plain(*t, (int)device, at::kBFloat16) || t->sizes() != at::IntArrayRef(shape)) Py_RETURN_NONE;
    residual = t->data_ptr();
  }
  at::Tensor y = empty(shape, (int)device, at::kBFloat16);
  if (ftk_w4_project_bf16(x->data_ptr(), stride, gain, (float)eps, w, residual, y.data_ptr(), rows,
                          stream_of((int)device)) != FTK_OK)
    Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// A cache's codes and scales: its type and block, or false.
struct Cache {
  const at::Tensor *keys, *values, *k_scales, *v_scales;
  int64_t batch, heads, capacity, dim, block;
  int type, device;
};
bool cache_of(PyObject* const* args, Cache& c) {
  c.keys = tensor(args[0]);
  c.values = tensor(args[1]);
  c.k_scales = tensor(args[2]);
  c.v_scales = tensor(args[3]);
  if (!c.keys || !c.values || !c.k_scales || !c.v_scales || !c.keys->is_cuda()) return false;
  c.device = c.keys->get_device();
  const at::ScalarType type = c.keys->scalar_type();
  if (type != at::kFloat8_e4m3fn && type != at::kChar) return false;
  c.type = type == at::kChar ? FTK_Q8_INT8 : FTK_Q8_E4M3;
  if (!plain(*c.keys, c.device, type) || !plain(*c.values, c.device, type) ||
      !plain(*c.k_scales, c.device, at::kFloat) || !plain(*c.v_scales, c.device, at::kFloat))
    return false;
  if (c.keys->dim() != 4 || c.keys->sizes() != c.values->sizes() || c.k_scales->dim() != 3 ||
      c.k_scales->sizes() != c.v_scales->sizes())
    return false;
  c.batch = c.keys->size(0);
  c.heads = c.keys->size(1);
  c.capacity = c.keys->size(2);
  c.dim = c.keys->size(3);
  if (c.batch < 1 || c.heads < 1 || c.capacity < 1 || (c.dim != 64 && c.dim != 128)) return false;
  if (c.k_scales->size(0) != c.batch || c.k_scales->size(1) != c.heads) return false;
  for (c.block = 16; c.block <= 128; c.block *= 2)
    if ((c.capacity + c.block - 1) / c.block == c.k_scales->size(2)) break;
  return c.block <= 128 && aligned16(*c.keys) && aligned16(*c.values) && c10::hip::current_device() == c.device;
}

// attend(query, keys, values, k_scales, v_scales, position, scale, splits)
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Cache c;
  double scale;
  long long splits;
  if (n != 8 || !cache_of(args + 1, c) || !number(args[6], scale) || !integer(args[7], splits)) Py_RETURN_NONE;
  const at::Tensor *q = tensor(args[0]), *position = tensor(args[5]);
  if (!q || !position || !plain(*q, c.device, at::kBFloat16) || !plain(*position, c.device, at::kLong)) Py_RETURN_NONE;
  if (q->dim() != 4 || q->size(0) != c.batch || q->size(2) != 1 || q->size(3) != c.dim || !aligned16(*q)) Py_RETURN_NONE;
  const int64_t heads = q->size(1), positions = position->numel();
  if (position->dim() != 1 || (positions != 1 && positions != c.batch)) Py_RETURN_NONE;
  if (splits < 0 || splits > INT32_MAX) Py_RETURN_NONE;
  if (splits == 0) splits = ftk_decode_attention_q8_splits(c.batch, heads, c.heads, c.capacity, c.dim, 0);
  if (splits < 1) Py_RETURN_NONE;
  const int64_t need = ftk_decode_attention_q8_workspace_bytes(c.batch, heads, c.heads, c.dim, (int)splits);
  if (need < 0) Py_RETURN_NONE;
  at::Tensor out = empty({c.batch, 1, heads, c.dim}, c.device, at::kBFloat16), ws;
  if (need > 0) ws = empty({need}, c.device, at::kByte);
  if (ftk_decode_attention_q8(q->data_ptr(), c.keys->data_ptr(), c.values->data_ptr(),
                              (const float*)c.k_scales->data_ptr(), (const float*)c.v_scales->data_ptr(),
                              (const int64_t*)position->data_ptr(), (int)positions, out.data_ptr(), c.batch, heads,
                              c.heads, c.capacity, c.dim, c.block, c.type, scale, (int)splits,
                              need > 0 ? ws.data_ptr() : nullptr, need, stream_of(c.device)) != FTK_OK)
    Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// write(packed, q_weight, k_weight, q_eps, k_eps, cos, sin, position, keys, values, k_scales, v_scales, q_heads,
//       prefill, rows, phases or None)
PyObject* write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Cache c;
  double q_eps, k_eps;
  long long q_heads;
  if (n != 16 || !cache_of(args + 8, c) || !number(args[3], q_eps) || !number(args[4], k_eps) ||
      !integer(args[12], q_heads) || q_heads < 1 || !PyBool_Check(args[13]) || !PyBool_Check(args[14]))
    Py_RETURN_NONE;
  const bool prefill = args[13] == Py_True, rows = args[14] == Py_True;
  const at::Tensor *packed = tensor(args[0]), *qw = tensor(args[1]), *kw = tensor(args[2]), *cos = tensor(args[5]),
                   *sin = tensor(args[6]), *position = tensor(args[7]);
  for (const at::Tensor* t : {packed, qw, kw, cos, sin})
    if (!t || !plain(*t, c.device, at::kBFloat16)) Py_RETURN_NONE;
  if (!position || !plain(*position, c.device, at::kLong) || (prefill && rows)) Py_RETURN_NONE;
  if (packed->dim() != 3 || packed->size(0) != c.batch || packed->size(2) != (q_heads + 2 * c.heads) * c.dim)
    Py_RETURN_NONE;
  const int64_t tokens = packed->size(1);
  if (tokens < 1 || tokens > c.capacity || qw->numel() != c.dim || kw->numel() != c.dim) Py_RETURN_NONE;
  const void* phases = nullptr;
  if (args[15] != Py_None) {
    const at::Tensor* t = tensor(args[15]);
    if (!t || !rows || !plain(*t, c.device, at::kLong) || t->dim() != 2 || t->size(0) != c.batch ||
        t->size(1) != tokens || cos->dim() < 1 || cos->sizes() != sin->sizes() || cos->size(cos->dim() - 1) != c.dim)
      Py_RETURN_NONE;
    phases = t->data_ptr();
  } else if (cos->numel() != (rows ? c.batch : 1) * tokens * c.dim || sin->numel() != cos->numel()) {
    Py_RETURN_NONE;
  }
  if (position->dim() != 1 || position->numel() != (prefill ? tokens : rows ? c.batch : 1)) Py_RETURN_NONE;
  at::Tensor query = empty({c.batch, tokens, q_heads, c.dim}, c.device, at::kBFloat16);
  const int mode = (prefill ? FTK_ROPE_PREFILL : 0) | (rows ? FTK_ROPE_ROWS : 0) | (phases ? FTK_ROPE_TABLE : 0);
  if (ftk_qk_rope_cache_q8(packed->data_ptr(), qw->data_ptr(), kw->data_ptr(), (float)q_eps, (float)k_eps,
                           cos->data_ptr(), sin->data_ptr(), cos->numel() / c.dim,
                           (const int64_t*)position->data_ptr(), (const int64_t*)phases, query.data_ptr(),
                           c.keys->data_ptr(), c.values->data_ptr(), (float*)c.k_scales->data_ptr(),
                           (float*)c.v_scales->data_ptr(), c.batch, tokens, q_heads, c.heads, c.capacity, c.dim,
                           c.block, c.type, mode, stream_of(c.device)) != FTK_OK)
    Py_RETURN_NONE;
  return THPVariable_Wrap(query.transpose(1, 2));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"w4", (PyCFunction)(void*)w4, METH_FASTCALL, "A 4-bit projection's plain call, or None."},
    {"attend", (PyCFunction)(void*)attend, METH_FASTCALL, "Attention over an 8-bit cache, the plain call, or None."},
    {"write", (PyCFunction)(void*)write, METH_FASTCALL, "The 8-bit cache's write, the plain call, or None."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Eager calls of the few-bits operators.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
