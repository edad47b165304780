// The functional forms of the dynamic Linear and the expert operators as one native call each, for eager decode
// loops where the host sets the pace: checking a call's tensors, allocating its results and marshalling some
// twenty-five arguments takes 8 to 10 us in Python and about 2 us here.
//
// A function here serves the ordinary call only -- plain CUDA tensors of the current device, dense rows, the
// documented types and shapes -- and returns None for every other one; the Python form then converts, copies or
// refuses as it documents.  No refusal and no conversion is written twice.  An entry point's status other than 0
// comes back as an int.  C++ exceptions (out of memory) become Python's.
//
// Like _fastcall, the module does not link against liblucid_cuda: `bind(name, address)` hands it the entry points.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "lucid_cuda.h"

namespace {

decltype(&lc_expert_linear) p_expert_linear;
decltype(&lc_expert_linear_workspace_bytes) p_expert_linear_bytes;
decltype(&lc_route_experts) p_route_experts;
decltype(&lc_route_experts_workspace_bytes) p_route_experts_bytes;
decltype(&lc_combine_experts) p_combine_experts;

// the tensor behind an argument, or null: None, a subclass or another object
const at::Tensor* tensor(PyObject* o) {
  return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}
int float_code(at::ScalarType t) {
  return t == at::kFloat ? LC_F32 : t == at::kBFloat16 ? LC_BF16 : t == at::kHalf ? LC_F16 : -1;
}
bool dense_rows(const at::Tensor& t) { return t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= t.size(1); }
bool on(const at::Tensor& t, c10::DeviceIndex device) { return t.is_cuda() && t.get_device() == device; }

// an fp32 parameter of the given shape ([n], or [e, n] when e > 0); None is allowed where `optional`
bool parameter(PyObject* o, c10::DeviceIndex device, int64_t e, int64_t n, bool optional, const float** data) {
  *data = nullptr;
  if (o == Py_None) return optional;
  const at::Tensor* t = tensor(o);
  if (!t || !on(*t, device) || t->scalar_type() != at::kFloat || !t->is_contiguous()) return false;
  if (e > 0 ? t->dim() != 2 || t->size(0) != e || t->size(1) != n : t->dim() != 1 || t->size(0) != n) return false;
  *data = static_cast<const float*>(t->data_ptr());
  return true;
}
// a residual of the result's type and shape
bool residual_rows(PyObject* o, c10::DeviceIndex device, at::ScalarType type, int64_t rows, int64_t cols,
                   const void** data, int64_t* ld) {
  *data = nullptr;
  *ld = 0;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o);
  if (!t || !on(*t, device) || t->scalar_type() != type || !dense_rows(*t) || t->size(0) != rows || t->size(1) != cols)
    return false;
  *data = t->data_ptr();
  *ld = t->stride(0);
  return true;
}
const int32_t* int_data(const at::Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }
bool is_int32(const at::Tensor* t, c10::DeviceIndex device, int64_t dim) {
  return t && on(*t, device) && t->scalar_type() == at::kInt && t->dim() == dim && t->is_contiguous();
}
PyObject* none() { Py_RETURN_NONE; }

// product(x, weight, weight_scale, bias, activation, residual, out_dtype, positions, offsets)
//   dense: weight [N, K], positions and offsets None; experts: weight [E, N, K], offsets [E + 1], positions [T, k], or the
//   int tokens * top_k when the rows of x are in expert order
PyObject* product(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 9 || !p_expert_linear) return PyErr_Format(PyExc_TypeError, "product takes 9 arguments and needs bind()");
  const at::Tensor *x = tensor(args[0]), *w = tensor(args[1]);
  if (!x || !w || !x->is_cuda()) return none();
  const c10::DeviceIndex device = x->get_device();
  const bool experts = args[8] != Py_None;
  const int64_t lead = experts ? 1 : 0;
  if (device != c10::cuda::current_device() || !dense_rows(*x) || float_code(x->scalar_type()) < 0) return none();
  if (!on(*w, device) || w->scalar_type() != at::kChar || w->dim() != 2 + lead) return none();
  const int64_t e = experts ? w->size(0) : 0, n = w->size(lead), k = w->size(lead + 1), ldw = w->stride(lead);
  const int64_t stride = experts ? w->stride(0) : 0;
  if (k != x->size(1) || k < 1 || n < 1 || w->stride(lead + 1) != 1 || ldw < k || ldw % 16 || stride % 16 ||
      (e > 1 && stride < n * ldw) || reinterpret_cast<uintptr_t>(w->data_ptr()) % 16)
    return none();
  const long act = PyLong_AsLong(args[4]);
  if (act < LC_ACT_NONE || act > LC_ACT_SWIGLU || (act == LC_ACT_SWIGLU && n % 16)) return PyErr_Occurred() ? nullptr : none();
  at::ScalarType type = x->scalar_type();
  if (args[6] != Py_None) {
    if (!THPDtype_Check(args[6])) return none();
    type = reinterpret_cast<THPDtype*>(args[6])->scalar_type;
    if (float_code(type) < 0) return none();
  }
  const int64_t width = act == LC_ACT_SWIGLU ? n / 2 : n;
  int64_t rows = x->size(0), top_k = 1;
  const int32_t *positions = nullptr, *offsets = nullptr;
  if (experts) {
    const at::Tensor* o = tensor(args[8]);
    if (!is_int32(o, device, 1) || o->size(0) != e + 1 || e < 1 || e > 1024) return none();
    offsets = int_data(*o);
    if (PyLong_Check(args[7])) {
      if (PyLong_AsLongLong(args[7]) != rows) return none();
    } else {
      const at::Tensor* p = tensor(args[7]);
      if (!is_int32(p, device, 2) || p->size(0) != rows) return none();
      positions = int_data(*p);
      top_k = p->size(1);
      rows *= top_k;
    }
  }
  if (rows < 1) return none();
  const float *scale, *bias;
  const void* residual;
  int64_t ldr;
  if (!parameter(args[2], device, e, n, false, &scale) || !parameter(args[3], device, e, n, true, &bias) ||
      !residual_rows(args[5], device, type, rows, width, &residual, &ldr))
    return none();
  const int64_t need = p_expert_linear_bytes(rows, k);
  at::Tensor out = at::empty({rows, width}, x->options().dtype(type));
  at::Tensor work = at::empty({need}, x->options().dtype(at::kByte));
  const int32_t rc = p_expert_linear(x->data_ptr(), float_code(x->scalar_type()), x->size(0), x->stride(0), positions, top_k,
                                     offsets, experts ? e : 1, rows, static_cast<const int8_t*>(w->data_ptr()), ldw, stride, n,
                                     k, scale, bias, static_cast<int32_t>(act), residual, ldr, out.data_ptr(),
                                     float_code(type), width, work.data_ptr(), need, nullptr,
                                     c10::cuda::getCurrentCUDAStream(device).stream());
  if (rc != LC_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// route(logits, top_k, renormalize) -> (weights, experts, offsets, positions)
PyObject* route(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 3 || !p_route_experts) return PyErr_Format(PyExc_TypeError, "route takes 3 arguments and needs bind()");
  const at::Tensor* x = tensor(args[0]);
  if (!x || !x->is_cuda() || !PyLong_Check(args[1])) return none();
  const c10::DeviceIndex device = x->get_device();
  if (device != c10::cuda::current_device() || !dense_rows(*x) || float_code(x->scalar_type()) < 0) return none();
  const int64_t tokens = x->size(0), experts = x->size(1), top_k = PyLong_AsLongLong(args[1]);
  const int renormalize = PyObject_IsTrue(args[2]);
  if (renormalize < 0 || PyErr_Occurred()) return nullptr;
  if (tokens < 1 || experts < 1 || experts > 1024 || top_k < 1 || top_k > 32 || top_k > experts) return none();
  const auto ints = x->options().dtype(at::kInt);
  at::Tensor weights = at::empty({tokens, top_k}, x->options().dtype(at::kFloat));
  at::Tensor chosen = at::empty({tokens, top_k}, ints), positions = at::empty({tokens, top_k}, ints);
  at::Tensor offsets = at::empty({experts + 1}, ints), work;
  const int64_t need = p_route_experts_bytes(tokens, experts);
  if (need > 0) work = at::empty({need}, x->options().dtype(at::kByte));
  const int32_t rc = p_route_experts(x->data_ptr(), float_code(x->scalar_type()), tokens, experts, x->stride(0), top_k,
                                     renormalize, static_cast<float*>(weights.data_ptr()),
                                     static_cast<int32_t*>(chosen.data_ptr()), static_cast<int32_t*>(offsets.data_ptr()),
                                     static_cast<int32_t*>(positions.data_ptr()), need > 0 ? work.data_ptr() : nullptr, need,
                                     c10::cuda::getCurrentCUDAStream(device).stream());
  if (rc != LC_OK) return PyLong_FromLong(rc);
  return Py_BuildValue("(NNNN)", THPVariable_Wrap(std::move(weights)), THPVariable_Wrap(std::move(chosen)),
                       THPVariable_Wrap(std::move(offsets)), THPVariable_Wrap(std::move(positions)));
  END_HANDLE_TH_ERRORS
}

// combine(y, weights, positions, residual)
PyObject* combine(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 4 || !p_combine_experts) return PyErr_Format(PyExc_TypeError, "combine takes 4 arguments and needs bind()");
  const at::Tensor *y = tensor(args[0]), *w = tensor(args[1]), *p = tensor(args[2]);
  if (!y || !w || !y->is_cuda()) return none();
  const c10::DeviceIndex device = y->get_device();
  if (device != c10::cuda::current_device() || !dense_rows(*y) || float_code(y->scalar_type()) < 0 || y->size(1) < 1 ||
      !is_int32(p, device, 2))
    return none();
  const int64_t tokens = p->size(0), top_k = p->size(1);
  if (tokens < 1 || top_k < 1 || y->size(0) != tokens * top_k || !on(*w, device) || w->scalar_type() != at::kFloat ||
      w->dim() != 2 || w->size(0) != tokens || w->size(1) != top_k || !w->is_contiguous())
    return none();
  const void* residual;
  int64_t ldr;
  if (!residual_rows(args[3], device, y->scalar_type(), tokens, y->size(1), &residual, &ldr)) return none();
  at::Tensor out = at::empty({tokens, y->size(1)}, y->options());
  const int32_t rc = p_combine_experts(y->data_ptr(), float_code(y->scalar_type()), y->size(0), y->size(1), y->stride(0),
                                       static_cast<const float*>(w->data_ptr()), int_data(*p), tokens, top_k, residual, ldr,
                                       out.data_ptr(), y->size(1), c10::cuda::getCurrentCUDAStream(device).stream());
  if (rc != LC_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* bind(PyObject*, PyObject* args) {
  const char* name;
  unsigned long long address;
  if (!PyArg_ParseTuple(args, "sK", &name, &address)) return nullptr;
  void* const p = reinterpret_cast<void*>(static_cast<uintptr_t>(address));
  const std::string key(name);
  if (key == "lc_expert_linear") p_expert_linear = reinterpret_cast<decltype(p_expert_linear)>(p);
  else if (key == "lc_expert_linear_workspace_bytes") p_expert_linear_bytes = reinterpret_cast<decltype(p_expert_linear_bytes)>(p);
  else if (key == "lc_route_experts") p_route_experts = reinterpret_cast<decltype(p_route_experts)>(p);
  else if (key == "lc_route_experts_workspace_bytes") p_route_experts_bytes = reinterpret_cast<decltype(p_route_experts_bytes)>(p);
  else if (key == "lc_combine_experts") p_combine_experts = reinterpret_cast<decltype(p_combine_experts)>(p);
  else return PyErr_Format(PyExc_KeyError, "no binding for %s", name);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, "bind(name, address): the address of a liblucid_cuda entry point"},
    {"product", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(product)), METH_FASTCALL, "dense or grouped product"},
    {"route", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(route)), METH_FASTCALL, "router"},
    {"combine", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(combine)), METH_FASTCALL, "combination"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torchcall", "eager calls into liblucid_cuda on torch tensors", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__torchcall(void) { return PyModule_Create(&module); }
