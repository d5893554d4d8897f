// The common case of the 4-bit operators' wrappers, without the interpreter: a
// product for one token takes the GPU about 5 us and its Python wrapper took the
// host 11.  Each function checks that its arguments are what the kernels take as
// they are (plain tensors on the current device, right types and shapes,
// contiguous where that is needed, no gradient wanted), allocates the result and
// calls the C ABI of libqi8.  For anything else, and for any error, it returns
// None: the Python wrapper then goes its own way, which converts what can be
// converted and raises what has to be raised.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "../../include/qi8.h"

namespace {

decltype(&qi8_quant_weight_i4) quant_fn;
decltype(&qi8_dequant_i4) dequant_fn;
decltype(&qi8_gemm_w4) gemm_fn;
decltype(&qi8_moe_w4) moe_fn;
decltype(&qi8_moe_w4_workspace_bytes) moe_bytes_fn;

int code(at::ScalarType t) {
  return t == at::kBFloat16 ? QI8_BF16 : t == at::kHalf ? QI8_F16 : t == at::kFloat ? QI8_F32 : -1;
}
int64_t padded(int64_t k) { return (k + 127) / 128 * 128; }

const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

// A Python integer of 64 bits; -1, which no argument here may be, for all others.
int64_t integer(PyObject* o) {
  if (!PyLong_CheckExact(o)) return -1;
  int overflow = 0;
  const int64_t v = PyLong_AsLongLongAndOverflow(o, &overflow);  // raises nothing
  return overflow ? -1 : v;
}

// On the current device, and nobody waits for its gradient or has given it a tangent.
bool plain(const at::Tensor& t, int device) {
  return t.is_cuda() && t.layout() == at::kStrided && t.get_device() == device &&
         !(c10::GradMode::is_enabled() && t.requires_grad()) && !t._fw_grad(0).defined();
}

// q [..., n, padded(k) / 2] and s [..., n, padded(k) / group], `dims` dimensions
bool weight(const at::Tensor& q, const at::Tensor& s, int64_t k, int64_t group, int64_t dims, int device) {
  if ((group != 32 && group != 64 && group != 128) || k <= 0) return false;
  if (!plain(q, device) || !plain(s, device) || q.scalar_type() != at::kByte || s.scalar_type() != at::kBFloat16)
    return false;
  if (q.dim() != dims || s.dim() != dims || !q.is_contiguous() || !s.is_contiguous()) return false;
  for (int64_t i = 0; i + 1 < dims; ++i)
    if (q.size(i) != s.size(i)) return false;
  return q.size(dims - 1) * 2 == padded(k) && s.size(dims - 1) * group == padded(k);
}

// Activations as they are: 16 bits, contiguous, rows on 16-byte boundaries.
bool activations(const at::Tensor& x, int device) {
  return plain(x, device) && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf) && x.dim() >= 2 &&
         x.is_contiguous() && x.numel() > 0;
}

void* stream(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (...) {  // the Python wrapper meets the same error and reports it
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// x, q, scale, group, bias or None
PyObject* gemm_w4(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 5 || !gemm_fn) Py_RETURN_NONE;
    const at::Tensor *x = tensor(args[0]), *q = tensor(args[1]), *s = tensor(args[2]);
    const at::Tensor* b = args[4] == Py_None ? nullptr : tensor(args[4]);
    if (!x || !q || !s || (!b && args[4] != Py_None)) Py_RETURN_NONE;
    const int64_t group = integer(args[3]);
    const int device = c10::cuda::current_device();
    if (!activations(*x, device)) Py_RETURN_NONE;
    const int64_t k = x->size(-1), m = x->numel() / k, n = q->dim() == 2 ? q->size(0) : 0;
    if (!weight(*q, *s, k, group, 2, device) || n == 0) Py_RETURN_NONE;
    if (m > 16 && (k % 8 || reinterpret_cast<uintptr_t>(x->data_ptr()) % 16)) Py_RETURN_NONE;  // wants a workspace
    if (b && (!plain(*b, device) || b->dim() != 1 || b->size(0) != n || !b->is_contiguous() ||
              code(b->scalar_type()) < 0))
      Py_RETURN_NONE;
    at::Tensor out;
    if (x->dim() == 2) {
      out = at::empty({m, n}, x->options());
    } else {
      std::vector<int64_t> shape(x->sizes().begin(), x->sizes().end());
      shape.back() = n;
      out = at::empty(shape, x->options());
    }
    const int dt = code(x->scalar_type());
    if (gemm_fn(x->data_ptr(), dt, m, k, k, static_cast<const uint8_t*>(q->data_ptr()), s->data_ptr(), n, (int)group,
                b ? b->data_ptr() : nullptr, b ? code(b->scalar_type()) : 0, out.data_ptr(), dt, n, nullptr, 0,
                stream(device)))
      Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// w, group
PyObject* quant_weight_i4(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 2 || !quant_fn) Py_RETURN_NONE;
    const at::Tensor* w = tensor(args[0]);
    if (!w) Py_RETURN_NONE;
    const int64_t group = integer(args[1]);
    const int device = c10::cuda::current_device();
    if (!plain(*w, device) || w->dim() < 2 || !w->is_contiguous() || w->numel() == 0 || code(w->scalar_type()) < 0 ||
        (group != 32 && group != 64 && group != 128))
      Py_RETURN_NONE;
    const int64_t k = w->size(-1), kp = padded(k);
    std::vector<int64_t> shape(w->sizes().begin(), w->sizes().end());
    shape.back() = kp / 2;
    at::Tensor q = at::empty(shape, w->options().dtype(at::kByte));
    shape.back() = kp / group;
    at::Tensor s = at::empty(shape, w->options().dtype(at::kBFloat16));
    if (quant_fn(w->data_ptr(), code(w->scalar_type()), w->numel() / k, k, k, (int)group,
                 static_cast<uint8_t*>(q.data_ptr()), s.data_ptr(), stream(device)))
      Py_RETURN_NONE;
    PyObject* pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(q)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(s)));
    return pair;
  });
}

// q, scale, k, group, output dtype
PyObject* dequant_i4(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 5 || !dequant_fn) Py_RETURN_NONE;
    const at::Tensor *q = tensor(args[0]), *s = tensor(args[1]);
    if (!q || !s || !THPDtype_Check(args[4])) Py_RETURN_NONE;
    const int64_t k = integer(args[2]), group = integer(args[3]);
    const at::ScalarType t = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
    const int device = c10::cuda::current_device();
    if (code(t) < 0 || q->dim() < 2 || q->numel() == 0 || !weight(*q, *s, k, group, q->dim(), device)) Py_RETURN_NONE;
    std::vector<int64_t> shape(q->sizes().begin(), q->sizes().end());
    shape.back() = k;
    at::Tensor out = at::empty(shape, q->options().dtype(t));
    if (dequant_fn(static_cast<const uint8_t*>(q->data_ptr()), s->data_ptr(), out.numel() / k, k, (int)group,
                   out.data_ptr(), code(t), k, stream(device)))
      Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// x, router, q13, s13, q2, s2, top_k, group, renormalize, activation code
PyObject* moe_w4(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 10 || !moe_fn) Py_RETURN_NONE;
    const at::Tensor* t[6];
    for (int i = 0; i < 6; ++i)
      if (!(t[i] = tensor(args[i]))) Py_RETURN_NONE;
    if (!PyBool_Check(args[8])) Py_RETURN_NONE;
    const int64_t top_k = integer(args[6]), group = integer(args[7]), act = integer(args[9]);
    const int device = c10::cuda::current_device();
    const at::Tensor &x = *t[0], &router = *t[1], &q13 = *t[2], &q2 = *t[4];
    if (!activations(x, device) || !plain(router, device) || router.dim() != 2 || !router.is_contiguous())
      Py_RETURN_NONE;
    const int64_t h = x.size(-1), tokens = x.numel() / h;
    if (q13.dim() != 3 || !weight(q13, *t[3], h, group, 3, device) || q13.size(1) % 2) Py_RETURN_NONE;
    const int64_t e = q13.size(0), i = q13.size(1) / 2;
    if (q2.dim() != 3 || !weight(q2, *t[5], i, group, 3, device) || q2.size(0) != e || q2.size(1) != h ||
        router.size(0) != e || router.size(1) != h || top_k <= 0 || top_k > e || act < 0 || act > QI8_ACT_SILU)
      Py_RETURN_NONE;
    const int64_t bytes = moe_bytes_fn(tokens, h, e, i, (int)top_k);
    if (bytes <= 0) Py_RETURN_NONE;
    at::Tensor out = at::empty(x.sizes(), x.options());
    at::Tensor ws = at::empty({bytes}, x.options().dtype(at::kByte));
    if (moe_fn(x.data_ptr(), code(x.scalar_type()), tokens, h, h, router.data_ptr(), code(router.scalar_type()), e,
               static_cast<const uint8_t*>(q13.data_ptr()), t[3]->data_ptr(), i,
               static_cast<const uint8_t*>(q2.data_ptr()), t[5]->data_ptr(), (int)group, (int)top_k,
               args[8] == Py_True, (int)act, out.data_ptr(), h, ws.data_ptr(), bytes,
               stream(device)))
      Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// addresses of qi8_quant_weight_i4, qi8_dequant_i4, qi8_gemm_w4, qi8_moe_w4, qi8_moe_w4_workspace_bytes
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  void* p[5];
  if (n_args != 5) {
    PyErr_SetString(PyExc_TypeError, "bind takes five addresses");
    return nullptr;
  }
  for (int i = 0; i < 5; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  quant_fn = reinterpret_cast<decltype(quant_fn)>(p[0]);
  dequant_fn = reinterpret_cast<decltype(dequant_fn)>(p[1]);
  gemm_fn = reinterpret_cast<decltype(gemm_fn)>(p[2]);
  moe_fn = reinterpret_cast<decltype(moe_fn)>(p[3]);
  moe_bytes_fn = reinterpret_cast<decltype(moe_bytes_fn)>(p[4]);
  Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(gemm_w4), FAST(quant_weight_i4), FAST(dequant_i4), FAST(moe_w4), FAST(bind),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__call() { return PyModule_Create(&module_def); }
