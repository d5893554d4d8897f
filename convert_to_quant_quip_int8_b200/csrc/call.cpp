// The common case of the 4-bit and fp8 operators' wrappers, without the
// interpreter: a product for one token takes the GPU about 5 us and its Python
// wrapper took the host 11 (4 bits) or 20 (fp8), with this 5.  Each function checks
// that its arguments are what the kernels take as they are (plain tensors on the
// current device, right types and shapes, contiguous where that is needed, no
// gradient wanted), allocates the result and calls the C ABI of libqi8.  For anything
// else, and for any error, it returns None: the Python wrapper then goes its own way,
// which converts what can be converted and raises what has to be raised.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <type_traits>
#include <vector>

#include "../../include/qi8.h"

namespace {

decltype(&qi8_quant_weight_i4) quant_fn;
decltype(&qi8_dequant_i4) dequant_fn;
decltype(&qi8_gemm_w4) gemm_fn;
decltype(&qi8_moe_w4) moe_fn;
decltype(&qi8_moe_w4_workspace_bytes) moe_bytes_fn;
decltype(&qi8_quant_rows_f8) quant_rows_f8_fn;
decltype(&qi8_quant_weight_f8) quant_weight_f8_fn;
decltype(&qi8_gemm_f8_workspace_bytes) gemm_f8_bytes_fn;
decltype(&qi8_gemm_f8) gemm_f8_fn;
decltype(&qi8_linear_f8_workspace_bytes) linear_f8_bytes_fn;
decltype(&qi8_linear_f8) linear_f8_fn;
decltype(&qi8_rms_norm_quant) norm_fn;
decltype(&qi8_gated_quant) gated_fn;
decltype(&qi8_dequant) dequant8_fn;

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

// On the current device, its memory as it reads, and nobody waits for its gradient or
// has given it a tangent.
bool plain(const at::Tensor& t, int device) {
  return t.is_cuda() && t.layout() == at::kStrided && t.get_device() == device && !t.is_neg() &&
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

// ---------------------------------------------------------------- fp8

// at::empty on the current device, past the dispatcher: three of them were half of a call.
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_generic(sizes, c10::cuda::CUDACachingAllocator::get(),
                                   c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}

constexpr int64_t F8_BLOCK = 128;
int64_t blocks(int64_t n) { return (n + F8_BLOCK - 1) / F8_BLOCK; }

// A float type on the current device with at least one element.
bool numbers(const at::Tensor& t, int device) {
  return plain(t, device) && code(t.scalar_type()) >= 0 && t.dim() >= 1 && t.numel() > 0;
}

// Whether `t` [..., n] is rows with unit column stride a fixed stride apart, which is
// what the kernels take: that stride, or -1.
int64_t row_stride(const at::Tensor& t) {
  const int64_t d = t.dim(), n = t.size(d - 1);
  if (t.stride(d - 1) != 1 && n > 1) return -1;
  if (d == 1 || t.numel() == n) return n;
  int64_t step = -1, ld = 0;  // stride that the next outer dimension has to have
  for (int64_t i = d - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (step < 0) ld = t.stride(i);
    else if (t.stride(i) != step) return -1;
    step = t.stride(i) * t.size(i);
  }
  return ld >= n ? ld : -1;
}

// e4m3 codes [..., n] and contiguous e8m0 scales [lead..., blocks(n)].
bool codes(const at::Tensor& q, const at::Tensor& s, bool weight, int device) {
  if (!plain(q, device) || !plain(s, device) || q.scalar_type() != at::kFloat8_e4m3fn ||
      s.scalar_type() != at::kFloat8_e8m0fnu || q.dim() != s.dim() || q.dim() < (weight ? 2 : 1) || q.numel() == 0 ||
      !s.is_contiguous())
    return false;
  const int64_t d = q.dim();
  if (weight) return d == 2 && s.size(0) == blocks(q.size(0)) && s.size(1) == blocks(q.size(1));
  for (int64_t i = 0; i + 1 < d; ++i)
    if (q.size(i) != s.size(i)) return false;
  return s.size(d - 1) == blocks(q.size(d - 1));
}

c10::SmallVector<int64_t, 6> with_last(const at::Tensor& t, int64_t last) {
  c10::SmallVector<int64_t, 6> shape(t.sizes().begin(), t.sizes().end());
  shape.back() = last;
  return shape;
}

// Room for codes whose rows start on 16-byte boundaries.
at::Tensor new_codes(const at::Tensor& like) {
  const int64_t n = like.size(-1), pitch = (n + 15) / 16 * 16;
  if (pitch == n) return empty(like.sizes(), at::kFloat8_e4m3fn);
  return empty(with_last(like, pitch), at::kFloat8_e4m3fn).narrow(-1, 0, n);
}
int64_t code_pitch(const at::Tensor& q) { return (q.size(-1) + 15) / 16 * 16; }

PyObject* tuple_of(at::Tensor&& a, at::Tensor&& b) {
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(a)));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(b)));
  return t;
}

// x
PyObject* quant_rows_f8(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    const at::Tensor* x = n_args == 1 && quant_rows_f8_fn ? tensor(args[0]) : nullptr;
    const int device = c10::cuda::current_device();
    if (!x || !numbers(*x, device)) Py_RETURN_NONE;
    const int64_t n = x->size(-1), ld = row_stride(*x);
    if (ld < 0) Py_RETURN_NONE;
    at::Tensor q = new_codes(*x), s = empty(with_last(*x, blocks(n)), at::kFloat8_e8m0fnu);
    if (quant_rows_f8_fn(x->data_ptr(), code(x->scalar_type()), x->numel() / n, n, ld,
                         static_cast<uint8_t*>(q.data_ptr()), code_pitch(q), static_cast<uint8_t*>(s.data_ptr()),
                         stream(device)))
      Py_RETURN_NONE;
    return tuple_of(std::move(q), std::move(s));
  });
}

// w
PyObject* quant_weight_f8(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    const at::Tensor* w = n_args == 1 && quant_weight_f8_fn ? tensor(args[0]) : nullptr;
    const int device = c10::cuda::current_device();
    if (!w || !numbers(*w, device) || w->dim() != 2) Py_RETURN_NONE;
    const int64_t n = w->size(0), k = w->size(1), ld = row_stride(*w);
    if (ld < 0) Py_RETURN_NONE;
    at::Tensor q = new_codes(*w), s = empty({blocks(n), blocks(k)}, at::kFloat8_e8m0fnu);
    if (quant_weight_f8_fn(w->data_ptr(), code(w->scalar_type()), n, k, ld, static_cast<uint8_t*>(q.data_ptr()),
                           code_pitch(q), static_cast<uint8_t*>(s.data_ptr()), stream(device)))
      Py_RETURN_NONE;
    return tuple_of(std::move(q), std::move(s));
  });
}

// The weight and bias of a product over k columns: checked, the weight's row stride and the bias's pointer.
bool f8_weight(PyObject* qo, PyObject* so, PyObject* bo, int64_t k, int device, const at::Tensor*& q,
               const at::Tensor*& s, const at::Tensor*& bias, int64_t& ld) {
  q = tensor(qo);
  s = tensor(so);
  bias = bo == Py_None ? nullptr : tensor(bo);
  if (!q || !s || (!bias && bo != Py_None) || !codes(*q, *s, true, device) || q->size(1) != k) return false;
  if (bias && (!plain(*bias, device) || bias->dim() != 1 || bias->size(0) != q->size(0) || !bias->is_contiguous() ||
               code(bias->scalar_type()) < 0))
    return false;
  ld = row_stride(*q);
  return ld > 0;
}
at::Tensor workspace(int64_t bytes) {
  return bytes > 0 ? empty({bytes}, at::kByte) : at::Tensor();
}

// a, a_scale, b, b_scale, bias or None, output dtype
PyObject* gemm_f8(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 6 || !gemm_f8_fn || !THPDtype_Check(args[5])) Py_RETURN_NONE;
    const at::Tensor *a = tensor(args[0]), *a_s = tensor(args[1]), *b, *b_s, *bias;
    const at::ScalarType t = reinterpret_cast<THPDtype*>(args[5])->scalar_type;
    const int device = c10::cuda::current_device();
    int64_t ld_b;
    if (!a || !a_s || code(t) < 0 || !codes(*a, *a_s, false, device)) Py_RETURN_NONE;
    const int64_t k = a->size(-1), m = a->numel() / k, ld_a = row_stride(*a);
    if (ld_a < 0 || !f8_weight(args[2], args[3], args[4], k, device, b, b_s, bias, ld_b)) Py_RETURN_NONE;
    const int64_t n = b->size(0);
    const auto *ap = static_cast<const uint8_t*>(a->data_ptr()), *bp = static_cast<const uint8_t*>(b->data_ptr());
    at::Tensor out = empty(with_last(*a, n), t);
    const int64_t bytes = gemm_f8_bytes_fn(ap, m, k, ld_a, bp, n, ld_b);
    at::Tensor ws = workspace(bytes);
    if (gemm_f8_fn(ap, static_cast<const uint8_t*>(a_s->data_ptr()), m, k, ld_a, bp,
                   static_cast<const uint8_t*>(b_s->data_ptr()), n, ld_b, bias ? bias->data_ptr() : nullptr,
                   bias ? code(bias->scalar_type()) : 0, out.data_ptr(), code(t), n, bytes ? ws.data_ptr() : nullptr,
                   bytes, stream(device)))
      Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// x, b, b_scale, bias or None
PyObject* linear_f8(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    const at::Tensor *x = n_args == 4 && linear_f8_fn ? tensor(args[0]) : nullptr, *b, *b_s, *bias;
    const int device = c10::cuda::current_device();
    if (!x || !numbers(*x, device)) Py_RETURN_NONE;
    const int64_t k = x->size(-1), m = x->numel() / k, ld = row_stride(*x);
    int64_t ld_b;
    if (ld < 0 || !f8_weight(args[1], args[2], args[3], k, device, b, b_s, bias, ld_b)) Py_RETURN_NONE;
    const int64_t n = b->size(0);
    const auto* bp = static_cast<const uint8_t*>(b->data_ptr());
    at::Tensor out = empty(with_last(*x, n), x->scalar_type());
    const int64_t bytes = linear_f8_bytes_fn(m, k, bp, n, ld_b);
    at::Tensor ws = workspace(bytes);
    const int dt = code(x->scalar_type());
    if (linear_f8_fn(x->data_ptr(), dt, m, k, ld, bp, static_cast<const uint8_t*>(b_s->data_ptr()), n, ld_b,
                     bias ? bias->data_ptr() : nullptr, bias ? code(bias->scalar_type()) : 0, out.data_ptr(), dt, n,
                     bytes ? ws.data_ptr() : nullptr, bytes, stream(device)))
      Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// The codes and scales of a producer's output mode.
bool new_output(const at::Tensor& like, int64_t mode, at::Tensor& q, at::Tensor& s) {
  const int64_t n = like.size(-1);
  if (mode == QI8_Q_FP8) {
    q = new_codes(like);
    s = empty(with_last(like, blocks(n)), at::kFloat8_e8m0fnu);
    return true;
  }
  if (mode != QI8_Q_TOKEN && (mode != QI8_Q_BLOCK || n % F8_BLOCK)) return false;
  q = empty(like.sizes(), at::kChar);
  s = empty(with_last(like, mode == QI8_Q_TOKEN ? 1 : n / F8_BLOCK), at::kFloat);
  return true;
}

// x, weight or None, eps, residual or None, mode
PyObject* rms_norm_quant(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 5 || !norm_fn || !PyFloat_CheckExact(args[2])) Py_RETURN_NONE;
    const at::Tensor* x = tensor(args[0]);
    const at::Tensor* w = args[1] == Py_None ? nullptr : tensor(args[1]);
    const at::Tensor* r = args[3] == Py_None ? nullptr : tensor(args[3]);
    const int device = c10::cuda::current_device();
    if (!x || (!w && args[1] != Py_None) || (!r && args[3] != Py_None) || !numbers(*x, device)) Py_RETURN_NONE;
    const int64_t n = x->size(-1), ld = row_stride(*x), mode = integer(args[4]);
    if (ld < 0 || (w && (!plain(*w, device) || w->dim() != 1 || w->size(0) != n || !w->is_contiguous() ||
                         code(w->scalar_type()) < 0)))
      Py_RETURN_NONE;
    if (r && (!plain(*r, device) || r->scalar_type() != x->scalar_type() || r->sizes() != x->sizes())) Py_RETURN_NONE;
    const int64_t ld_r = r ? row_stride(*r) : 0;
    at::Tensor q, s, h;
    if (ld_r < 0 || !new_output(*x, mode, q, s)) Py_RETURN_NONE;
    if (r) h = empty(x->sizes(), x->scalar_type());
    if (norm_fn(x->data_ptr(), code(x->scalar_type()), x->numel() / n, n, ld, r ? r->data_ptr() : nullptr, ld_r,
                w ? w->data_ptr() : nullptr, w ? code(w->scalar_type()) : 0, PyFloat_AS_DOUBLE(args[2]), (int)mode,
                q.data_ptr(), mode == QI8_Q_FP8 ? code_pitch(q) : n, s.data_ptr(), r ? h.data_ptr() : nullptr, n,
                stream(device)))
      Py_RETURN_NONE;
    if (!r) return tuple_of(std::move(q), std::move(s));
    PyObject* t = PyTuple_New(3);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(q)));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(s)));
    PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(std::move(h)));
    return t;
  });
}

// gate, up, activation code, mode
PyObject* gated_quant(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 4 || !gated_fn) Py_RETURN_NONE;
    const at::Tensor *g = tensor(args[0]), *u = tensor(args[1]);
    const int device = c10::cuda::current_device();
    if (!g || !u || !numbers(*g, device) || !plain(*u, device) || u->scalar_type() != g->scalar_type() ||
        u->sizes() != g->sizes())
      Py_RETURN_NONE;
    const int64_t n = g->size(-1), ld_g = row_stride(*g), ld_u = row_stride(*u);
    const int64_t act = integer(args[2]), mode = integer(args[3]);
    at::Tensor q, s;
    if (ld_g < 0 || ld_u < 0 || act < 0 || act > QI8_ACT_GELU_TANH || !new_output(*g, mode, q, s)) Py_RETURN_NONE;
    if (gated_fn(g->data_ptr(), ld_g, u->data_ptr(), ld_u, code(g->scalar_type()), g->numel() / n, n, (int)act, (int)mode,
                 q.data_ptr(), mode == QI8_Q_FP8 ? code_pitch(q) : n, s.data_ptr(), stream(device)))
      Py_RETURN_NONE;
    return tuple_of(std::move(q), std::move(s));
  });
}

// q int8, scale, kind, block, output dtype: the int8 outputs of the two above, read back
PyObject* dequant(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 5 || !dequant8_fn || !THPDtype_Check(args[4])) Py_RETURN_NONE;
    const at::Tensor *q = tensor(args[0]), *s = tensor(args[1]);
    const at::ScalarType t = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
    const int device = c10::cuda::current_device();
    const int64_t kind = integer(args[2]), block = integer(args[3]);
    if (!q || !s || code(t) < 0 || !plain(*q, device) || !plain(*s, device) || q->scalar_type() != at::kChar ||
        s->scalar_type() != at::kFloat || q->dim() < 1 || q->numel() == 0 || !q->is_contiguous() || !s->is_contiguous())
      Py_RETURN_NONE;
    const int64_t n = q->size(-1), rows = q->numel() / n;
    // as many scales as the kernel reads
    if (kind == QI8_S_SCALAR ? s->numel() < 1
        : kind == QI8_S_ROW ? s->numel() != rows
                            : kind != QI8_S_ROW_KBLOCK || block <= 0 || n % block || s->numel() != rows * (n / block))
      Py_RETURN_NONE;
    at::Tensor out = empty(q->sizes(), t);
    if (dequant8_fn(static_cast<const int8_t*>(q->data_ptr()), rows, n, static_cast<const float*>(s->data_ptr()),
                    (int)kind, (int)block, out.data_ptr(), code(t), stream(device)))
      Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// addresses of the entry points, in the order of the assignments below
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  constexpr int N = 14;
  void* p[N];
  if (n_args != N) {
    PyErr_SetString(PyExc_TypeError, "bind takes fourteen addresses");
    return nullptr;
  }
  for (int i = 0; i < N; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  int i = 0;
  auto set = [&](auto& fn) { fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(p[i++]); };
  set(quant_fn);
  set(dequant_fn);
  set(gemm_fn);
  set(moe_fn);
  set(moe_bytes_fn);
  set(quant_rows_f8_fn);
  set(quant_weight_f8_fn);
  set(gemm_f8_bytes_fn);
  set(gemm_f8_fn);
  set(linear_f8_bytes_fn);
  set(linear_f8_fn);
  set(norm_fn);
  set(gated_fn);
  set(dequant8_fn);
  Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(gemm_w4), FAST(quant_weight_i4), FAST(dequant_i4), FAST(moe_w4), FAST(quant_rows_f8),
                         FAST(quant_weight_f8), FAST(gemm_f8), FAST(linear_f8), FAST(rms_norm_quant), FAST(gated_quant),
                         FAST(dequant),
                         FAST(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__call() { return PyModule_Create(&module_def); }
