// htr_amd._fast: the host side of a packed linear, of a routed-expert layer and of the operators around them on torch tensors, in C++.
//
// A decode launch takes the GPU 6 microseconds and took the interpreter 16 (a dozen attribute reads, shape checks, two
// dictionary look-ups, a 19-argument foreign call), so small calls ran at the interpreter's pace; collecting the 512
// tensors of a 64-expert layer took it half a millisecond.  Here the same checks read the tensors' fields directly.  Every
// function returns None where something is not as expected: the caller's Python path then handles the call, or says
// what is wrong with it.  Only torch's C++ interface is used; the kernels stay behind the C ABI of libhtr_gfx950.so, whose
// entry points bind() takes as addresses.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <chrono>
#include <cstdint>
#include <cstring>
#include <vector>
#include "../../include/htr_gfx950.h"

namespace {

// the library's entry points, with the types that its header declares
decltype(&htr_linear) f_linear = nullptr;
decltype(&htr_stream_capture_id) f_capture = nullptr;
decltype(&htr_moe_scratch_bytes) f_moe_bytes = nullptr;
decltype(&htr_moe_experts) f_moe = nullptr;
decltype(&htr_linear_route) f_route = nullptr;
decltype(&htr_dequant_w) f_dequant = nullptr;
decltype(&htr_rms_norm) f_norm = nullptr;
decltype(&htr_quantize_e4m3) f_quantize = nullptr;
decltype(&htr_product) f_product = nullptr;
decltype(&htr_product_rounds) f_rounds = nullptr;
decltype(&htr_moe_stacked_scratch_bytes) f_stacked_bytes = nullptr;
decltype(&htr_moe_stacked) f_stacked = nullptr;

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: return -1;
  }
}

struct Owned {      // one reference, given back at the end of the scope
  PyObject* p;
  ~Owned() { Py_XDECREF(p); }
};

const at::Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// Memory of its own (not the wrapper of a function transform such as torch.func.grad)
bool raw_ok(const at::Tensor& t) { return t.has_storage(); }
// Whether torch follows derivatives through t now, backward or forward
bool differentiable(const at::Tensor& t) { return (c10::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined(); }

struct Shape { int64_t m = 0, n = 0, K = 0; };

// One HTR-W1 tensor set (qweight int32 [m/16, n/16, 8K], scales float16 [m], su uint8 [n/8], sv uint8 [m/8], all contiguous on
// device `dev`): its shape, or false.
bool weight_ok(const at::Tensor& qw, const at::Tensor& sc, const at::Tensor& su, const at::Tensor& sv, c10::Device dev, Shape& s) {
  if (qw.dim() != 3 || qw.scalar_type() != at::kInt || sc.scalar_type() != at::kHalf || su.scalar_type() != at::kByte || sv.scalar_type() != at::kByte)
    return false;
  const int64_t W = qw.size(2);
  s.m = qw.size(0) * 16; s.n = qw.size(1) * 16; s.K = W / 8;
  if (W % 8 || s.K < 2 || s.K > 8 || s.m % 128 || s.n % 128 || s.m == 0 || s.n == 0) return false;
  if (sc.numel() != s.m || su.numel() * 8 != s.n || sv.numel() * 8 != s.m) return false;
  for (const at::Tensor* t : {&qw, &sc, &su, &sv})
    if (t->device() != dev || !t->is_contiguous()) return false;
  return true;
}

// linear(x, qweight, scales, su, sv, bias, workspace address, its bytes, address of its failure word (0: none), stream, rows)
// -> tensor or None; None also while the stream is being captured (a capture has workspaces of its own), after a launch
// on the workspace gave up, and for more activation rows than `rows` (128 if not given).  Beyond 128 rows the call goes where
// htr_linear_route says, as in ops._linear_impl: one launch, or the weight dequantized and multiplied by torch, for which the workspace may
// be missing (address 0).
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs < 10 || nargs > 11 || f_linear == nullptr || !THPVariable_CheckExact(args[0])) Py_RETURN_NONE;
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i) t[i] = args[i] == Py_None ? nullptr : tensor_of(args[i]);
  for (int i = 0; i < 5; ++i) if (t[i] == nullptr) Py_RETURN_NONE;
  if (args[5] != Py_None && t[5] == nullptr) Py_RETURN_NONE;
  const at::Tensor& x = *t[0];
  Shape s;
  const int code = dtype_code(x.scalar_type());
  if (code < 0 || !x.is_cuda() || x.dim() < 1 || !x.is_contiguous() || !weight_ok(*t[1], *t[2], *t[3], *t[4], x.device(), s)) Py_RETURN_NONE;
  if (x.size(-1) != s.n) Py_RETURN_NONE;
  const int64_t M = x.numel() / s.n;
  if (t[5] != nullptr && (t[5]->scalar_type() != x.scalar_type() || t[5]->numel() != s.m || t[5]->device() != x.device() || !t[5]->is_contiguous()))
    Py_RETURN_NONE;
  void* ws = PyLong_AsVoidPtr(args[6]);
  const size_t bytes = PyLong_AsSize_t(args[7]);
  const volatile int* failed = (const volatile int*)PyLong_AsVoidPtr(args[8]);
  void* stream = PyLong_AsVoidPtr(args[9]);
  const long rows = nargs > 10 && f_route != nullptr && f_dequant != nullptr ? PyLong_AsLong(args[10]) : HTR_MAX_ROWS_PER_TILE;
  if (PyErr_Occurred()) return nullptr;
  if (M < 1 || M > rows) Py_RETURN_NONE;
  int route = 0;
  if (M > HTR_MAX_ROWS_PER_TILE) {
    // torch's product can be differentiated and transformed, a launch on raw pointers cannot: the general path tells them apart
    if (M > HTR_MAX_BATCH || !raw_ok(x) || differentiable(x) || (t[5] != nullptr && (!raw_ok(*t[5]) || differentiable(*t[5])))) Py_RETURN_NONE;
    route = f_route((int)s.m, (int)s.n, (int)s.K, (int)M, code, 1);
    if (route < HTR_ROUTE_DEQUANTIZE) Py_RETURN_NONE;
  }
  if ((failed != nullptr && *failed != 0) || f_capture(stream) != 0) Py_RETURN_NONE;
  at::Tensor y;
  int rc;
  {
    // other threads run meanwhile: a launch waits where the stream's queue is full.  The caller's frame holds the tensors.
    pybind11::gil_scoped_release no_lock;
    c10::DeviceGuard guard(x.device());
    at::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = s.m;
    if (route == HTR_ROUTE_DEQUANTIZE) {
      at::Tensor w = at::empty({s.m, s.n}, x.options().dtype(at::kBFloat16));
      rc = f_dequant(t[1]->const_data_ptr(), t[2]->const_data_ptr(), t[3]->const_data_ptr(), t[4]->const_data_ptr(), w.mutable_data_ptr(),
                     (int)s.m, (int)s.n, (int)s.K, stream);
      if (rc == HTR_OK) {
        // rows and columns only: with more dimensions, and an outer one of size 1 whose stride is not the inner ones' product (a prompt cut
        // from a longer buffer), torch takes a batched product with a transposed view of the weight
        y = at::linear(x.view({M, s.n}), code == 0 ? w : w.to(x.scalar_type()),
                       t[5] == nullptr ? std::optional<at::Tensor>() : std::optional<at::Tensor>(*t[5])).view(shape);
        if (y.scalar_type() != x.scalar_type()) y = y.to(x.scalar_type());      // autocast
      }
    } else {
      y = at::empty(shape, x.options());
      rc = f_linear(t[1]->const_data_ptr(), t[2]->const_data_ptr(), t[3]->const_data_ptr(), t[4]->const_data_ptr(), x.const_data_ptr(),
                  t[5] == nullptr ? nullptr : t[5]->const_data_ptr(), y.mutable_data_ptr(), (int)s.m, (int)s.n, (int)s.K, (int)M, code, code, route,
                  ws, bytes, stream);
    }
  }
  if (rc != HTR_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// The tensor addresses of one tuple of HTR-W1 tuples into every eighth slot group of `ptrs`; false where one is not like the first.
// The tensors of an expert given as a list, which another thread may change, go to `keep`.
bool collect(PyObject* experts, int offset, c10::Device dev, Shape& shape, std::vector<const void*>& ptrs, std::vector<at::Tensor>& keep) {
  const Py_ssize_t E = PyTuple_GET_SIZE(experts);
  for (Py_ssize_t e = 0; e < E; ++e) {
    PyObject* tup = PyTuple_GET_ITEM(experts, e);
    if (!(PyTuple_Check(tup) || PyList_Check(tup)) || PySequence_Fast_GET_SIZE(tup) != 4) return false;
    const at::Tensor* t[4];
    for (int k = 0; k < 4; ++k) { t[k] = tensor_of(PySequence_Fast_GET_ITEM(tup, k)); if (t[k] == nullptr) return false; }
    Shape s;
    if (!weight_ok(*t[0], *t[1], *t[2], *t[3], dev, s)) return false;
    if (e == 0) shape = s;
    else if (s.m != shape.m || s.n != shape.n || s.K != shape.K) return false;
    for (int k = 0; k < 4; ++k) ptrs[8 * e + offset + k] = t[k]->const_data_ptr();
    if (PyList_Check(tup)) for (int k = 0; k < 4; ++k) keep.push_back(*t[k]);
  }
  return true;
}

// moe(x, ids, weights, gate_up, down, host word address (0: none), ticket, stream) -> float32 [tokens, hidden], None, or the status of
// a launch that the runtime refused
PyObject* moe(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 8 || f_moe == nullptr) Py_RETURN_NONE;
  const at::Tensor *xt = tensor_of(args[0]), *it = tensor_of(args[1]), *wt = tensor_of(args[2]);
  if (xt == nullptr || it == nullptr || wt == nullptr || !xt->is_cuda() || xt->dim() != 2 || it->dim() != 2 || wt->dim() != 2) Py_RETURN_NONE;
  const int64_t T = xt->size(0), H = xt->size(1), top = it->size(1);
  const int code = dtype_code(xt->scalar_type());
  if (code < 0 || it->size(0) != T || wt->size(0) != T || wt->size(1) != top || it->device() != xt->device() || wt->device() != xt->device()) Py_RETURN_NONE;
  if ((it->scalar_type() != at::kLong && it->scalar_type() != at::kInt) || !wt->is_floating_point()) Py_RETURN_NONE;
  // the result is differentiable in the routing weights only where torch adds it up: not behind a raw pointer
  if (!raw_ok(*xt) || !raw_ok(*it) || !raw_ok(*wt) || differentiable(*wt)) Py_RETURN_NONE;
  // plain lists and tuples only: another kind of collection may load an expert when it is asked for, and is asked for the chosen ones
  for (int i = 3; i < 5; ++i) if (!PyTuple_CheckExact(args[i]) && !PyList_CheckExact(args[i])) Py_RETURN_NONE;
  Owned gu{PySequence_Tuple(args[3])}, dn{PySequence_Tuple(args[4])};      // own references to the experts: no other thread can drop one
  if (gu.p == nullptr || dn.p == nullptr) return nullptr;
  const Py_ssize_t E = PyTuple_GET_SIZE(gu.p);
  if (E < 1 || PyTuple_GET_SIZE(dn.p) != E) Py_RETURN_NONE;
  std::vector<const void*> ptrs((size_t)E * 8);
  std::vector<at::Tensor> keep;
  Shape s1, s2;
  if (!collect(gu.p, 0, xt->device(), s1, ptrs, keep) || !collect(dn.p, 4, xt->device(), s2, ptrs, keep)) Py_RETURN_NONE;
  const int64_t F = s1.m / 2;
  if (s1.n != H || s2.m != H || s2.n != F || T < 1 || top < 1 || T > (1 << 24) || E > (1 << 20)) Py_RETURN_NONE;
  unsigned int* word = (unsigned int*)PyLong_AsVoidPtr(args[5]);
  const unsigned int ticket = (unsigned int)PyLong_AsUnsignedLong(args[6]);
  void* stream = PyLong_AsVoidPtr(args[7]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor y;
  int rc;
  {
    pybind11::gil_scoped_release no_lock;      // as in linear()
    c10::DeviceGuard guard(xt->device());
    at::Tensor x = xt->contiguous(), ids = it->contiguous(), w = wt->to(at::kFloat).contiguous();
    if ((uintptr_t)x.const_data_ptr() & 15) x = x.clone();
    const size_t need = f_moe_bytes((int)T, (int)top, (int)E, (int)H, (int)F);
    if (need == 0) {
      rc = HTR_ERR_SHAPE;
    } else {
      at::Tensor scratch = at::empty({(int64_t)need}, x.options().dtype(at::kByte));
      y = at::empty({T, H}, x.options().dtype(at::kFloat));
      rc = f_moe(x.const_data_ptr(), code, ids.const_data_ptr(), ids.scalar_type() == at::kLong ? 1 : 0, (const float*)w.const_data_ptr(), (int)T,
                 (int)top, ptrs.data(), (int)E, (int)H, (int)F, (int)s1.K, (int)s2.K, (float*)y.mutable_data_ptr(), scratch.mutable_data_ptr(),
                 need, word, ticket, stream);
    }
  }
  if (rc == HTR_ERR_LAUNCH) return PyLong_FromLong(rc);      // part of the layer may be queued: an error, not another way to run it
  if (rc != HTR_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// wait_word(address, ticket, seconds) -> the word's low bit once its upper bits are the ticket, or None after that time
PyObject* wait_word(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 3) Py_RETURN_NONE;
  const volatile unsigned int* word = (const volatile unsigned int*)PyLong_AsVoidPtr(args[0]);
  const unsigned int ticket = (unsigned int)PyLong_AsUnsignedLong(args[1]) & 0x7FFFFFFFu;
  const double seconds = PyFloat_AsDouble(args[2]);
  if (PyErr_Occurred()) return nullptr;
  unsigned int v = 0;
  bool done = false;
  Py_BEGIN_ALLOW_THREADS
  const auto until = std::chrono::steady_clock::now() + std::chrono::duration<double>(seconds);
  for (;;) {
    for (int i = 0; i < 256 && !done; ++i) { v = *word; done = (v >> 1) == ticket; __builtin_ia32_pause(); }
    if (done || std::chrono::steady_clock::now() > until) break;
  }
  Py_END_ALLOW_THREADS
  if (!done) Py_RETURN_NONE;
  return PyLong_FromLong((long)(v & 1u));
  END_HANDLE_TH_ERRORS
}

// ---- the operators around the packed linears (htr_amd/unpacked.py): the common case of each, None where the Python path is to handle the call or refuse it
bool float_of(const at::Tensor& t) { return dtype_code(t.scalar_type()) >= 0; }
bool half_of(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
bool aligned16(const at::Tensor& t) { return ((uintptr_t)t.const_data_ptr() & 15) == 0; }
// consecutive memory on `dev` from a 16-byte boundary on, that torch does not follow
bool plain(const at::Tensor& t, c10::Device dev) { return t.device() == dev && raw_ok(t) && t.is_contiguous() && aligned16(t) && !differentiable(t); }
at::ScalarType type_of(long code) { return code == 0 ? at::kBFloat16 : code == 1 ? at::kHalf : at::kFloat; }
// dims of 8-bit rows' scales (rows = true) or matrices' for values q
bool scales_ok(const at::Tensor& q, const at::Tensor& s, bool rows) {
  if (s.scalar_type() != at::kFloat || s.dim() != q.dim() || q.dim() < (rows ? 1 : 2) || q.size(-1) % 128 || s.size(-1) != q.size(-1) / 128) return false;
  for (int64_t k = 0; k + 1 < q.dim(); ++k) {
    const bool m = !rows && k + 2 == q.dim();
    if (s.size(k) != (m ? (q.size(k) + 127) / 128 : q.size(k))) return false;
  }
  return true;
}
// x as 8-bit rows; a tensor of floats is rounded.  False: not as expected; rc: what the launch returned
bool rows8(const at::Tensor& x, const at::Tensor* s, c10::Device dev, void* stream, at::Tensor& q, at::Tensor& qs, int& rc) {
  if (s != nullptr) {
    if (x.scalar_type() != at::kFloat8_e4m3fn || !scales_ok(x, *s, true) || !plain(*s, dev)) return false;
    q = x; qs = *s;
    return true;
  }
  const int64_t n = x.size(-1);
  if (!float_of(x) || n % 128) return false;
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  q = at::empty(shape, x.options().dtype(at::kFloat8_e4m3fn));
  shape.back() = n / 128;
  qs = at::empty(shape, x.options().dtype(at::kFloat));
  rc = f_quantize(x.const_data_ptr(), n, x.numel() / n, (int)n, dtype_code(x.scalar_type()), q.mutable_data_ptr(), qs.mutable_data_ptr(), stream);
  return rc == HTR_OK;
}
// optional tensor argument: false where it is neither None nor a tensor
bool optional(PyObject* o, const at::Tensor*& t) { t = o == Py_None ? nullptr : tensor_of(o); return o == Py_None || t != nullptr; }

// rms_norm(x, weight, eps, residual or None, quantize, stream)
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor *x, *w, *r;
  if (nargs != 6 || f_norm == nullptr || !THPVariable_CheckExact(args[0]) || !optional(args[1], w) || w == nullptr || !optional(args[3], r)) Py_RETURN_NONE;
  x = tensor_of(args[0]);
  const double eps = PyFloat_AsDouble(args[2]);
  const int quantize = PyObject_IsTrue(args[4]);
  void* stream = PyLong_AsVoidPtr(args[5]);
  if (PyErr_Occurred()) return nullptr;
  if (!x->is_cuda() || x->dim() < 1 || !float_of(*x) || x->numel() == 0) Py_RETURN_NONE;
  const c10::Device dev = x->device();
  const int64_t n = x->size(-1), rows = x->numel() / n;
  if (!plain(*x, dev) || !plain(*w, dev) || w->scalar_type() != x->scalar_type() || w->dim() != 1 || w->size(0) != n || (quantize && n % 128) || n > (1 << 30)) Py_RETURN_NONE;
  if (r != nullptr && (!plain(*r, dev) || r->scalar_type() != x->scalar_type() || r->sizes() != x->sizes())) Py_RETURN_NONE;
  at::Tensor y, s, t;
  int rc;
  {
    pybind11::gil_scoped_release no_lock;      // as in linear()
    c10::DeviceGuard guard(dev);
    y = at::empty(x->sizes(), quantize ? x->options().dtype(at::kFloat8_e4m3fn) : x->options());
    if (quantize) {
      at::DimVector shape(x->sizes().begin(), x->sizes().end());
      shape.back() = n / 128;
      s = at::empty(shape, x->options().dtype(at::kFloat));
    }
    if (r != nullptr) t = at::empty(x->sizes(), x->options());
    rc = f_norm(x->const_data_ptr(), n, r == nullptr ? nullptr : r->const_data_ptr(), n, w->const_data_ptr(), rows, (int)n, eps, dtype_code(x->scalar_type()),
                y.mutable_data_ptr(), quantize ? s.mutable_data_ptr() : nullptr, r == nullptr ? nullptr : t.mutable_data_ptr(), stream);
  }
  if (rc != HTR_OK) Py_RETURN_NONE;
  PyObject* out = THPVariable_Wrap(std::move(y));
  if (quantize) out = PyTuple_Pack(2, Owned{out}.p, Owned{THPVariable_Wrap(std::move(s))}.p);
  if (r != nullptr) out = PyTuple_Pack(2, Owned{out}.p, Owned{THPVariable_Wrap(std::move(t))}.p);
  return out;
  END_HANDLE_TH_ERRORS
}

// product(x, its scales or None, weight, its scales or None, bias or None, ends or None, the result's type code, stream): linear_fp8 where ends is None,
// otherwise grouped_mm
PyObject* product(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor *x, *xs, *w, *ws, *bias, *ends;
  if (nargs != 8 || f_product == nullptr || !THPVariable_CheckExact(args[0]) || !optional(args[1], xs) || !optional(args[2], w) || w == nullptr ||
      !optional(args[3], ws) || !optional(args[4], bias) || !optional(args[5], ends))
    Py_RETURN_NONE;
  x = tensor_of(args[0]);
  const long code = PyLong_AsLong(args[6]);
  void* stream = PyLong_AsVoidPtr(args[7]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t dims = ends == nullptr ? 2 : 3;
  if (code < 0 || code > 2 || !x->is_cuda() || x->dim() < 1 || x->numel() == 0 || w->dim() != dims || w->numel() == 0) Py_RETURN_NONE;
  const c10::Device dev = x->device();
  const int64_t n = w->size(-1), m = w->size(-2), experts = ends == nullptr ? 1 : w->size(0);
  const bool eight = ws != nullptr;
  if (x->size(-1) != n || !plain(*x, dev) || !plain(*w, dev) || m > (1 << 30) || n > (1 << 30) || experts > (1 << 30)) Py_RETURN_NONE;
  if (ends != nullptr && (x->dim() != 2 || ends->scalar_type() != at::kInt || ends->dim() != 1 || ends->size(0) != experts || ends->device() != dev || !ends->is_contiguous()))
    Py_RETURN_NONE;
  if (eight ? w->scalar_type() != at::kFloat8_e4m3fn || !scales_ok(*w, *ws, false) || ws->device() != dev || !ws->is_contiguous() || differentiable(*ws)
            : ends == nullptr || xs != nullptr || !half_of(*w) || x->scalar_type() != w->scalar_type() || n % 8)
    Py_RETURN_NONE;
  if (bias != nullptr && (ends != nullptr || bias->scalar_type() != type_of(code) || bias->dim() != 1 || bias->size(0) != m || bias->device() != dev ||
                          !bias->is_contiguous() || !raw_ok(*bias) || differentiable(*bias)))
    Py_RETURN_NONE;
  at::Tensor y, q, qs;
  int rc = HTR_OK;
  {
    pybind11::gil_scoped_release no_lock;      // as in linear()
    c10::DeviceGuard guard(dev);
    // few 16-bit rows are rounded by the product itself
    const bool as_is = !eight || (xs == nullptr && half_of(*x) && f_rounds(x->numel() / n, (int)experts, ends != nullptr));
    if (as_is) q = *x;
    if (!as_is && !rows8(*x, xs, dev, stream, q, qs, rc)) {
      rc = HTR_ERR_SIZE;
    } else {
      at::DimVector shape(x->sizes().begin(), x->sizes().end());
      shape.back() = m;
      y = at::empty(shape, x->options().dtype(type_of(code)));
      rc = f_product(q.const_data_ptr(), as_is ? dtype_code(x->scalar_type()) : HTR_E4M3, as_is ? nullptr : qs.const_data_ptr(), w->const_data_ptr(), eight ? ws->const_data_ptr() : nullptr,
                     bias == nullptr ? nullptr : bias->const_data_ptr(), ends == nullptr ? nullptr : (const int32_t*)ends->const_data_ptr(), y.mutable_data_ptr(),
                     x->numel() / n, (int)m, (int)n, (int)experts, eight ? HTR_E4M3 : dtype_code(w->scalar_type()), (int)code, stream);
    }
  }
  if (rc != HTR_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// moe_stacked(x, ids, weights, gate_up, its scales or None, down, its scales or None, stream)
PyObject* moe_stacked(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor* t[7];
  if (nargs != 8 || f_stacked == nullptr || !THPVariable_CheckExact(args[0])) Py_RETURN_NONE;
  for (int i = 0; i < 7; ++i) if (!optional(args[i], t[i]) || (t[i] == nullptr && i != 4 && i != 6)) Py_RETURN_NONE;
  void* stream = PyLong_AsVoidPtr(args[7]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor &x = *t[0], &ids = *t[1], &wt = *t[2], &gu = *t[3], &dn = *t[5];
  const bool eight = t[4] != nullptr;
  if (!x.is_cuda() || x.dim() != 2 || !half_of(x) || x.numel() == 0 || ids.dim() != 2 || ids.numel() == 0 || gu.dim() != 3 || dn.dim() != 3 || eight != (t[6] != nullptr))
    Py_RETURN_NONE;
  const c10::Device dev = x.device();
  const int64_t T = x.size(0), H = x.size(1), top = ids.size(1), E = dn.size(0), F = dn.size(2);
  if (!plain(x, dev) || !plain(gu, dev) || !plain(dn, dev) || dn.size(1) != H || gu.size(0) != E || gu.size(1) != 2 * F || gu.size(2) != H || F < 1 || E < 1) Py_RETURN_NONE;
  if (E > (1 << 20) || F > (1 << 28) || H > (1 << 28) || top > (1 << 20)) Py_RETURN_NONE;
  if (eight) {
    for (int i = 3; i < 7; i += 2)
      if (t[i]->scalar_type() != at::kFloat8_e4m3fn || !scales_ok(*t[i], *t[i + 1], false) || t[i + 1]->device() != dev || !t[i + 1]->is_contiguous() || differentiable(*t[i + 1]))
        Py_RETURN_NONE;
  } else if (gu.scalar_type() != x.scalar_type() || dn.scalar_type() != x.scalar_type()) {
    Py_RETURN_NONE;
  }
  if (ids.size(0) != T || wt.dim() != 2 || wt.size(0) != T || wt.size(1) != top || ids.device() != dev || !ids.is_contiguous() || !raw_ok(ids) ||
      (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt) || wt.device() != dev || wt.scalar_type() != at::kFloat || !wt.is_contiguous() || !raw_ok(wt) ||
      differentiable(wt))
    Py_RETURN_NONE;
  const int dtype = dtype_code(x.scalar_type()), type = eight ? HTR_E4M3 : dtype;
  const size_t need = f_stacked_bytes(T, (int)top, (int)E, (int)H, (int)F, type);
  if (need == 0) Py_RETURN_NONE;
  at::Tensor y;
  int rc;
  {
    pybind11::gil_scoped_release no_lock;      // as in linear()
    c10::DeviceGuard guard(dev);
    at::Tensor scratch = at::empty({(int64_t)need}, x.options().dtype(at::kByte));
    y = at::empty({T, H}, x.options());
    rc = f_stacked(x.const_data_ptr(), dtype, ids.const_data_ptr(), ids.scalar_type() == at::kLong ? 1 : 0, (const float*)wt.const_data_ptr(), T, (int)top,
                   gu.const_data_ptr(), eight ? t[4]->const_data_ptr() : nullptr, dn.const_data_ptr(), eight ? t[6]->const_data_ptr() : nullptr, (int)E, (int)H, (int)F, type,
                   y.mutable_data_ptr(), scratch.mutable_data_ptr(), need, stream);
  }
  if (rc == HTR_ERR_LAUNCH) return PyLong_FromLong(rc);      // part of the layer may be queued: an error, not another way to run it
  if (rc != HTR_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// bind_unpacked(addresses of htr_rms_norm, htr_quantize_e4m3, htr_product, htr_product_rounds, htr_moe_stacked_scratch_bytes, htr_moe_stacked), after bind()
PyObject* bind_unpacked(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 6) { PyErr_SetString(PyExc_TypeError, "bind_unpacked wants six addresses"); return nullptr; }
  void* p[6];
  for (int i = 0; i < 6; ++i) p[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred()) return nullptr;
  f_norm = (decltype(f_norm))p[0]; f_quantize = (decltype(f_quantize))p[1]; f_product = (decltype(f_product))p[2];
  f_rounds = (decltype(f_rounds))p[3]; f_stacked_bytes = (decltype(f_stacked_bytes))p[4]; f_stacked = (decltype(f_stacked))p[5];
  Py_RETURN_NONE;
}

// bind(version of the library's C ABI, version of the running torch, addresses of htr_linear, htr_stream_capture_id,
// htr_moe_scratch_bytes, htr_moe_experts and, for linear() beyond 128 rows, htr_linear_route and htr_dequant_w); ImportError where either
// version is not the one that this file was compiled with
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 6 && nargs != 8) { PyErr_SetString(PyExc_TypeError, "bind wants two versions and four or six addresses"); return nullptr; }
  const long abi = PyLong_AsLong(args[0]);
  const char* torch_version = PyUnicode_AsUTF8(args[1]);
  void* p[6] = {};
  for (int i = 0; i < nargs - 2; ++i) p[i] = PyLong_AsVoidPtr(args[2 + i]);
  if (PyErr_Occurred()) return nullptr;
  if (abi != HTR_ABI_VERSION) return PyErr_Format(PyExc_ImportError, "compiled for version %d of the library's C ABI, not %ld", HTR_ABI_VERSION, abi);
  if (strcmp(torch_version, HTR_BUILD_TORCH) != 0) return PyErr_Format(PyExc_ImportError, "compiled for torch %s, not %s", HTR_BUILD_TORCH, torch_version);
  f_linear = (decltype(f_linear))p[0]; f_capture = (decltype(f_capture))p[1];
  f_moe_bytes = (decltype(f_moe_bytes))p[2]; f_moe = (decltype(f_moe))p[3];
  f_route = (decltype(f_route))p[4]; f_dequant = (decltype(f_dequant))p[5];
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", (PyCFunction)(void*)bind, METH_FASTCALL, nullptr},
                         {"linear", (PyCFunction)(void*)linear, METH_FASTCALL, nullptr},
                         {"moe", (PyCFunction)(void*)moe, METH_FASTCALL, nullptr},
                         {"bind_unpacked", (PyCFunction)(void*)bind_unpacked, METH_FASTCALL, nullptr},
                         {"rms_norm", (PyCFunction)(void*)rms_norm, METH_FASTCALL, nullptr},
                         {"product", (PyCFunction)(void*)product, METH_FASTCALL, nullptr},
                         {"moe_stacked", (PyCFunction)(void*)moe_stacked, METH_FASTCALL, nullptr},
                         {"wait_word", (PyCFunction)(void*)wait_word, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast(void) { return PyModule_Create(&module); }
