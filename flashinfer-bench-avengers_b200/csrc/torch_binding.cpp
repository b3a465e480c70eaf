// Python binding of the dense operators (module _moe_b200_torch): takes torch
// tensors, tests the conditions the library relies on, allocates outputs and
// scratch from torch's caching allocator, and calls the C ABI on the current
// stream of the tensors' device.
//
// A call from Python costs little beyond its launches this way: 8 us instead
// of 15.5 for the feed-forward block, 5 instead of 11 for the quantiser, 6
// instead of 13 for the 4-bit linear at one token, against the same conditions
// and allocations in Python; that was most of a call on few tokens.
//
// Every function returns None where a condition fails; ffn_host then goes
// through the arguments one by one for the message. A status code of the
// library comes back as an integer. The library's entry points are handed over
// by address (bind), so the module does not link to it.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <optional>

#include "../../include/moe_b200.h"

namespace {

constexpr int64_t kMaxDim = 65536;

struct Library {
  decltype(&moe_b200_gated_ffn) gated_ffn;
  decltype(&moe_b200_gated_ffn_workspace_bytes) gated_ffn_bytes;
  decltype(&moe_b200_gated_ffn_backward) gated_ffn_backward;
  decltype(&moe_b200_gated_ffn_backward_workspace_bytes) gated_ffn_backward_bytes;
  decltype(&moe_b200_mxfp4_quantize) quantize;
  decltype(&moe_b200_mxfp4_dequantize) dequantize;
  decltype(&moe_b200_mxfp4_matmul) matmul;
  decltype(&moe_b200_mxfp4_linear) linear;
  decltype(&moe_b200_mxfp4_linear_workspace_bytes) linear_bytes;
  decltype(&moe_b200_mxfp4_gated_ffn) mx_ffn;
  decltype(&moe_b200_mxfp4_gated_ffn_workspace_bytes) mx_ffn_bytes;
};
Library lib;
bool bound = false;

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ------------------------------------------------------------- conditions
const at::Tensor* tensor(PyObject* o) {
  return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return MOE_B200_TYPE_BF16;
    case at::kHalf: return MOE_B200_TYPE_FP16;
    case at::kFloat: return MOE_B200_TYPE_FP32;
    default: return -1;
  }
}

std::optional<at::ScalarType> scalar_type(long code) {
  switch (code) {
    case MOE_B200_TYPE_BF16: return at::kBFloat16;
    case MOE_B200_TYPE_FP16: return at::kHalf;
    case MOE_B200_TYPE_FP32: return at::kFloat;
    default: return std::nullopt;
  }
}

bool strided_cuda(const at::Tensor& t) { return t.defined() && t.is_cuda() && t.layout() == at::kStrided; }

bool aligned(const at::Tensor& t, uintptr_t a) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % a == 0; }

// Elements between the rows of a matrix the kernels can read, else -1: rows
// contiguous, not overlapping, each starting on 16 bytes. A lone row has no
// pitch; its length, a multiple of 16 bytes where the size checks pass, stands
// in.
int64_t pitch_of(const at::Tensor& t) {
  if (t.dim() != 2) return -1;
  const int64_t rows = t.size(0), cols = t.size(1);
  const int64_t pitch = rows > 1 ? t.stride(0) : cols;
  if ((t.stride(1) != 1 && cols > 1) || pitch < cols || rows > MOE_B200_MAX_TOKENS) return -1;
  if (rows > 0 && (!aligned(t, 16) || (rows > 1 && pitch * t.element_size() % 16 != 0))) return -1;
  return pitch;
}

bool dense(const at::Tensor* t, int64_t rows, int64_t cols, at::ScalarType type, at::Device dev, uintptr_t align = 16) {
  return t != nullptr && strided_cuda(*t) && t->dim() == 2 && t->size(0) == rows && t->size(1) == cols &&
         t->scalar_type() == type && t->device() == dev && t->is_contiguous() && aligned(*t, align);
}

bool dim_ok(int64_t d, int64_t multiple) { return d >= multiple && d <= kMaxDim && d % multiple == 0; }

struct Ffn {
  const at::Tensor *x, *w13, *w2;
  int64_t T, H, I, pitch;
  int type;
};

bool read_ffn(PyObject* x, PyObject* w13, PyObject* w2, Ffn* f) {
  f->x = tensor(x), f->w13 = tensor(w13), f->w2 = tensor(w2);
  if (!f->x || !f->w13 || !f->w2 || !strided_cuda(*f->x) || f->w2->dim() != 2 || f->x->dim() != 2) return false;
  f->pitch = pitch_of(*f->x);
  f->type = type_code(f->x->scalar_type());
  f->T = f->x->size(0), f->H = f->w2->size(0), f->I = f->w2->size(1);
  const at::Device dev = f->x->device();
  return f->pitch >= 0 && f->x->size(1) == f->H &&
         (f->type == MOE_B200_TYPE_BF16 || f->type == MOE_B200_TYPE_FP16) && dim_ok(f->H, 8) && dim_ok(f->I, 8) &&
         dense(f->w13, 2 * f->I, f->H, f->x->scalar_type(), dev) && dense(f->w2, f->H, f->I, f->x->scalar_type(), dev);
}

// A 4-bit matrix: codes [rows, cols / 2] and tiled exponents.
struct Mx {
  const at::Tensor *q, *scale;
  int64_t rows, cols;
};

bool read_mx(PyObject* q, PyObject* scale, const at::Device* dev, Mx* m) {
  m->q = tensor(q), m->scale = tensor(scale);
  if (!m->q || !m->scale || !strided_cuda(*m->q) || !strided_cuda(*m->scale) || m->q->dim() != 2) return false;
  m->rows = m->q->size(0), m->cols = 2 * m->q->size(1);
  const at::Tensor& s = *m->scale;
  return (!dev || m->q->device() == *dev) && m->q->scalar_type() == at::kByte && m->q->is_contiguous() &&
         m->rows <= MOE_B200_MAX_TOKENS && dim_ok(m->cols, 32) && aligned(*m->q, 16) && s.scalar_type() == at::kByte &&
         s.device() == m->q->device() && s.is_contiguous() && aligned(s, 16) && s.dim() == 5 &&
         s.size(0) == div_up(m->rows, 128) && s.size(1) == div_up(m->cols, 128) && s.size(2) == 32 && s.size(3) == 4 &&
         s.size(4) == 4;
}

// ------------------------------------------------------------ allocation
at::Tensor matrix(int64_t rows, int64_t cols, at::ScalarType type, at::Device dev) {
  return at::empty({rows, cols}, at::TensorOptions().dtype(type).device(dev));
}

// Device memory for this call; freed into the stream's order at its end.
struct Scratch {
  at::Tensor t;
  Scratch(size_t bytes, at::Device dev)
      : t(at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(dev))) {}
  void* ptr() const { return t.data_ptr(); }
  size_t bytes() const { return static_cast<size_t>(t.numel()); }
};

void* current_stream(at::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// Bytes from a tensor's first element to its last.
uintptr_t span(const at::Tensor& t) {
  int64_t n = 1;
  for (int64_t d = 0; d < t.dim(); ++d) n += (t.size(d) - 1) * t.stride(d);
  return static_cast<uintptr_t>(n * t.element_size());
}

bool overlap(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.const_data_ptr());
  const uintptr_t pb = reinterpret_cast<uintptr_t>(b.const_data_ptr());
  return pa < pb + span(b) && pb < pa + span(a);
}

// Whether one of these carries a forward-mode tangent, which no call here
// computes. (Gradient mode says nothing about forward mode: torch.no_grad()
// leaves it on.)
bool tangents(std::initializer_list<const at::Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return false;
  for (const at::Tensor* t : ts)
    if (t->_fw_grad(0).defined()) return true;
  return false;
}

// Whether autograd is to record a call on x, which the 4-bit functions do not:
// their results would silently cut the graph.
bool recorded(const at::Tensor& x) { return at::GradMode::is_enabled() && x.requires_grad(); }

// `given` if it is an output of this shape and type, a new tensor if it is
// None; nullopt if it will not do. A given one is written in place: it may
// overlap no input, autograd must not follow it (a tangent would stay that of the
// old values), and its version goes up, so that a backward pass which saved it
// notices.
std::optional<at::Tensor> output(PyObject* given, int64_t rows, int64_t cols, at::ScalarType type, at::Device dev,
                                 std::initializer_list<const at::Tensor*> inputs) {
  if (given == Py_None) return matrix(rows, cols, type, dev);
  const at::Tensor* t = tensor(given);
  if (!dense(t, rows, cols, type, dev) || (at::GradMode::is_enabled() && t->requires_grad()) || tangents({t}))
    return std::nullopt;
  for (const at::Tensor* in : inputs)
    if (overlap(*t, *in)) return std::nullopt;
  if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return *t;
}

PyObject* result(int code, const at::Tensor& t) { return code ? PyLong_FromLong(code) : THPVariable_Wrap(t); }

PyObject* tuple_of(std::initializer_list<const at::Tensor*> ts) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (out == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor* t : ts) {
    PyObject* o = t->defined() ? THPVariable_Wrap(*t) : Py_NewRef(Py_None);
    if (o == nullptr) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

bool ready(Py_ssize_t n, Py_ssize_t want) {
  if (bound && n == want) return true;
  PyErr_SetString(PyExc_TypeError, bound ? "wrong number of arguments" : "bind() comes first");
  return false;
}

// -------------------------------------------------------------- functions
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void** slots = reinterpret_cast<void**>(&lib);
  constexpr Py_ssize_t kCount = sizeof(Library) / sizeof(void*);
  if (n != kCount) {
    PyErr_SetString(PyExc_TypeError, "one address per entry point");
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < n; ++i) {
    slots[i] = PyLong_AsVoidPtr(a[i]);
    if (slots[i] == nullptr && PyErr_Occurred()) return nullptr;
  }
  bound = true;
  Py_RETURN_NONE;
}

// (x, w13, w2, activation, output or None) -> output; False where gradients
// are to be recorded.
PyObject* gated_ffn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!ready(n, 5)) return nullptr;
  Ffn f;
  if (!read_ffn(a[0], a[1], a[2], &f) || tangents({f.x, f.w13, f.w2})) Py_RETURN_NONE;
  if (at::GradMode::is_enabled() && (f.x->requires_grad() || f.w13->requires_grad() || f.w2->requires_grad()))
    Py_RETURN_FALSE;
  const at::Device dev = f.x->device();
  const std::optional<at::Tensor> out = output(a[4], f.T, f.H, f.x->scalar_type(), dev, {f.x, f.w13, f.w2});
  if (!out) Py_RETURN_NONE;
  int code = 0;
  if (f.T > 0) {
    const c10::cuda::CUDAGuard guard(dev);
    const Scratch ws(lib.gated_ffn_bytes(f.T, f.H, f.I), dev);
    code = lib.gated_ffn(f.x->const_data_ptr(), f.pitch, f.w13->const_data_ptr(), f.w2->const_data_ptr(), f.type,
                         static_cast<int>(PyLong_AsLong(a[3])), f.T, f.H, f.I, out->mutable_data_ptr(), nullptr,
                         nullptr, ws.ptr(), ws.bytes(), current_stream(dev));
  }
  return result(code, *out);
  END_HANDLE_TH_ERRORS
}

// (x, w13, w2, activation) -> (output, u and g, hidden)
PyObject* gated_ffn_save(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!ready(n, 4)) return nullptr;
  Ffn f;
  if (!read_ffn(a[0], a[1], a[2], &f) || tangents({f.x, f.w13, f.w2})) Py_RETURN_NONE;
  const at::Device dev = f.x->device();
  const at::Tensor out = matrix(f.T, f.H, f.x->scalar_type(), dev);
  const at::Tensor preact = matrix(f.T, 2 * f.I, at::kFloat, dev);
  const at::Tensor hidden = matrix(f.T, f.I, f.x->scalar_type(), dev);
  int code = 0;
  if (f.T > 0) {
    const c10::cuda::CUDAGuard guard(dev);
    // (a few tokens keep a second part of the hidden in the workspace)
    const Scratch ws(f.T <= MOE_B200_FFN_TWO_PART_TOKENS ? lib.gated_ffn_bytes(f.T, f.H, f.I) : 0, dev);
    code = lib.gated_ffn(f.x->const_data_ptr(), f.pitch, f.w13->const_data_ptr(), f.w2->const_data_ptr(), f.type,
                         static_cast<int>(PyLong_AsLong(a[3])), f.T, f.H, f.I, out.mutable_data_ptr(),
                         static_cast<float*>(preact.mutable_data_ptr()), hidden.mutable_data_ptr(), ws.ptr(),
                         ws.bytes(), current_stream(dev));
  }
  return code ? PyLong_FromLong(code) : tuple_of({&out, &preact, &hidden});
  END_HANDLE_TH_ERRORS
}

// (grad_output, x, w13, w2, u and g, hidden, activation, needs x, w13, w2)
// -> (grad_x, grad_w13, grad_w2), None where not needed
PyObject* gated_ffn_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!ready(n, 10)) return nullptr;
  Ffn f;
  const at::Tensor *dy = tensor(a[0]), *preact = tensor(a[4]), *hidden = tensor(a[5]);
  if (!read_ffn(a[1], a[2], a[3], &f) || !dy || !strided_cuda(*dy)) Py_RETURN_NONE;
  const at::ScalarType type = f.x->scalar_type();
  const at::Device dev = f.x->device();
  const int64_t dy_pitch = pitch_of(*dy);
  if (dy_pitch < 0 || dy->size(0) != f.T || dy->size(1) != f.H || dy->scalar_type() != type || dy->device() != dev ||
      !dense(preact, f.T, 2 * f.I, at::kFloat, dev, 32) || !dense(hidden, f.T, f.I, type, dev) ||
      tangents({dy, f.x, f.w13, f.w2, preact, hidden}))
    Py_RETURN_NONE;
  at::Tensor grads[3];
  const int64_t shape[3][2] = {{f.T, f.H}, {2 * f.I, f.H}, {f.H, f.I}};
  bool any = false;
  for (int i = 0; i < 3; ++i) {
    const int need = PyObject_IsTrue(a[7 + i]);
    if (need < 0) return nullptr;
    if (need) grads[i] = matrix(shape[i][0], shape[i][1], type, dev);
    any = any || need;
  }
  int code = 0;
  if (any) {
    const c10::cuda::CUDAGuard guard(dev);
    // [du | dg], which the gradient of w2 alone does not read
    const bool dact = grads[0].defined() || grads[1].defined();
    const Scratch ws(dact ? lib.gated_ffn_backward_bytes(f.T, f.H, f.I) : 0, dev);
    auto at_of = [](const at::Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; };
    code = lib.gated_ffn_backward(dy->const_data_ptr(), dy_pitch, f.x->const_data_ptr(), f.pitch,
                                  f.w13->const_data_ptr(), f.w2->const_data_ptr(),
                                  static_cast<const float*>(preact->const_data_ptr()), hidden->const_data_ptr(),
                                  f.type, static_cast<int>(PyLong_AsLong(a[6])), f.T, f.H, f.I, at_of(grads[0]),
                                  at_of(grads[1]), at_of(grads[2]), ws.ptr(), ws.bytes(), current_stream(dev));
  }
  return code ? PyLong_FromLong(code) : tuple_of({&grads[0], &grads[1], &grads[2]});
  END_HANDLE_TH_ERRORS
}

// Unquantised rows of a 4-bit operand, or -1.
int64_t read_rows(const at::Tensor* x) {
  if (!x || !strided_cuda(*x) || type_code(x->scalar_type()) < 0) return -1;
  const int64_t pitch = pitch_of(*x);
  return pitch >= 0 && dim_ok(x->size(1), 32) ? pitch : -1;
}

// (x) -> (codes, exponents)
PyObject* mxfp4_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!ready(n, 1)) return nullptr;
  const at::Tensor* x = tensor(a[0]);
  const int64_t pitch = read_rows(x);
  if (pitch < 0) Py_RETURN_NONE;
  const at::Device dev = x->device();
  const int64_t R = x->size(0), K = x->size(1);
  const at::Tensor q = matrix(R, K / 2, at::kByte, dev);
  const at::Tensor scale = at::empty({div_up(R, 128), div_up(K, 128), 32, 4, 4}, q.options());
  int code = 0;
  if (R > 0) {
    const c10::cuda::CUDAGuard guard(dev);
    code = lib.quantize(x->const_data_ptr(), pitch, type_code(x->scalar_type()), R, K, q.mutable_data_ptr(),
                        scale.mutable_data_ptr(), current_stream(dev));
  }
  return code ? PyLong_FromLong(code) : tuple_of({&q, &scale});
  END_HANDLE_TH_ERRORS
}

// (codes, exponents, type code) -> values
PyObject* mxfp4_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!ready(n, 3)) return nullptr;
  Mx m;
  const std::optional<at::ScalarType> type = scalar_type(PyLong_AsLong(a[2]));
  if (!type || !read_mx(a[0], a[1], nullptr, &m)) Py_RETURN_NONE;
  const at::Device dev = m.q->device();
  const at::Tensor out = matrix(m.rows, m.cols, *type, dev);
  int code = 0;
  if (m.rows > 0) {
    const c10::cuda::CUDAGuard guard(dev);
    code = lib.dequantize(m.q->const_data_ptr(), m.scale->const_data_ptr(), m.rows, m.cols, type_code(*type),
                          out.mutable_data_ptr(), current_stream(dev));
  }
  return result(code, out);
  END_HANDLE_TH_ERRORS
}

// (a codes, a exponents, b codes, b exponents, type code, output or None)
PyObject* mxfp4_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!ready(n, 6)) return nullptr;
  Mx l, r;
  const std::optional<at::ScalarType> type = scalar_type(PyLong_AsLong(a[4]));
  if (!type || !read_mx(a[0], a[1], nullptr, &l)) Py_RETURN_NONE;
  const at::Device dev = l.q->device();
  if (!read_mx(a[2], a[3], &dev, &r) || r.cols != l.cols || r.rows == 0) Py_RETURN_NONE;
  const std::optional<at::Tensor> out = output(a[5], l.rows, r.rows, *type, dev, {l.q, l.scale, r.q, r.scale});
  if (!out) Py_RETURN_NONE;
  int code = 0;
  if (l.rows > 0) {
    const c10::cuda::CUDAGuard guard(dev);
    code = lib.matmul(l.q->const_data_ptr(), l.scale->const_data_ptr(), r.q->const_data_ptr(),
                      r.scale->const_data_ptr(), l.rows, r.rows, l.cols, type_code(*type), out->mutable_data_ptr(),
                      current_stream(dev));
  }
  return result(code, *out);
  END_HANDLE_TH_ERRORS
}

// (x, w codes, w exponents, output or None)
PyObject* mxfp4_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!ready(n, 4)) return nullptr;
  const at::Tensor* x = tensor(a[0]);
  const int64_t pitch = read_rows(x);
  if (pitch < 0) Py_RETURN_NONE;
  const at::Device dev = x->device();
  const int64_t T = x->size(0), K = x->size(1);
  Mx w;
  if (!read_mx(a[1], a[2], &dev, &w) || w.cols != K || w.rows == 0 || tangents({x}) || recorded(*x))
    Py_RETURN_NONE;
  const std::optional<at::Tensor> out = output(a[3], T, w.rows, x->scalar_type(), dev, {x, w.q, w.scale});
  if (!out) Py_RETURN_NONE;
  int code = 0;
  if (T > 0) {
    const c10::cuda::CUDAGuard guard(dev);
    const Scratch ws(lib.linear_bytes(T, K), dev);
    code = lib.linear(x->const_data_ptr(), pitch, type_code(x->scalar_type()), w.q->const_data_ptr(),
                      w.scale->const_data_ptr(), T, w.rows, K, out->mutable_data_ptr(), ws.ptr(), ws.bytes(),
                      current_stream(dev));
  }
  return result(code, *out);
  END_HANDLE_TH_ERRORS
}

// (x, w13 codes, w13 exponents, w2 codes, w2 exponents, activation, output or None)
PyObject* mxfp4_gated_ffn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!ready(n, 7)) return nullptr;
  const at::Tensor* x = tensor(a[0]);
  const int64_t pitch = read_rows(x);
  if (pitch < 0) Py_RETURN_NONE;
  const at::Device dev = x->device();
  const int64_t T = x->size(0), H = x->size(1);
  Mx w13, w2;
  if (!read_mx(a[1], a[2], &dev, &w13) || !read_mx(a[3], a[4], &dev, &w2) || w13.cols != H || w2.rows != H ||
      w13.rows != 2 * w2.cols || tangents({x}) || recorded(*x))
    Py_RETURN_NONE;
  const std::optional<at::Tensor> out =
      output(a[6], T, H, x->scalar_type(), dev, {x, w13.q, w13.scale, w2.q, w2.scale});
  if (!out) Py_RETURN_NONE;
  int code = 0;
  if (T > 0) {
    const c10::cuda::CUDAGuard guard(dev);
    const Scratch ws(lib.mx_ffn_bytes(T, H, w2.cols), dev);
    code = lib.mx_ffn(x->const_data_ptr(), pitch, type_code(x->scalar_type()), w13.q->const_data_ptr(),
                      w13.scale->const_data_ptr(), w2.q->const_data_ptr(), w2.scale->const_data_ptr(),
                      static_cast<int>(PyLong_AsLong(a[5])), T, H, w2.cols, out->mutable_data_ptr(), ws.ptr(),
                      ws.bytes(), current_stream(dev));
  }
  return result(code, *out);
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {
    method<bind>("bind"),
    method<gated_ffn>("gated_ffn"),
    method<gated_ffn_save>("gated_ffn_save"),
    method<gated_ffn_backward>("gated_ffn_backward"),
    method<mxfp4_quantize>("mxfp4_quantize"),
    method<mxfp4_dequantize>("mxfp4_dequantize"),
    method<mxfp4_matmul>("mxfp4_matmul"),
    method<mxfp4_linear>("mxfp4_linear"),
    method<mxfp4_gated_ffn>("mxfp4_gated_ffn"),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_moe_b200_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__moe_b200_torch(void) { return PyModule_Create(&module); }
