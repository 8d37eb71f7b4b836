// torch_binding.cpp — the block operators of foundry_trainer_b200.ops over
// torch tensors: argument checks, output and workspace allocation, device and
// stream, and the call of the C ABI (include/foundry_attn.h). A compiled
// module because these calls are short: through ctypes and Python checks a
// layer norm of one row spent 20 to 30 us on the host for a 2.5 us kernel.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>
#include <vector>

#include "foundry_attn.h"

namespace {

using at::Tensor;

PyObject* g_check = nullptr;  // _lib.check(status, where): raises FaError

struct Refusal {  // an argument error: becomes ValueError or TypeError
  PyObject* type;
  std::string text;
};
struct Raised {};  // a Python error is set

[[noreturn]] void refuse(const std::string& text) { throw Refusal{PyExc_ValueError, text}; }
[[noreturn]] void refuse_type(const std::string& text) { throw Refusal{PyExc_TypeError, text}; }

void checked(int status, const char* where) {
  if (status == FA_OK) return;
  PyObject* r = PyObject_CallFunction(g_check, "is", status, where);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, where);
  throw Raised{};
}

std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse_type(std::string(name) + " must be a torch.Tensor");
  return THPVariable_Unpack(o);
}
// an undefined tensor stands for None
const Tensor& maybe(PyObject* o, const char* name) {
  static const Tensor none;
  return o == Py_None ? none : tensor(o, name);
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return v;
}
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v != 0;
}

int to_int(int64_t v, const char* name) {
  if (v > INT32_MAX) refuse(std::string(name) + ": too many elements in a dimension");
  return (int)v;
}

int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return FA_DTYPE_BF16;
  if (t.scalar_type() == at::kFloat) return FA_DTYPE_F32;
  refuse_type(std::string("unsupported dtype ") + c10::toString(t.scalar_type()) +
              ": the op computes in bf16 or f32");
}

void need_cuda(const Tensor& t) {
  if (!t.is_cuda()) refuse("tensor must live on a CUDA device");
}
void same_device(const Tensor& ref, const Tensor& t, const char* name) {
  if (t.defined() && t.device() != ref.device())
    refuse(std::string(name) + " is on " + t.device().str() + ", the first operand on " +
           ref.device().str());
}

// The device of the first operand made current, with the caller's
// torch.cuda.Stream as its current stream where one is given: outputs,
// workspaces and copies belong to the stream that the kernels run on.
struct Place {
  c10::cuda::CUDAGuard guard;
  c10::cuda::OptionalCUDAStreamGuard on;
  c10::cuda::CUDAStream stream;

  Place(const Tensor& t, PyObject* s)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index())) {
    if (s == Py_None) return;
    auto field = [&](const char* n) {
      PyObject* v = PyObject_GetAttrString(s, n);
      if (v == nullptr) throw Raised{};
      const int64_t r = PyLong_AsLongLong(v);
      Py_DECREF(v);
      if (r == -1 && PyErr_Occurred()) throw Raised{};
      return r;
    };
    stream = c10::cuda::CUDAStream::unpack3(field("stream_id"),
                                            (c10::DeviceIndex)field("device_index"),
                                            (c10::DeviceType)field("device_type"));
    if (stream.device() != t.device()) refuse("the stream is on another device than the tensors");
    on.reset_stream(stream);
  }
  void* ptr() const { return stream.stream(); }
};

// a tensor to write to: every element its own
void writable(const Tensor& t) {
  if (at::has_internal_overlap(t) == at::MemOverlap::Yes)
    refuse("out has elements that share memory (an expanded tensor)");
}

Tensor scratch(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ---------------------------------------------------------------- layer norm

struct NormShape {
  int groups, rows, dim;
};

NormShape norm_shape(const Tensor& x) {
  if (x.dim() != 2 && x.dim() != 3)
    refuse("expected (rows, D) or (groups, rows, D), got " + shape_of(x));
  const int64_t g = x.dim() == 3 ? x.size(0) : 1;
  return {to_int(g, "x"), to_int(x.size(-2), "x"), to_int(x.size(-1), "x")};
}

// (rows, D) or (groups, rows, D) as the C ABI's (groups, rows, 1, D)
fa_tensor_t norm_desc(const Tensor& t) {
  return {t.data_ptr(), t.dim() == 3 ? t.stride(0) : 0, t.stride(-2), 0,
          t.size(-1) > 1 ? t.stride(-1) : 1};
}

void like_x(const Tensor& x, const Tensor& t, const char* name) {
  if (t.sizes() != x.sizes() || t.scalar_type() != x.scalar_type())
    refuse(std::string(name) + " must have x's shape and dtype");
}

struct NormParams {
  Tensor w, b;  // undefined: none
  int dtype = FA_DTYPE_F32;
  int64_t stride = 0;
  bool copy = false;

  // two modulation chunks share the stride of their rows; others are copied
  // (D values a group)
  void settle(int64_t dim) {
    if (!copy) return;
    if (w.defined()) w = w.contiguous();
    if (b.defined()) b = b.contiguous();
    if (stride != 0) stride = dim;
  }
};

NormParams norm_params(const Tensor& x, const Tensor& w, const Tensor& b) {
  NormParams p;
  const Tensor& first = w.defined() ? w : b;
  if (!first.defined()) return p;
  const bool shared = first.dim() == 1;
  for (const Tensor* t : {&w, &b}) {
    if (!t->defined()) continue;
    const bool fits = shared ? t->dim() == 1 && t->size(0) == x.size(-1)
                             : t->dim() == 2 && x.dim() == 3 && t->size(0) == x.size(0) &&
                                   t->size(1) == x.size(-1);
    if (!fits || t->scalar_type() != first.scalar_type())
      refuse("weight and bias must be (D,), or (groups, D) with x (groups, rows, D), and of one "
             "dtype: got " + shape_of(*t) + " for x " + shape_of(x));
  }
  p.dtype = dtype_code(first);
  p.w = w;
  p.b = b;
  if (!shared) {
    p.stride = first.stride(0);
    p.copy = p.stride <= 0 || x.size(0) == 1;
  }
  for (const Tensor* t : {&w, &b})
    if (t->defined())
      p.copy = p.copy || (t->stride(-1) != 1 && t->size(-1) > 1) ||
               (!shared && t->stride(0) != p.stride);
  if (!shared && p.stride <= 0) p.stride = 1;  // (settle gives it the copy's)
  return p;
}

PyObject* pair(const Tensor& a, const Tensor& b) {
  PyObject* t = PyTuple_New(2);
  if (t == nullptr) throw Raised{};
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(b));
  return t;
}
PyObject* wrap_or_none(const Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}
PyObject* triple(const Tensor& a, const Tensor& b, const Tensor& c) {
  PyObject* t = PyTuple_New(3);
  if (t == nullptr) throw Raised{};
  PyTuple_SET_ITEM(t, 0, wrap_or_none(a));
  PyTuple_SET_ITEM(t, 1, wrap_or_none(b));
  PyTuple_SET_ITEM(t, 2, wrap_or_none(c));
  return t;
}

// (x, weight, bias, unit_offset, eps, out, stream) -> (y, stats)
PyObject* layer_norm(PyObject* const* a) {
  const Tensor &x = tensor(a[0], "x"), &w = maybe(a[1], "weight"), &b = maybe(a[2], "bias"),
               &out = maybe(a[5], "out");
  const bool unit = truth(a[3]);
  const float eps = (float)number(a[4]);
  const NormShape s = norm_shape(x);
  const int dt = dtype_code(x);
  NormParams p = norm_params(x, w, b);
  if (out.defined()) {
    like_x(x, out, "out");
    writable(out);
  }
  need_cuda(x);
  same_device(x, w, "weight");
  same_device(x, b, "bias");
  same_device(x, out, "out");
  const Place at(x, a[6]);
  p.settle(s.dim);
  Tensor y = out.defined() ? out : at::empty_like(x);
  Tensor stats = at::empty({2, (int64_t)s.groups * s.rows}, x.options().dtype(at::kFloat));
  const fa_tensor_t dx = norm_desc(x), dy = norm_desc(y);
  checked(fa_layer_norm_fwd(dt, s.groups, s.rows, s.dim, &dx, ptr(p.w), ptr(p.b), p.dtype, p.stride,
                            unit, eps, &dy, stats.data_ptr<float>(), at.ptr()),
          "fa_layer_norm_fwd");
  return pair(y, stats);
}

// (x, weight, dy, stats, unit_offset, params, stream) -> (dx, dweight, dbias)
PyObject* layer_norm_bwd(PyObject* const* a) {
  const Tensor &x = tensor(a[0], "x"), &w = maybe(a[1], "weight"), &dy = tensor(a[2], "dy"),
               &stats = tensor(a[3], "stats");
  const bool unit = truth(a[4]), params = truth(a[5]);
  const NormShape s = norm_shape(x);
  const int dt = dtype_code(x);
  like_x(x, dy, "dy");
  NormParams p = norm_params(x, w, Tensor());
  need_cuda(x);
  same_device(x, w, "weight");
  same_device(x, dy, "dy");
  same_device(x, stats, "stats");
  const int64_t n = (int64_t)s.groups * s.rows;
  if (stats.scalar_type() != at::kFloat || stats.dim() != 2 || stats.size(0) != 2 ||
      stats.size(1) != n || !stats.is_contiguous())
    refuse("stats must be layer_norm's (2, rows) float32 tensor");
  const Place at(x, a[6]);
  p.settle(s.dim);
  Tensor dx = at::empty_like(x), dw, db;
  if (params) {
    const auto o = x.options().dtype(at::kFloat);
    dw = p.stride == 0 ? at::empty({s.dim}, o) : at::empty({s.groups, s.dim}, o);
    db = at::empty_like(dw);
  }
  const size_t nb = fa_layer_norm_bwd_workspace_bytes(s.groups, s.rows, s.dim);
  const Tensor ws = scratch(nb, x);
  const fa_tensor_t tx = norm_desc(x), tdy = norm_desc(dy), tdx = norm_desc(dx);
  checked(fa_layer_norm_bwd(dt, s.groups, s.rows, s.dim, &tx, ptr(p.w), p.dtype, p.stride, unit,
                            &tdy, stats.data_ptr<float>(), &tdx, (float*)ptr(dw), (float*)ptr(db),
                            ptr(ws), nb, at.ptr()),
          "fa_layer_norm_bwd");
  return triple(dx, dw, db);
}

// ----------------------------------------------------------- adapter linears

// (..., K) as one (rows, K) matrix, without a copy
Tensor rows_of(const Tensor& t, const char* name) {
  if (t.dim() == 2) return t;
  if (t.dim() < 2) refuse(std::string(name) + ": expected (..., features), got " + shape_of(t));
  const int64_t k = t.size(-1);
  int64_t want = -1, rows = 1;
  if (t.numel() == 0) {
    for (int64_t d = 0; d < t.dim() - 1; ++d) rows *= t.size(d);
    return at::empty({rows, k}, t.options());
  }
  // one stride has to run through all leading dimensions
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (want >= 0 && t.stride(d) != want)
      refuse(std::string(name) + ": the leading dimensions must be one strided set of rows; "
                                 "reshape it first");
    if (want < 0) want = t.stride(d);
    rows *= t.size(d);
    want *= t.size(d);
  }
  int64_t step = k;
  for (int64_t d = t.dim() - 2; d >= 0; --d)
    if (t.size(d) != 1) {
      step = t.stride(d);
      break;
    }
  return t.as_strided({rows, k}, {step, t.stride(-1)});
}

fa_matrix_t matrix(const Tensor& t, const char* name) {
  if (t.size(-1) > 1 && t.stride(-1) != 1)
    refuse(std::string(name) + ": the last dimension must be contiguous");
  // a stride that no element uses may be anything: give it a legal one
  const int64_t sr = t.size(-2) > 1 ? t.stride(-2) : (t.size(-1) + 7) / 8 * 8;
  int64_t sb = 0;
  if (t.dim() == 3) sb = t.size(0) > 1 ? t.stride(0) : t.size(1) * sr;
  return {t.data_ptr(), sb, sr};
}

// An uninitialised (rows, cols) bf16 matrix whose rows start on 16 bytes
Tensor aligned_rows(int64_t rows, int64_t cols, const Tensor& like) {
  const int64_t ld = (cols + 7) / 8 * 8;
  Tensor t = at::empty({rows, ld}, like.options().dtype(at::kBFloat16));
  return ld == cols ? t : t.narrow(1, 0, cols);
}

Tensor shaped_like(const Tensor& m, const Tensor& x) {  // (rows, c) as (x's leading dims, c)
  if (x.dim() == 2) return m;
  std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end()), strides(x.dim());
  sizes.back() = m.size(1);
  strides.back() = 1;
  int64_t step = m.stride(0);
  for (int64_t d = x.dim() - 2; d >= 0; --d) {
    strides[d] = step;
    step *= sizes[d];
  }
  return m.as_strided(sizes, strides);
}

void check_lora(const Tensor& x2, const Tensor& w, const Tensor& a, const Tensor& b,
                const Tensor& bias, bool stacked) {
  const Tensor* ts[] = {&x2, &w, &a, &b, &bias};
  const char* names[] = {"x", "w", "a", "b", "bias"};
  for (int i = 0; i < 5; ++i) {
    if (!ts[i]->defined()) continue;
    if (ts[i]->scalar_type() != at::kBFloat16)
      refuse_type(std::string(names[i]) + ": the linear with adapters computes in bf16, got " +
                  c10::toString(ts[i]->scalar_type()));
  }
  const int64_t nd = stacked ? 3 : 2;
  if (w.dim() != 2 || a.dim() != nd || b.dim() != nd)
    refuse("expected w (out, in) and factors a (..., rank, in), b (..., out, rank)");
  if (x2.size(1) != w.size(1) || a.size(-1) != w.size(1) || b.size(-2) != w.size(0) ||
      a.size(-2) != b.size(-1) || (stacked && a.size(0) != b.size(0)))
    refuse("shapes do not fit: x (..., " + std::to_string(x2.size(1)) + "), w " + shape_of(w) +
           ", a " + shape_of(a) + ", b " + shape_of(b));
  if (bias.defined() && (bias.dim() != 1 || bias.size(0) != w.size(0) || !bias.is_contiguous()))
    refuse("bias must be a contiguous (out,) vector");
  for (const Tensor* t : {&x2, &w, &a})
    for (int64_t n : t->sizes()) to_int(n, "x, w or a");
  need_cuda(x2);
  for (int i = 1; i < 5; ++i) same_device(x2, *ts[i], names[i]);
}

int64_t low_dim(int64_t rank) { return (rank + 15) / 16 * 32; }

// b with rows that start on 16 bytes: itself, or a copy (a rank that is no
// multiple of 8, a slice)
Tensor aligned_b(const Tensor& b, const Place& at) {
  if (b.stride(-1) != 1 && b.size(-1) > 1) refuse("b: the last dimension must be contiguous");
  const bool ok = reinterpret_cast<uintptr_t>(b.data_ptr()) % 16 == 0 &&
                  (b.size(-2) == 1 || b.stride(-2) % 8 == 0) &&
                  (b.dim() == 2 || b.size(0) == 1 || b.stride(0) % 8 == 0);
  if (ok || b.numel() == 0) return b;
  const int64_t r = b.size(-1), ld = (r + 7) / 8 * 8;
  // adapters that are no one strided set of rows (a slice of each)
  if (b.dim() == 3 && b.size(0) > 1 && b.size(1) > 1 && b.stride(0) != b.size(1) * b.stride(1)) {
    Tensor t = at::empty({b.size(0), b.size(1), ld}, b.options()).narrow(2, 0, r);
    t.copy_(b.detach());
    return t;
  }
  Tensor rows = rows_of(b, "b");
  Tensor t = at::empty({rows.size(0), ld}, b.options());
  checked(fa_pad_rows((int64_t)rows.size(0), (int)r, rows.data_ptr(), rows.stride(0), t.data_ptr(),
                      ld, at.ptr()),
          "fa_pad_rows");
  t = t.narrow(1, 0, r);
  return b.dim() == 2 ? t : t.as_strided(b.sizes(), {b.size(1) * ld, ld, 1});
}

// (x, w, a, b, scale, bias, stream) -> (y, low)
PyObject* lora_linear(PyObject* const* a_) {
  const Tensor &x = tensor(a_[0], "x"), &w = tensor(a_[1], "w"), &a = tensor(a_[2], "a"),
               &b = tensor(a_[3], "b"), &bias = maybe(a_[5], "bias");
  const float scale = (float)number(a_[4]);
  const Tensor x2 = rows_of(x, "x");
  check_lora(x2, w, a, b, bias, false);
  const Place at(x, a_[6]);
  const Tensor bb = aligned_b(b, at);
  const int64_t N = x2.size(0), K = w.size(1), M = w.size(0), r = a.size(0);
  Tensor y = aligned_rows(N, M, x), low = at::empty({N, low_dim(r)}, x.options());
  const fa_matrix_t mx = matrix(x2, "x"), mw = matrix(w, "w"), ma = matrix(a, "a"),
                    mb = matrix(bb, "b"), my = matrix(y, "y");
  checked(fa_lora_linear_fwd(FA_DTYPE_BF16, (int)N, (int)K, (int)M, (int)r, &mx, &mw, &ma, &mb,
                             scale, ptr(bias), &my, low.data_ptr(), at.ptr()),
          "fa_lora_linear_fwd");
  return pair(shaped_like(y, x), low);
}

// (x, w, a, b, dy, low, scale, need_dx, need_factors, stream) -> (dx, da, db)
PyObject* lora_linear_bwd(PyObject* const* a_) {
  const Tensor &x = tensor(a_[0], "x"), &w = tensor(a_[1], "w"), &a = tensor(a_[2], "a"),
               &b = tensor(a_[3], "b"), &dy = tensor(a_[4], "dy"), &low = tensor(a_[5], "low");
  const float scale = (float)number(a_[6]);
  const bool need_dx = truth(a_[7]), need_factors = truth(a_[8]);
  const Tensor x2 = rows_of(x, "x"), dy2 = rows_of(dy, "dy");
  check_lora(x2, w, a, b, Tensor(), false);
  same_device(x, dy, "dy");
  same_device(x, low, "low");
  const int64_t N = x2.size(0), K = w.size(1), M = w.size(0), r = a.size(0);
  if (dy2.scalar_type() != at::kBFloat16 || dy2.size(0) != N || dy2.size(1) != M)
    refuse("dy must be bf16 (..., " + std::to_string(M) + ") with x's rows");
  if (low.scalar_type() != at::kBFloat16 || low.dim() != 2 || low.size(0) != N ||
      low.size(1) != low_dim(r) || !low.is_contiguous())
    refuse("low must be the tensor lora_linear returned for these rows");
  const Place at(x, a_[9]);
  const Tensor bb = aligned_b(b, at);
  Tensor dx, da, db;
  if (need_dx) dx = aligned_rows(N, K, x);
  if (need_factors) {
    da = at::empty({r, K}, x.options());
    db = at::empty({M, r}, x.options());
  }
  const size_t nb = fa_lora_linear_bwd_workspace_bytes((int)N, (int)r);
  const Tensor ws = scratch(nb, x);
  const fa_matrix_t mx = matrix(x2, "x"), mw = matrix(w, "w"), ma = matrix(a, "a"),
                    mb = matrix(bb, "b"), mdy = matrix(dy2, "dy");
  fa_matrix_t mdx{};
  if (need_dx) mdx = matrix(dx, "dx");
  checked(fa_lora_linear_bwd(FA_DTYPE_BF16, (int)N, (int)K, (int)M, (int)r, &mx, &mw, &ma, &mb,
                             scale, low.data_ptr(), &mdy, need_dx ? &mdx : nullptr, ptr(da), ptr(db),
                             ptr(ws), nb, at.ptr()),
          "fa_lora_linear_bwd");
  return triple(need_dx ? shaped_like(dx, x) : dx, da, db);
}

// (x, w, a, b, ids, scales, bias, stream) -> y
PyObject* lora_linear_many(PyObject* const* a_) {
  const Tensor &x = tensor(a_[0], "x"), &w = tensor(a_[1], "w"), &a = tensor(a_[2], "a"),
               &b = tensor(a_[3], "b"), &ids = tensor(a_[4], "ids"),
               &scales = tensor(a_[5], "scales"), &bias = maybe(a_[6], "bias");
  const Tensor x2 = rows_of(x, "x");
  check_lora(x2, w, a, b, bias, true);
  same_device(x, ids, "ids");
  same_device(x, scales, "scales");
  const int64_t N = x2.size(0), K = w.size(1), M = w.size(0), r = a.size(1), E = a.size(0);
  if (ids.scalar_type() != at::kInt || ids.dim() != 1 || ids.size(0) != N || !ids.is_contiguous())
    refuse("ids must be a contiguous int32 (" + std::to_string(N) + ",) tensor");
  if (scales.scalar_type() != at::kFloat || scales.dim() != 1 || scales.size(0) != E ||
      !scales.is_contiguous())
    refuse("scales must be a contiguous float32 (" + std::to_string(E) + ",) tensor");
  const Place at(x, a_[7]);
  const Tensor bb = aligned_b(b, at);
  Tensor y = aligned_rows(N, M, x);
  const size_t nb = fa_lora_linear_many_workspace_bytes((int)N, (int)r);
  const Tensor ws = scratch(nb, x);
  const fa_matrix_t mx = matrix(x2, "x"), mw = matrix(w, "w"), ma = matrix(a, "a"),
                    mb = matrix(bb, "b"), my = matrix(y, "y");
  checked(fa_lora_linear_many(FA_DTYPE_BF16, (int)N, (int)K, (int)M, (int)r, (int)E, &mx, &mw, &ma,
                              &mb, ids.data_ptr<int32_t>(), scales.data_ptr<float>(), ptr(bias), &my,
                              ptr(ws), nb, at.ptr()),
          "fa_lora_linear_many");
  return THPVariable_Wrap(shaped_like(y, x));
}

// ------------------------------------------------------------ orthogonalise

// (..., m, n) as (batch, m, n), without a copy
Tensor matrices_of(const Tensor& t, const char* name) {
  const int64_t m = t.size(-2), n = t.size(-1);
  if (n > 1 && t.stride(-1) != 1)
    refuse(std::string(name) + "'s last dimension must be contiguous");
  if (t.dim() == 3) return t;
  if (t.dim() == 2) return t.unsqueeze(0);
  int64_t want = -1, batch = 1, step = 0;
  for (int64_t d = t.dim() - 3; d >= 0; --d) {
    batch *= t.size(d);
    if (t.size(d) == 1) continue;
    if (want >= 0 && t.stride(d) != want && t.numel() > 0)
      refuse(std::string(name) + ": the leading dimensions must be one strided set of matrices; "
                                 "reshape it first");
    if (want < 0) step = want = t.stride(d);
    want *= t.size(d);
  }
  return t.as_strided({batch, m, n}, {step, t.stride(-2), t.stride(-1)});
}

// (g, steps, a, b, c, eps, out, stream) -> o
PyObject* orthogonalize(PyObject* const* a_) {
  const Tensor &g = tensor(a_[0], "g"), &out = maybe(a_[6], "out");
  const int steps = to_int(std::max<int64_t>(integer(a_[1]), -1), "steps");
  const float a = (float)number(a_[2]), b = (float)number(a_[3]), c = (float)number(a_[4]),
              eps = (float)number(a_[5]);
  if (g.dim() < 2) refuse("expected (..., m, n), got " + shape_of(g));
  const int dt = dtype_code(g);
  if (out.defined()) {
    if (out.sizes() != g.sizes() || out.scalar_type() != at::kBFloat16)
      refuse("out must be bf16 with g's shape");
    writable(out);
  }
  need_cuda(g);
  same_device(g, out, "out");
  const Tensor g3 = matrices_of(g, "g");
  const int B = to_int(g3.size(0), "g"), m = to_int(g3.size(1), "g"), n = to_int(g3.size(2), "g");
  const Place at(g, a_[7]);
  Tensor o, o3;
  if (out.defined()) {
    o = out;
    o3 = matrices_of(out, "out");
  } else {
    const int64_t ld = ((int64_t)n + 7) / 8 * 8;
    o = at::empty({(int64_t)B * m, ld}, g.options().dtype(at::kBFloat16));
    std::vector<int64_t> strides(g.dim());
    strides.back() = 1;
    int64_t step = ld;
    for (int64_t d = g.dim() - 2; d >= 0; --d) {
      strides[d] = step;
      step *= g.size(d);
    }
    o = o.as_strided(g.sizes(), strides);
    o3 = matrices_of(o, "out");
  }
  const fa_matrix_t mo = matrix(o3, "out");
  const size_t nb = fa_orthogonalize_workspace_bytes(B, m, n, steps);
  const Tensor ws = scratch(nb, g);
  checked(fa_orthogonalize(dt, B, m, n, g3.data_ptr(), g3.stride(0), g3.stride(1), mo.data,
                           mo.stride_batch, mo.stride_row, steps, a, b, c, eps, ptr(ws), nb,
                           at.ptr()),
          "fa_orthogonalize");
  return THPVariable_Wrap(o);
}

// ------------------------------------------------------------------- module

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  HANDLE_TH_ERRORS
  try {
    return F(args);
  } catch (const Refusal& r) {
    PyErr_SetString(r.type, r.text.c_str());
    return nullptr;
  } catch (const Raised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* set_check(PyObject*, PyObject* f) {
  Py_XINCREF(f);
  Py_XDECREF(g_check);
  g_check = f;
  Py_RETURN_NONE;
}

#define FA_METHOD(F, N) \
  {#F, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<F, N>)), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {FA_METHOD(layer_norm, 7),
                         FA_METHOD(layer_norm_bwd, 7),
                         FA_METHOD(lora_linear, 7),
                         FA_METHOD(lora_linear_bwd, 10),
                         FA_METHOD(lora_linear_many, 8),
                         FA_METHOD(orthogonalize, 8),
                         {"set_check", &set_check, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fa_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__fa_torch(void) { return PyModule_Create(&module); }
