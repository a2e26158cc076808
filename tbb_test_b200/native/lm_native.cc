// The calls of norm, norm_grad, clip and sample (tbb_test_b200/lm.py) on torch tensors, in C++: what they check, allocate and hand to the C ABI takes as
// long in Python as the kernels of small calls take on the GPU (a norm of one row 13 us of the caller's time, 300 tensors to be clipped 240). Nothing is kept between calls
// but the entries' addresses, which lm.py gives, so that both bindings use the same library.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <exception>
#include <limits>
#include <string>
#include <utility>
#include <vector>

#include "../../include/b200mlp.h"

namespace {

decltype(&b2_norm) p_norm;
decltype(&b2_norm_grad_workspace) p_norm_grad_workspace;
decltype(&b2_norm_grad) p_norm_grad;
decltype(&b2_clip_workspace) p_clip_workspace;
decltype(&b2_clip) p_clip;
decltype(&b2_sample_workspace) p_sample_workspace;
decltype(&b2_sample) p_sample;
decltype(&b2_last_error) p_last_error;
PyObject* error_class;  // _capi.B2Error

// A Python exception that is already set.
struct Raised {};

[[noreturn]] void refuse(const std::string& text) {
  PyErr_SetString(PyExc_ValueError, text.c_str());
  throw Raised();
}
void check(int rc) {
  if (rc == B2_OK) return;
  PyObject* e = PyObject_CallFunction(error_class, "is", rc, p_last_error(nullptr));
  if (e) {
    PyErr_SetObject(error_class, e);
    Py_DECREF(e);
  }
  throw Raised();
}

int type_code(at::ScalarType t) { return t == at::kFloat ? B2_DTYPE_F32 : t == at::kBFloat16 ? B2_DTYPE_BF16 : -1; }
std::string shape_text(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
bool given(PyObject* x) { return x && x != Py_None; }
const at::Tensor& tensor(const char* name, PyObject* x) {
  if (!THPVariable_Check(x)) refuse(std::string(name) + ": a tensor is wanted");
  return THPVariable_Unpack(x);
}

struct Matrix {
  void* p = nullptr;
  size_t rows = 0, cols = 0, ld = 0;
  int type = 0;
};
// A two-dimensional CUDA tensor with unit stride along its rows; `like`: of its type, shape and device.
Matrix matrix(const char* name, const at::Tensor& t, const at::Tensor* like = nullptr) {
  const std::string n(name);
  if (t.dim() != 2) refuse(n + ": a two-dimensional tensor is wanted");
  if (!t.is_cuda() || (like && t.device() != like->device())) refuse(n + ": on " + t.device().str() + ", wanted on " + (like ? like->device().str() : "a CUDA device"));
  Matrix m;
  m.type = type_code(t.scalar_type());
  if (m.type < 0 || (like && t.scalar_type() != like->scalar_type()))
    refuse(n + ": " + c10::toString(t.scalar_type()) + ", wanted " + (like ? c10::toString(like->scalar_type()) : "float32 or bfloat16"));
  if (like && t.sizes() != like->sizes()) refuse(n + ": shape " + shape_text(t) + ", wanted " + shape_text(*like));
  m.rows = t.size(0);
  m.cols = t.size(1);
  if (m.cols > 1 && t.stride(1) != 1) refuse(n + ": rows need unit stride");
  m.ld = m.rows <= 1 ? m.cols : t.stride(0);
  if (m.rows > 1 && t.stride(0) < (int64_t)m.cols) refuse(n + ": rows overlap");
  m.p = t.data_ptr();
  return m;
}
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, c10::Device device) { return at::detail::empty_cuda(sizes, type, device, std::nullopt); }
at::Tensor workspace(size_t bytes, c10::Device device) { return fresh({(int64_t)(bytes ? bytes : 1)}, at::kByte, device); }

// A given tensor that a call has written to counts as changed in place, where autograd keeps count.
void changed(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

// The device of a call made the current one, and the address of its current stream.
struct On {
  c10::cuda::OptionalCUDAGuard guard;
  void* stream;
  explicit On(c10::Device d) : guard(d), stream(c10::cuda::getCurrentCUDAStream(d.index()).stream()) {}
};
template <class Call>
int without_gil(Call call) {
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = call();
  Py_END_ALLOW_THREADS;
  return rc;
}

double number(PyObject* x) {
  const double v = PyFloat_AsDouble(x);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}
long integer(PyObject* x) {
  const long v = PyLong_AsLong(x);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}

// A norm's weight: one element per column, of the matrices' type or float32.
std::pair<void*, int> weight_of(PyObject* w, const at::Tensor& x) {
  if (!given(w)) return {nullptr, type_code(x.scalar_type())};
  const at::Tensor& t = tensor("weight", w);
  if (t.dim() != 1 || t.size(0) != x.size(1) || t.device() != x.device())
    refuse("weight: a tensor of " + std::to_string(x.size(1)) + " elements on " + x.device().str() + " is wanted");
  if (t.scalar_type() != x.scalar_type() && t.scalar_type() != at::kFloat)
    refuse(std::string("weight: ") + c10::toString(t.scalar_type()) + ", wanted " + c10::toString(x.scalar_type()) + " or float32");
  if (t.size(0) > 1 && t.stride(0) != 1) refuse("weight: unit stride is wanted");
  return {t.data_ptr(), type_code(t.scalar_type())};
}

template <class Body>
PyObject* guarded(Py_ssize_t given_args, Py_ssize_t wanted, Body body) {
  try {
    if (given_args != wanted) {
      PyErr_Format(PyExc_TypeError, "%zd arguments, %zd wanted", given_args, wanted);
      throw Raised();
    }
    return body();
  } catch (const Raised&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// x, weight, residual, eps, total, out, e4m3 (False: an output of x's type), block (of e4m3 only)
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 8, [&]() -> PyObject* {
    const bool e4m3 = a[6] == Py_True;
    const long block = e4m3 ? integer(a[7]) : 0;
    const at::Tensor& x = tensor("x", a[0]);
    const Matrix mx = matrix("x", x);
    const auto [pw, wt] = weight_of(a[1], x);
    const double eps = number(a[3]);
    if (block != 0 && block != 128) refuse("block: " + std::to_string(block) + ", wanted 0 or 128");
    Matrix mr, mt, mo;
    at::Tensor total, out, scales;
    if (given(a[2])) {
      mr = matrix("residual", tensor("residual", a[2]), &x);
      total = given(a[4]) ? tensor("total", a[4]) : fresh(x.sizes(), x.scalar_type(), x.device());
      mt = matrix("total", total, &x);
    } else if (given(a[4])) {
      refuse("total goes with residual");
    }
    size_t lds = 0;
    if (e4m3) {
      out = fresh(x.sizes(), at::kFloat8_e4m3fn, x.device());
      lds = block ? (mx.cols + block - 1) / block : 1;
      scales = fresh({(int64_t)mx.rows, (int64_t)lds}, at::kFloat, x.device());
      mo.p = out.data_ptr();
      mo.ld = mx.cols;
    } else {
      out = given(a[5]) ? tensor("out", a[5]) : fresh(x.sizes(), x.scalar_type(), x.device());
      mo = matrix("out", out, &x);
    }
    const On on(x.device());
    check(without_gil([&] {
      return p_norm(mx.rows, mx.cols, mx.type, mx.p, mx.ld, mr.p, mr.ld, pw, wt, (float)eps, mt.p, mt.ld, e4m3 ? B2_DTYPE_E4M3 : mx.type, mo.p, mo.ld,
                    e4m3 ? static_cast<float*>(scales.data_ptr()) : nullptr, lds, block, on.stream);
    }));
    if (given(a[4])) changed(total);
    if (!e4m3 && given(a[5])) changed(out);
    if (!given(a[2])) return e4m3 ? Py_BuildValue("(NN)", wrap(out), wrap(scales)) : wrap(out);
    return e4m3 ? Py_BuildValue("(NNN)", wrap(out), wrap(scales), wrap(total)) : Py_BuildValue("(NN)", wrap(out), wrap(total));
  });
}

// dy, t, weight, dtotal, eps, dx
PyObject* norm_grad(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 6, [&]() -> PyObject* {
    const at::Tensor& dy = tensor("dy", a[0]);
    const Matrix md = matrix("dy", dy), mt = matrix("t", tensor("t", a[1]), &dy);
    const auto [pw, wt] = weight_of(a[2], dy);
    const Matrix mm = given(a[3]) ? matrix("dtotal", tensor("dtotal", a[3]), &dy) : Matrix();
    const double eps = number(a[4]);
    const at::Tensor dx = given(a[5]) ? tensor("dx", a[5]) : fresh(dy.sizes(), dy.scalar_type(), dy.device());
    const Matrix mx = matrix("dx", dx, &dy);
    at::Tensor dw;
    if (pw || given(a[2])) dw = fresh({(int64_t)md.cols}, wt == B2_DTYPE_F32 ? at::kFloat : at::kBFloat16, dy.device());
    size_t need = 0;
    check(p_norm_grad_workspace(md.rows, md.cols, md.type, &need));
    const On on(dy.device());
    const at::Tensor ws = workspace(need, dy.device());
    check(without_gil([&] {
      return p_norm_grad(md.rows, md.cols, md.type, md.p, md.ld, mt.p, mt.ld, mm.p, mm.ld, pw, wt, (float)eps, mx.p, mx.ld, dw.defined() ? dw.data_ptr() : nullptr,
                         ws.data_ptr(), ws.numel(), on.stream);
    }));
    if (given(a[5])) changed(dx);
    return dw.defined() ? Py_BuildValue("(NN)", wrap(dx), wrap(dw)) : wrap(dx);
  });
}

// Width and distance of rows of a tensor as b2_clip takes it: a matrix with gaps, or (elements, elements) where it lies in memory without gaps, whatever its order.
std::pair<size_t, size_t> rows_of(const char* list, size_t i, const at::Tensor& t) {
  const size_t n = t.numel();
  if (t.is_contiguous()) return {n, n};
  if (t.dim() == 2 && (t.size(1) == 1 || t.stride(1) == 1) && t.stride(0) >= t.size(1)) return {t.size(1), t.stride(0)};
  if (!t.is_non_overlapping_and_dense()) refuse(std::string(list) + "[" + std::to_string(i) + "]: neither dense nor a matrix with unit stride along its rows");
  return {n, n};
}
std::vector<at::Tensor> listed(const char* name, PyObject* x) {
  std::vector<at::Tensor> all;
  if (THPVariable_Check(x)) {
    all.push_back(THPVariable_Unpack(x));
    return all;
  }
  PyObject* fast = PySequence_Fast(x, "a tensor or a sequence of tensors is wanted");
  if (!fast) {
    if (PyErr_ExceptionMatches(PyExc_TypeError)) {
      PyErr_Clear();
      refuse(std::string(name) + ": a tensor or a sequence of tensors is wanted");
    }
    throw Raised();
  }
  struct Owner {
    PyObject* p;
    ~Owner() { Py_DECREF(p); }
  } owner{fast};
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
  all.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* item = PySequence_Fast_GET_ITEM(fast, i);
    if (!THPVariable_Check(item)) refuse(std::string(name) + ": tensors on one CUDA device are wanted");
    all.push_back(THPVariable_Unpack(item));
  }
  return all;
}

// tensors, max_norm, out
PyObject* clip(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 3, [&]() -> PyObject* {
    const std::vector<at::Tensor> xs = listed("tensors", a[0]);
    if (xs.empty()) refuse("tensors: none");
    const double limit = given(a[1]) ? number(a[1]) : std::numeric_limits<double>::infinity();
    if (!(limit >= 0.0)) refuse("max_norm: negative or not a number");
    const bool limited = limit <= std::numeric_limits<double>::max();
    // the same as any limit that fp32 has not: norms beyond it leave the values as they are
    const float most = std::numeric_limits<float>::max(), max_norm = !limited ? std::numeric_limits<float>::infinity() : limit < most ? (float)limit : most;
    const bool apart = given(a[2]);
    std::vector<at::Tensor> ys;
    if (apart) {
      ys = listed("out", a[2]);
      if (!limited) refuse("out goes with a limit");
      if (ys.size() != xs.size()) refuse("out: " + std::to_string(ys.size()) + " tensors for " + std::to_string(xs.size()));
    }
    const size_t n = xs.size();
    const c10::Device device = xs[0].device();
    std::vector<const void*> px(n);
    std::vector<void*> py(apart ? n : 0);
    std::vector<size_t> elements(n), widths(n), ldx(n), ldy(n);
    std::vector<int> types(n);
    bool dense = true;
    for (size_t i = 0; i < n; ++i) {
      const at::Tensor& x = xs[i];
      const auto at = [&](const char* list, const char* what) { refuse(std::string(list) + "[" + std::to_string(i) + "]: " + what); };
      if (!x.is_cuda() || x.device() != device) at("tensors", "on one CUDA device with the others is wanted");
      if ((types[i] = type_code(x.scalar_type())) < 0) at("tensors", "float32 or bfloat16 is wanted");
      px[i] = x.data_ptr();
      elements[i] = x.numel();
      const auto [wx, lx] = rows_of("tensors", i, x);
      size_t wy = wx, ly = lx;
      if (apart) {
        const at::Tensor& y = ys[i];
        if (y.device() != device || y.scalar_type() != x.scalar_type() || y.sizes() != x.sizes()) at("out", "device, type and shape like those of its tensor are wanted");
        std::tie(wy, ly) = rows_of("out", i, y);
        // a whole piece in another order than the other side's
        if (elements[i] > 1 && x.strides() != y.strides() && ((wx == elements[i] && !x.is_contiguous()) || (wy == elements[i] && !y.is_contiguous())))
          at("out", "elements lie in another order than in its tensor");
        py[i] = y.data_ptr();
      }
      widths[i] = wx < wy ? wx : wy;
      ldx[i] = wx == widths[i] ? lx : widths[i];
      ldy[i] = wy == widths[i] ? ly : widths[i];
      dense = dense && widths[i] == elements[i];
    }
    const at::Tensor norm = fresh({}, at::kFloat, device);
    size_t need = 0;
    check(p_clip_workspace(n, &need));
    const On on(device);
    const at::Tensor ws = workspace(need, device);
    check(without_gil([&] {
      return p_clip(n, px.data(), apart ? py.data() : nullptr, elements.data(), types.data(), dense ? nullptr : widths.data(), ldx.data(), ldy.data(),
                    max_norm, static_cast<float*>(norm.data_ptr()), ws.data_ptr(), ws.numel(), on.stream);
    }));
    if (limited)
      for (const at::Tensor& t : apart ? ys : xs) changed(t);
    return wrap(norm);
  });
}

// A number for all rows, or the address of one for each.
template <typename V>
const V* per_row(const char* name, PyObject* x, at::ScalarType type, const char* type_name, const at::Tensor& logits) {
  if (!THPVariable_Check(x)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(x);
  if (t.dim() != 1 || t.size(0) != logits.size(0) || t.scalar_type() != type || t.device() != logits.device() || (t.size(0) > 1 && t.stride(0) != 1))
    refuse(std::string(name) + ": a number, or a contiguous " + type_name + " tensor of " + std::to_string(logits.size(0)) + " on " + logits.device().str() + ", is wanted");
  return static_cast<const V*>(t.data_ptr());
}

// logits, u, temperature, top_k, top_p, min_p, logprob, out
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 8, [&]() -> PyObject* {
    const at::Tensor& logits = tensor("logits", a[0]);
    const Matrix m = matrix("logits", logits);
    const auto floats = [&](const char* name, PyObject* x) { return per_row<float>(name, x, at::kFloat, "float32", logits); };
    if (!THPVariable_Check(a[1])) refuse("u: a tensor is wanted");
    const float* u = floats("u", a[1]);
    b2_sample_options o{1.f, 0, 1.f, 0.f, floats("temperature", a[2]), per_row<int>("top_k", a[3], at::kInt, "int32", logits), floats("top_p", a[4]), floats("min_p", a[5])};
    if (!THPVariable_Check(a[2])) o.temperature = (float)number(a[2]);
    if (!THPVariable_Check(a[3])) {
      const long k = integer(a[3]);
      o.top_k = k < 0 ? 0 : k > std::numeric_limits<int>::max() ? std::numeric_limits<int>::max() : (int)k;
    }
    if (!THPVariable_Check(a[4])) o.top_p = (float)number(a[4]);
    if (!THPVariable_Check(a[5])) o.min_p = (float)number(a[5]);
    const int with_logprob = PyObject_IsTrue(a[6]);
    if (with_logprob < 0) throw Raised();
    at::Tensor out, logprob;
    if (given(a[7])) {
      out = tensor("out", a[7]);
      if (out.dim() != 1 || out.size(0) != (int64_t)m.rows || (out.scalar_type() != at::kLong && out.scalar_type() != at::kInt) || out.device() != logits.device() ||
          (m.rows > 1 && out.stride(0) != 1))
        refuse("out: a contiguous int64 or int32 tensor of " + std::to_string(m.rows) + " on " + logits.device().str() + " is wanted");
    } else {
      out = fresh({(int64_t)m.rows}, at::kLong, logits.device());
    }
    if (with_logprob) logprob = fresh({(int64_t)m.rows}, at::kFloat, logits.device());
    size_t need = 0;
    check(p_sample_workspace(m.rows, m.cols, &need));
    const On on(logits.device());
    const at::Tensor ws = workspace(need, logits.device());
    check(without_gil([&] {
      return p_sample(m.rows, m.cols, m.type, m.p, m.ld, u, &o, out.data_ptr(), out.scalar_type() == at::kLong ? 8 : 4,
                      with_logprob ? static_cast<float*>(logprob.data_ptr()) : nullptr, ws.data_ptr(), ws.numel(), on.stream);
    }));
    if (given(a[7])) changed(out);
    return with_logprob ? Py_BuildValue("(NN)", wrap(out), wrap(logprob)) : wrap(out);
  });
}

// addresses of the entries in the order below, and the class of errors that they return
PyObject* use(PyObject*, PyObject* args) {
  unsigned long long at[8];
  PyObject* cls;
  if (!PyArg_ParseTuple(args, "KKKKKKKKO", &at[0], &at[1], &at[2], &at[3], &at[4], &at[5], &at[6], &at[7], &cls)) return nullptr;
  p_norm = reinterpret_cast<decltype(p_norm)>(at[0]);
  p_norm_grad_workspace = reinterpret_cast<decltype(p_norm_grad_workspace)>(at[1]);
  p_norm_grad = reinterpret_cast<decltype(p_norm_grad)>(at[2]);
  p_clip_workspace = reinterpret_cast<decltype(p_clip_workspace)>(at[3]);
  p_clip = reinterpret_cast<decltype(p_clip)>(at[4]);
  p_sample_workspace = reinterpret_cast<decltype(p_sample_workspace)>(at[5]);
  p_sample = reinterpret_cast<decltype(p_sample)>(at[6]);
  p_last_error = reinterpret_cast<decltype(p_last_error)>(at[7]);
  Py_INCREF(cls);
  Py_XSETREF(error_class, cls);
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef methods[] = {{"use", use, METH_VARARGS, nullptr},         {"norm", FAST(norm), nullptr}, {"norm_grad", FAST(norm_grad), nullptr},
                         {"clip", FAST(clip), nullptr}, {"sample", FAST(sample), nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_lm_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__lm_native() { return PyModule_Create(&module); }
