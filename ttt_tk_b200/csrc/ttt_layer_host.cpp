// Host side of the layer-side sequence operators (`ttt_tk_b200.ssm`, the block end in `ttt_tk_b200.glue`): argument validation,
// the outputs and scratch, the C ABI's argument structs and the launch, in native code: decoding calls them for a token at a time.
//
// Plain CPython functions (METH_FASTCALL, positional arguments); a failed check raises ValueError, a failed launch RuntimeError.
// Shapes and types are checked before devices, so that every refusal but the last is the same without a GPU.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/ttt_mlp_b200.h"

namespace {

using at::Tensor;

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct PythonError {};

[[noreturn]] void refuse(const std::string& msg) { throw Refused(msg); }

std::string shape_text(at::IntArrayRef s) {
  std::string o = "[";
  for (size_t i = 0; i < s.size(); ++i) o += (i ? ", " : "") + std::to_string(s[i]);
  return o + "]";
}

int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonError();
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);      // (a tensor of several values is neither)
  if (v < 0) throw PythonError();
  return v == 1;
}

// The tensors of a call: checked one by one against shape and type, their devices at the end.
class Call {
 public:
  explicit Call(const char* what) : what_(what) {}

  const Tensor* any(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(what_) + ": " + name + " must be a tensor");
    const Tensor& t = THPVariable_Unpack(o);
    if (count_ == kMost) throw std::runtime_error("too many tensors");
    seen_[count_] = &t;
    names_[count_++] = name;
    return &t;
  }
  // the tensor that sets the activations' type
  const Tensor* first(PyObject* o, const char* name, int64_t dims, const char* shape) {
    const Tensor* t = any(o, name);
    if (t->dim() != dims) refuse(std::string(what_) + ": " + name + " must be " + shape + ", got " + shape_text(t->sizes()));
    type_ = t->scalar_type();
    if (type_ != at::kBFloat16 && type_ != at::kHalf && type_ != at::kFloat)
      refuse(std::string(what_) + ": " + name + " must be bfloat16, float16 or float32");
    rows(*t, name);
    return t;
  }
  int dtype() const { return type_ == at::kBFloat16 ? TTT_B200_BF16 : type_ == at::kHalf ? TTT_B200_FP16 : TTT_B200_FP32; }
  at::ScalarType type() const { return type_; }

  const Tensor* shaped(PyObject* o, const char* name, at::ScalarType type, std::initializer_list<int64_t> want) {
    const Tensor* t = any(o, name);
    const at::IntArrayRef w(want.begin(), want.size());
    if (t->sizes() != w) refuse(std::string(what_) + ": " + name + " must be " + shape_text(w) + ", got " + shape_text(t->sizes()));
    if (t->scalar_type() != type)
      refuse(std::string(what_) + ": " + name + " must have type " + at::toString(type) + ", got " + at::toString(t->scalar_type()));
    return t;
  }
  // activations with any strides but the innermost
  const Tensor* act(PyObject* o, const char* name, std::initializer_list<int64_t> want) {
    const Tensor* t = shaped(o, name, type_, want);
    rows(*t, name);
    return t;
  }
  void* whole(PyObject* o, const char* name, at::ScalarType type, std::initializer_list<int64_t> want) {
    if (o == Py_None) return nullptr;
    const Tensor* t = shaped(o, name, type, want);
    if (!t->is_contiguous()) refuse(std::string(what_) + ": " + name + " must be contiguous");
    return t->data_ptr();
  }
  float* f32(PyObject* o, const char* name, std::initializer_list<int64_t> want) {
    return static_cast<float*>(whole(o, name, at::kFloat, want));
  }
  int32_t* i32(PyObject* o, const char* name, int64_t n) { return static_cast<int32_t*>(whole(o, name, at::kInt, {n})); }
  // a weight that has to be there
  float* weight(PyObject* o, const char* name, std::initializer_list<int64_t> want) {
    if (o == Py_None) refuse(std::string(what_) + ": " + name + " must be a tensor");
    return f32(o, name, want);
  }

  // all tensors seen are on one CUDA device
  c10::Device device() const {
    const c10::Device d = seen_[0]->device();
    for (int i = 0; i < count_; ++i) {
      if (!seen_[i]->is_cuda()) refuse(std::string(what_) + ": " + names_[i] + " must be a CUDA tensor");
      if (seen_[i]->device() != d) refuse(std::string(what_) + ": " + names_[i] + " must be on " + d.str());
    }
    return d;
  }
  void need(bool ok, const char* msg) const {
    if (!ok) refuse(std::string(what_) + ": " + msg);
  }
  void sized(int64_t v, const char* name) const {
    if (v > (1 << 30)) refuse(std::string(what_) + ": " + name + " is too large");
  }

 private:
  void rows(const Tensor& t, const char* name) const {
    if (t.size(-1) > 1 && t.stride(-1) != 1) refuse(std::string(what_) + ": the last dimension of " + name + " must be contiguous");
  }
  static constexpr int kMost = 20;
  const char* what_;
  const Tensor* seen_[kMost];
  const char* names_[kMost];
  int count_ = 0;
  at::ScalarType type_ = at::kFloat;
};

// a dimension of size one is never stepped over
int64_t step_of(const Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  PyObject* o = THPVariable_Wrap(t);
  if (!o) throw PythonError();
  return o;
}
PyObject* tuple_of(std::initializer_list<Tensor> ts) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!r) throw PythonError();
  Py_ssize_t i = 0;
  for (const Tensor& t : ts) {
    PyObject* o;
    try {
      o = wrap(t);
    } catch (...) {
      Py_DECREF(r);
      throw;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

template <class Args> void launch(int (*fn)(const Args*, void*), const Args& a, const c10::Device& dev) {
  if (fn(&a, at::cuda::getCurrentCUDAStream(dev.index()).stream()) != 0) throw std::runtime_error(ttt_b200_last_error());
}
Tensor scratch_of(uint64_t bytes, const c10::Device& dev) {
  return bytes ? at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(dev)) : Tensor();
}
template <class Args> void give(Args& a, const Tensor& scratch) {
  a.scratch = scratch.defined() ? scratch.data_ptr() : nullptr;
  a.scratch_bytes = scratch.defined() ? static_cast<uint64_t>(scratch.numel()) : 0;
}
// An output, from the allocator itself: at::empty takes 0.2 us longer (decoding has little else).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const c10::Device& dev) { return at::Tensor(at::detail::empty_cuda(sizes, type, dev, c10::nullopt)); }
// What a call has changed in place says so to autograd: a backward that kept it refuses then (inference tensors have no version).
void changed(PyObject* o) {
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }

template <class Fn> PyObject* guarded(const char* what, Py_ssize_t nargs, Py_ssize_t want, Fn fn) {
  if (nargs != want) {
    PyErr_Format(PyExc_TypeError, "%s: wrong number of arguments", what);
    return nullptr;
  }
  try {
    return fn();
  } catch (const PythonError&) {
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* kind = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (kind) PyErr_SetString(kind, e.what_without_backtrace());
    Py_XDECREF(kind);
    Py_XDECREF(torch);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "internal error");
  return nullptr;
}

// ---- short convolution ---------------------------------------------------------------------------------------------------
void conv_weights(Call& c, ttt_b200_conv_args& a, PyObject* w, PyObject* b) {
  c.need(THPVariable_Check(w) && THPVariable_Unpack(w).dim() == 2 && THPVariable_Unpack(w).size(1) >= 2 && THPVariable_Unpack(w).size(1) <= 4,
         "weight must be [D, K] with K = 2, 3 or 4");
  a.K = static_cast<int32_t>(THPVariable_Unpack(w).size(1));
  a.weight = c.weight(w, "weight", {a.D, a.K});
  a.bias = c.f32(b, "bias", {a.D});
}

// x [B, T, D] and what the forward and the backward share: v = weight, bias, activation, state, lengths, heads
void conv_inputs(Call& c, ttt_b200_conv_args& a, PyObject* x, PyObject* const* v) {
  const Tensor& t = *c.first(x, "x", 3, "[B, T, D]");
  for (int i = 0; i < 3; ++i) c.sized(t.size(i), "a dimension of x");
  a.B = static_cast<int32_t>(t.size(0));
  a.T = static_cast<int32_t>(t.size(1));
  a.D = static_cast<int32_t>(t.size(2));
  c.need(a.D >= 1, "x has no channels");
  a.x = t.data_ptr();
  a.x_stride[0] = step_of(t, 0);
  a.x_stride[1] = step_of(t, 1);
  a.dtype = c.dtype();
  conv_weights(c, a, v[0], v[1]);
  a.activation = static_cast<int32_t>(integer(v[2]));
  a.state = c.whole(v[3], "state", c.type(), {a.B, a.K - 1, a.D});
  a.lengths = c.i32(v[4], "lengths", a.B);
  a.heads = truth(v[5]);
  if (a.heads) c.need(a.D % 64 == 0 && a.T % 64 == 0, "heads need multiples of 64 channels and tokens");
}

// conv(x, weight, bias, activation, state, lengths, heads, want_state) -> (y, final state or None)
PyObject* conv(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("conv", nargs, 8, [&]() -> PyObject* {
    Call c("short_conv");
    ttt_b200_conv_args a = {};
    conv_inputs(c, a, v[0], v + 1);
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const auto opt = at::TensorOptions().dtype(c.type()).device(dev);
    const Tensor y = a.heads ? at::empty({a.B, a.D / 64, a.T / 64, 64, 64}, opt) : at::empty({a.B, a.T, a.D}, opt);
    Tensor end;
    const bool none = a.B == 0 || a.T == 0;
    if (truth(v[7])) {
      if (!none) end = at::empty({a.B, a.K - 1, a.D}, opt);
      else end = a.state ? THPVariable_Unpack(v[4]).detach().clone() : at::zeros({a.B, a.K - 1, a.D}, opt);
    }
    a.y = y.data_ptr();
    a.final_state = ptr(end);
    if (!none) launch(ttt_b200_short_conv, a, dev);
    return tuple_of({y, end});
  });
}

// conv_backward(grad_y, x, weight, bias, activation, state, lengths, heads, grad_final_state) -> (grad_x, grad_weight, grad_bias, grad_state)
PyObject* conv_backward(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("conv_backward", nargs, 9, [&]() -> PyObject* {
    Call c("short_conv_backward");
    ttt_b200_conv_args a = {};
    conv_inputs(c, a, v[1], v + 2);
    if (a.heads) {
      a.grad_y = c.whole(v[0], "grad_y", c.type(), {a.B, a.D / 64, a.T / 64, 64, 64});
      c.need(v[0] != Py_None, "grad_y must be a tensor");
    } else {
      const Tensor& g = *c.act(v[0], "grad_y", {a.B, a.T, a.D});
      a.grad_y = g.data_ptr();
      a.gy_stride[0] = step_of(g, 0);
      a.gy_stride[1] = step_of(g, 1);
    }
    a.grad_final_state = c.whole(v[8], "grad_final_state", c.type(), {a.B, a.K - 1, a.D});
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const auto opt = at::TensorOptions().dtype(c.type()).device(dev), f32 = opt.dtype(at::kFloat);
    const bool none = a.B == 0 || a.T == 0, st = v[5] != Py_None;
    if (none) {
      const Tensor gs = !st ? Tensor() : a.grad_final_state ? THPVariable_Unpack(v[8]).detach().clone() : at::zeros({a.B, a.K - 1, a.D}, opt);
      return tuple_of({at::empty({a.B, a.T, a.D}, opt), at::zeros({a.D, a.K}, f32), a.bias ? at::zeros({a.D}, f32) : Tensor(), gs});
    }
    const Tensor gx = at::empty({a.B, a.T, a.D}, opt), gw = at::empty({a.D, a.K}, f32);
    const Tensor gb = a.bias ? at::empty({a.D}, f32) : Tensor();
    const Tensor gs = st ? at::empty({a.B, a.K - 1, a.D}, opt) : Tensor();
    const Tensor scratch = scratch_of(ttt_b200_short_conv_scratch_bytes(&a), dev);
    a.grad_x = gx.data_ptr();
    a.grad_weight = fptr(gw);
    a.grad_bias = fptr(gb);
    a.grad_state = ptr(gs);
    give(a, scratch);
    launch(ttt_b200_short_conv_backward, a, dev);
    return tuple_of({gx, gw, gb, gs});
  });
}

// rows of a table of states, and the slots of the batch
int64_t table(Call& c, PyObject* state, int64_t dims, PyObject* slots, int64_t B) {
  c.need(THPVariable_Check(state) && THPVariable_Unpack(state).dim() == dims, "state has the wrong number of dimensions");
  const int64_t rows = THPVariable_Unpack(state).size(0);
  c.sized(rows, "the state");
  c.need(slots != Py_None || rows == B, "without slots the state must have a row for each row of x");
  c.need(slots == Py_None || rows >= 1 || B == 0, "the state has no rows");
  return rows;
}

// conv_step(x, state, weight, bias, activation, slots) -> y
PyObject* conv_step(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("conv_step", nargs, 6, [&]() -> PyObject* {
    Call c("short_conv_step");
    ttt_b200_conv_args a = {};
    const Tensor& t = *c.first(v[0], "x", 2, "[B, D]");
    for (int i = 0; i < 2; ++i) c.sized(t.size(i), "a dimension of x");
    a.B = static_cast<int32_t>(t.size(0));
    a.T = 1;
    a.D = static_cast<int32_t>(t.size(1));
    c.need(a.D >= 1, "x has no channels");
    a.x = t.data_ptr();
    a.x_stride[0] = step_of(t, 0);
    a.dtype = c.dtype();
    conv_weights(c, a, v[2], v[3]);
    a.activation = static_cast<int32_t>(integer(v[4]));
    a.rows = static_cast<int32_t>(table(c, v[1], 3, v[5], a.B));
    a.state_io = c.whole(v[1], "state", c.type(), {a.rows, a.K - 1, a.D});
    a.slots = c.i32(v[5], "slots", a.B);
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor y = at::empty({a.B, a.D}, t.options());
    a.y = y.data_ptr();
    if (a.B > 0) {
      launch(ttt_b200_short_conv_step, a, dev);
      changed(v[1]);
    }
    return wrap(y);
  });
}

// ---- state space scan ------------------------------------------------------------------------------------------------------
// v = x, dt, A, B, C, D, dt_bias, softplus; a step has no tokens' dimension
void scan_inputs(Call& c, ttt_b200_scan_args& a, PyObject* const* v, bool step) {
  const Tensor& x = *c.first(v[0], "x", step ? 2 : 3, step ? "[B, D]" : "[B, T, D]");
  for (int64_t i = 0; i < x.dim(); ++i) c.sized(x.size(i), "a dimension of x");
  a.B = static_cast<int32_t>(x.size(0));
  a.T = step ? 1 : static_cast<int32_t>(x.size(1));
  a.D = static_cast<int32_t>(x.size(-1));
  c.need(a.D >= 1, "x has no channels");
  a.dtype = c.dtype();
  c.need(THPVariable_Check(v[2]) && THPVariable_Unpack(v[2]).dim() == 2, "A must be [D, N]");
  const int64_t N = THPVariable_Unpack(v[2]).size(1);
  c.need(N >= 1 && N <= 64, "A must have 1 to 64 states");
  a.N = static_cast<int32_t>(N);
  a.A = c.weight(v[2], "A", {a.D, a.N});
  c.need(THPVariable_Check(v[3]) && THPVariable_Unpack(v[3]).dim() == x.dim() + 1, step ? "B must be [B, G, N]" : "B must be [B, T, G, N]");
  const int64_t G = THPVariable_Unpack(v[3]).size(-2);
  c.need(G >= 1 && G <= a.D && a.D % G == 0, "the groups of B and C must divide the channels");
  a.G = static_cast<int32_t>(G);
  const Tensor *dt, *b, *cc;
  if (step) {
    dt = c.act(v[1], "dt", {a.B, a.D});
    b = c.act(v[3], "B", {a.B, a.G, a.N});
    cc = c.act(v[4], "C", {a.B, a.G, a.N});
  } else {
    dt = c.act(v[1], "dt", {a.B, a.T, a.D});
    b = c.act(v[3], "B", {a.B, a.T, a.G, a.N});
    cc = c.act(v[4], "C", {a.B, a.T, a.G, a.N});
  }
  a.x = x.data_ptr();
  a.dt = dt->data_ptr();
  a.Bm = b->data_ptr();
  a.Cm = cc->data_ptr();
  a.x_stride[0] = step_of(x, 0);
  a.dt_stride[0] = step_of(*dt, 0);
  a.B_stride[0] = step_of(*b, 0);
  a.C_stride[0] = step_of(*cc, 0);
  a.B_stride[2] = step_of(*b, -2);
  a.C_stride[2] = step_of(*cc, -2);
  if (!step) {
    a.x_stride[1] = step_of(x, 1);
    a.dt_stride[1] = step_of(*dt, 1);
    a.B_stride[1] = step_of(*b, 1);
    a.C_stride[1] = step_of(*cc, 1);
  }
  a.Dskip = c.f32(v[5], "D", {a.D});
  a.dt_bias = c.f32(v[6], "dt_bias", {a.D});
  a.softplus = truth(v[7]);
}

int64_t checkpoints_of(const ttt_b200_scan_args& a) { return (static_cast<int64_t>(a.T) + TTT_B200_SCAN_INTERVAL - 1) / TTT_B200_SCAN_INTERVAL; }

// scan(x, dt, A, B, C, D, dt_bias, softplus, state, lengths, want_state, want_checkpoints) -> (y, final state or None, checkpoints or None)
PyObject* scan(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("scan", nargs, 12, [&]() -> PyObject* {
    Call c("ssm_scan");
    ttt_b200_scan_args a = {};
    scan_inputs(c, a, v, false);
    a.state = c.f32(v[8], "state", {a.B, a.D, a.N});
    a.lengths = c.i32(v[9], "lengths", a.B);
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const auto opt = at::TensorOptions().dtype(c.type()).device(dev), f32 = opt.dtype(at::kFloat);
    const bool none = a.B == 0 || a.T == 0;
    const Tensor y = at::empty({a.B, a.T, a.D}, opt);
    Tensor end, ck;
    if (truth(v[10])) {
      if (!none) end = at::empty({a.B, a.D, a.N}, f32);
      else end = a.state ? THPVariable_Unpack(v[8]).detach().clone() : at::zeros({a.B, a.D, a.N}, f32);
    }
    if (truth(v[11])) ck = at::empty({a.B, checkpoints_of(a), a.D, a.N}, f32);
    if (!none) {
      const Tensor scratch = scratch_of(ttt_b200_ssm_scan_scratch_bytes(&a, 0), dev);
      give(a, scratch);
      a.y = y.data_ptr();
      a.final_state = fptr(end);
      a.checkpoints = fptr(ck);
      launch(ttt_b200_ssm_scan, a, dev);
    }
    return tuple_of({y, end, ck});
  });
}

// scan_backward(grad_y, x, dt, A, B, C, D, dt_bias, softplus, checkpoints, lengths, grad_final_state)
//   -> (grad_x, grad_dt, grad_A, grad_B, grad_C, grad_D, grad_dt_bias, grad_state)
PyObject* scan_backward(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("scan_backward", nargs, 12, [&]() -> PyObject* {
    Call c("ssm_scan_backward");
    ttt_b200_scan_args a = {};
    scan_inputs(c, a, v + 1, false);
    const Tensor& g = *c.act(v[0], "grad_y", {a.B, a.T, a.D});
    a.grad_y = g.data_ptr();
    a.gy_stride[0] = step_of(g, 0);
    a.gy_stride[1] = step_of(g, 1);
    a.checkpoints = c.weight(v[9], "checkpoints", {a.B, checkpoints_of(a), a.D, a.N});
    a.lengths = c.i32(v[10], "lengths", a.B);
    a.grad_final_state = c.f32(v[11], "grad_final_state", {a.B, a.D, a.N});
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const auto opt = at::TensorOptions().dtype(c.type()).device(dev), f32 = opt.dtype(at::kFloat);
    const bool none = a.B == 0 || a.T == 0;
    auto sum = [&](at::IntArrayRef s) { return none ? at::zeros(s, f32) : at::empty(s, f32); };
    const Tensor gx = at::empty({a.B, a.T, a.D}, opt), gdt = at::empty({a.B, a.T, a.D}, opt), gA = sum({a.D, a.N});
    const Tensor gB = at::empty({a.B, a.T, a.G, a.N}, opt), gC = at::empty({a.B, a.T, a.G, a.N}, opt);
    const Tensor gD = a.Dskip ? sum({a.D}) : Tensor(), gb = a.dt_bias ? sum({a.D}) : Tensor();
    Tensor gs;
    if (none) {
      gs = a.grad_final_state ? THPVariable_Unpack(v[11]).detach().clone() : at::zeros({a.B, a.D, a.N}, f32);
    } else {
      gs = at::empty({a.B, a.D, a.N}, f32);
      const Tensor scratch = scratch_of(ttt_b200_ssm_scan_scratch_bytes(&a, 1), dev);
      give(a, scratch);
      a.grad_x = gx.data_ptr();
      a.grad_dt = gdt.data_ptr();
      a.grad_A = fptr(gA);
      a.grad_B = gB.data_ptr();
      a.grad_C = gC.data_ptr();
      a.grad_D = fptr(gD);
      a.grad_dt_bias = fptr(gb);
      a.grad_state = fptr(gs);
      launch(ttt_b200_ssm_scan_backward, a, dev);
    }
    return tuple_of({gx, gdt, gA, gB, gC, gD, gb, gs});
  });
}

// scan_step(x, dt, A, B, C, D, dt_bias, softplus, state, slots) -> y
PyObject* scan_step(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("scan_step", nargs, 10, [&]() -> PyObject* {
    Call c("ssm_scan_step");
    ttt_b200_scan_args a = {};
    scan_inputs(c, a, v, true);
    a.rows = static_cast<int32_t>(table(c, v[8], 3, v[9], a.B));
    a.state_io = c.f32(v[8], "state", {a.rows, a.D, a.N});
    a.slots = c.i32(v[9], "slots", a.B);
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor y = at::empty({a.B, a.D}, at::TensorOptions().dtype(c.type()).device(dev));
    a.y = y.data_ptr();
    if (a.B > 0) {
      launch(ttt_b200_ssm_scan_step, a, dev);
      changed(v[8]);
    }
    return wrap(y);
  });
}

// ---- gated linear recurrence -------------------------------------------------------------------------------------------------
int64_t gated_checkpoints_of(const ttt_b200_gated_args& a) { return (static_cast<int64_t>(a.T) + TTT_B200_GATED_INTERVAL - 1) / TTT_B200_GATED_INTERVAL; }

void gated_weights(Call& c, ttt_b200_gated_args& a, PyObject* A, PyObject* gate_bias, PyObject* input_bias, PyObject* mix, bool gated) {
  a.A = c.f32(A, "A", {a.D});
  a.gate_bias = c.f32(gate_bias, "gate_bias", {a.D});
  a.input_bias = c.f32(input_bias, "input_bias", {a.D});
  c.need(gated || !a.input_bias, "input_bias needs input_gate");
  a.mix = static_cast<int32_t>(integer(mix));
}

// v = x, gate, A, input_gate, gate_bias, input_bias, mix; a step has no tokens' dimension
void gated_inputs(Call& c, ttt_b200_gated_args& a, PyObject* const* v, bool step) {
  const Tensor& x = *c.first(v[0], "x", step ? 2 : 3, step ? "[B, D]" : "[B, T, D]");
  for (int64_t i = 0; i < x.dim(); ++i) c.sized(x.size(i), "a dimension of x");
  a.B = static_cast<int32_t>(x.size(0));
  a.T = step ? 1 : static_cast<int32_t>(x.size(1));
  a.D = static_cast<int32_t>(x.size(-1));
  c.need(a.D >= 1, "x has no channels");
  a.dtype = c.dtype();
  auto rows = [&](const Tensor& t, const void*& p, int64_t* stride) {
    p = t.data_ptr();
    stride[0] = step_of(t, 0);
    if (!step) stride[1] = step_of(t, 1);
  };
  auto like = [&](PyObject* o, const char* name) -> const Tensor& { return step ? *c.act(o, name, {a.B, a.D}) : *c.act(o, name, {a.B, a.T, a.D}); };
  rows(x, a.x, a.x_stride);
  rows(like(v[1], "gate"), a.gate, a.gate_stride);
  if (v[3] != Py_None) rows(like(v[3], "input_gate"), a.input_gate, a.input_stride);
  gated_weights(c, a, v[2], v[4], v[5], v[6], v[3] != Py_None);
}

// gated(x, gate, A, input_gate, gate_bias, input_bias, mix, state, lengths, want_state, want_checkpoints) -> (y, final state or None, checkpoints or None)
PyObject* gated(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("gated", nargs, 11, [&]() -> PyObject* {
    Call c("gated_scan");
    ttt_b200_gated_args a = {};
    gated_inputs(c, a, v, false);
    a.state = c.f32(v[7], "state", {a.B, a.D});
    a.lengths = c.i32(v[8], "lengths", a.B);
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const auto opt = at::TensorOptions().dtype(c.type()).device(dev), f32 = opt.dtype(at::kFloat);
    const bool none = a.B == 0 || a.T == 0;
    const Tensor y = fresh({a.B, a.T, a.D}, c.type(), dev);
    Tensor end, ck;
    if (truth(v[9])) {
      if (!none) end = fresh({a.B, a.D}, at::kFloat, dev);
      else end = a.state ? THPVariable_Unpack(v[7]).detach().clone() : at::zeros({a.B, a.D}, f32);
    }
    if (truth(v[10])) ck = fresh({a.B, gated_checkpoints_of(a), a.D}, at::kFloat, dev);
    a.y = y.data_ptr();
    a.final_state = fptr(end);
    a.checkpoints = fptr(ck);
    if (!none) {
      const Tensor scratch = scratch_of(ttt_b200_gated_scan_scratch_bytes(&a, 0), dev);
      give(a, scratch);
      launch(ttt_b200_gated_scan, a, dev);
    }
    return tuple_of({y, end, ck});
  });
}

// 8-bit values of a backward pass, as (values, scales); the first of a call sets the group
const Tensor& kept(Call& c, ttt_b200_gated_args& a, PyObject* o, const char* name, const void*& p, int64_t* stride, const float*& scales) {
  const std::string n = name;
  c.need(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 2, (n + " must be (values, scales), as the other inputs").c_str());
  const Tensor& q = *c.shaped(PyTuple_GET_ITEM(o, 0), name, at::kFloat8_e4m3fn, {a.B, a.T, a.D});
  const Tensor& s = *c.any(PyTuple_GET_ITEM(o, 1), name);
  c.need(q.is_contiguous() && s.is_contiguous(), (n + "'s values and scales must be contiguous").c_str());
  int group = 0;
  for (const int g : {32, 64, 128})
    if (s.dim() == 3 && s.size(0) == a.B && s.size(1) == a.T && s.size(2) == (a.D + g - 1) / g && (!a.group || a.group == g)) group = g;
  c.need(group && s.scalar_type() == at::kFloat, (n + "'s scales must be float32 [B, T, D / group], group 32, 64 or 128 and the same for all inputs").c_str());
  a.group = group;
  p = q.data_ptr();
  scales = static_cast<const float*>(s.data_ptr());
  stride[0] = static_cast<int64_t>(a.T) * a.D;
  stride[1] = a.D;
  return q;
}

// gated_backward(grad_y, x, gate, checkpoints, A, input_gate, gate_bias, input_bias, mix, lengths, grad_final_state)
//   -> (grad_x, grad_gate, grad_A, grad_input_gate, grad_gate_bias, grad_input_bias, grad_state); x and the gates may be (values, scales) in 8 bits
PyObject* gated_backward(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("gated_backward", nargs, 11, [&]() -> PyObject* {
    Call c("gated_scan_backward");
    ttt_b200_gated_args a = {};
    const Tensor* g;
    if (PyTuple_Check(v[1])) {
      g = c.first(v[0], "grad_y", 3, "[B, T, D]");
      for (int i = 0; i < 3; ++i) c.sized(g->size(i), "a dimension of grad_y");
      a.B = static_cast<int32_t>(g->size(0));
      a.T = static_cast<int32_t>(g->size(1));
      a.D = static_cast<int32_t>(g->size(2));
      c.need(a.D >= 1, "grad_y has no channels");
      a.dtype = c.dtype();
      kept(c, a, v[1], "x", a.x, a.x_stride, a.x_scales);
      kept(c, a, v[2], "gate", a.gate, a.gate_stride, a.gate_scales);
      if (v[5] != Py_None) kept(c, a, v[5], "input_gate", a.input_gate, a.input_stride, a.input_scales);
      gated_weights(c, a, v[4], v[6], v[7], v[8], v[5] != Py_None);
    } else {
      PyObject* const in[] = {v[1], v[2], v[4], v[5], v[6], v[7], v[8]};
      gated_inputs(c, a, in, false);
      g = c.act(v[0], "grad_y", {a.B, a.T, a.D});
    }
    a.grad_y = g->data_ptr();
    a.gy_stride[0] = step_of(*g, 0);
    a.gy_stride[1] = step_of(*g, 1);
    a.checkpoints = c.weight(v[3], "checkpoints", {a.B, gated_checkpoints_of(a), a.D});
    a.lengths = c.i32(v[9], "lengths", a.B);
    a.grad_final_state = c.f32(v[10], "grad_final_state", {a.B, a.D});
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const auto opt = at::TensorOptions().dtype(c.type()).device(dev), f32 = opt.dtype(at::kFloat);
    const bool none = a.B == 0 || a.T == 0;
    auto sum = [&](const float* w) { return !w ? Tensor() : none ? at::zeros({a.D}, f32) : fresh({a.D}, at::kFloat, dev); };
    const Tensor gx = fresh({a.B, a.T, a.D}, c.type(), dev), gg = fresh({a.B, a.T, a.D}, c.type(), dev);
    const Tensor gi = v[5] != Py_None ? fresh({a.B, a.T, a.D}, c.type(), dev) : Tensor();
    const Tensor gA = sum(a.A), gb = sum(a.gate_bias), gib = sum(a.input_bias);
    Tensor gs;
    if (none) {
      gs = a.grad_final_state ? THPVariable_Unpack(v[10]).detach().clone() : at::zeros({a.B, a.D}, f32);
    } else {
      gs = fresh({a.B, a.D}, at::kFloat, dev);
      const Tensor scratch = scratch_of(ttt_b200_gated_scan_scratch_bytes(&a, 1), dev);
      give(a, scratch);
      a.grad_x = gx.data_ptr();
      a.grad_gate = gg.data_ptr();
      a.grad_input = ptr(gi);
      a.grad_A = fptr(gA);
      a.grad_gate_bias = fptr(gb);
      a.grad_input_bias = fptr(gib);
      a.grad_state = fptr(gs);
      launch(ttt_b200_gated_scan_backward, a, dev);
    }
    return tuple_of({gx, gg, gA, gi, gb, gib, gs});
  });
}

// gated_step(x, gate, A, input_gate, gate_bias, input_bias, mix, state, slots) -> y
PyObject* gated_step(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("gated_step", nargs, 9, [&]() -> PyObject* {
    Call c("gated_scan_step");
    ttt_b200_gated_args a = {};
    gated_inputs(c, a, v, true);
    a.rows = static_cast<int32_t>(table(c, v[7], 2, v[8], a.B));
    a.state_io = c.f32(v[7], "state", {a.rows, a.D});
    a.slots = c.i32(v[8], "slots", a.B);
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor y = fresh({a.B, a.D}, c.type(), dev);
    a.y = y.data_ptr();
    if (a.B > 0) {
      launch(ttt_b200_gated_scan_step, a, dev);
      changed(v[7]);
    }
    return wrap(y);
  });
}

// ---- block end -------------------------------------------------------------------------------------------------------------
// rows [..., D] that are one after another at a fixed distance: that distance
int64_t row_stride(const Call& c, const Tensor& t, const char* msg) {
  if (t.numel() == 0) return 0;
  int64_t stride = 0, below = 1;      // `below`: tokens of the dimensions further in
  for (int64_t i = t.dim() - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (below == 1) stride = t.stride(i);
    else c.need(t.stride(i) == stride * below, msg);
    below *= t.size(i);
  }
  return stride;
}

// v = residual, gate, layer, activation, post_weight, post_bias, scale, pre_weight, pre_bias, eps
const Tensor& block_inputs(Call& c, ttt_b200_block_args& a, PyObject* o, PyObject* const* v) {
  const Tensor& t = *c.any(o, "o");
  c.need(t.dim() >= 1, "o must be [..., D]");
  c.first(o, "o", t.dim(), "[..., D]");
  c.need(t.size(-1) >= 1 && t.size(-1) <= 8192, "o must have 1 to 8192 values to a token");
  a.D = static_cast<int32_t>(t.size(-1));
  a.M = t.numel() / a.D;
  a.dtype = c.dtype();
  const char* even = "the tokens of o, residual, gate and their gradients must be at a fixed distance";
  a.o = t.data_ptr();
  a.o_stride = row_stride(c, t, even);
  if (v[0] != Py_None) {
    const Tensor& r = *c.any(v[0], "residual");
    c.need(r.sizes() == t.sizes(), "residual must have the shape of o");
    c.need(r.scalar_type() == c.type() || r.scalar_type() == at::kFloat, "residual must have the type of o, or float32");
    c.need(r.size(-1) == 1 || r.stride(-1) == 1, "the last dimension of residual must be contiguous");
    a.residual_fp32 = r.scalar_type() == at::kFloat && c.type() != at::kFloat;
    a.residual = r.data_ptr();
    a.residual_stride = row_stride(c, r, even);
  }
  if (v[1] != Py_None) {
    const Tensor& g = *c.any(v[1], "gate");
    c.need(g.sizes() == t.sizes() && g.scalar_type() == c.type(), "gate must have the shape and type of o");
    c.need(g.size(-1) == 1 || g.stride(-1) == 1, "the last dimension of gate must be contiguous");
    a.gate = g.data_ptr();
    a.gate_stride = row_stride(c, g, even);
  }
  a.layer = truth(v[2]);
  a.activation = static_cast<int32_t>(integer(v[3]));
  a.post_weight = c.f32(v[4], "post_weight", {a.D});
  a.post_bias = c.f32(v[5], "post_bias", {a.D});
  a.scale = c.f32(v[6], "scale", {a.D});
  a.pre_weight = c.f32(v[7], "pre_weight", {a.D});
  a.pre_bias = c.f32(v[8], "pre_bias", {a.D});
  c.need(a.post_weight || !a.post_bias, "post_bias needs post_weight");
  c.need(a.pre_weight || !a.pre_bias, "pre_bias needs pre_weight");
  a.eps = static_cast<float>(PyFloat_AsDouble(v[9]));
  if (PyErr_Occurred()) {
    if (!PyErr_ExceptionMatches(PyExc_TypeError)) throw PythonError();
    PyErr_Clear();
    refuse("norm_gate_residual: eps must be a number");
  }
  c.need(a.eps >= 0.f, "eps must be >= 0");
  return t;
}

// block(o, the nine of block_inputs, eps, want_stats) -> (x, n or None, stats or None)
PyObject* block(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("block", nargs, 12, [&]() -> PyObject* {
    Call c("norm_gate_residual");
    ttt_b200_block_args a = {};
    const Tensor& o = block_inputs(c, a, v[0], v + 1);
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const auto opt = at::TensorOptions().dtype(c.type()).device(dev), f32 = opt.dtype(at::kFloat);
    const Tensor x = at::empty(o.sizes(), a.residual_fp32 ? f32 : opt);
    const Tensor n = a.pre_weight ? at::empty(o.sizes(), opt) : Tensor();
    const Tensor stats = truth(v[11]) ? at::empty({a.M, 4}, f32) : Tensor();
    a.x = x.data_ptr();
    a.n = ptr(n);
    a.stats = fptr(stats);
    if (a.M > 0) launch(ttt_b200_norm_gate_residual, a, dev);
    return tuple_of({x, n, stats});
  });
}

// block_backward(grad_x, grad_n, o, stats, the nine of block_inputs, eps)
//   -> (grad_o, grad_residual, grad_gate, grad_post_weight, grad_post_bias, grad_scale, grad_pre_weight, grad_pre_bias)
PyObject* block_backward(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("block_backward", nargs, 14, [&]() -> PyObject* {
    Call c("norm_gate_residual_backward");
    ttt_b200_block_args a = {};
    const Tensor& o = block_inputs(c, a, v[2], v + 4);
    a.stats = c.weight(v[3], "stats", {a.M, 4});
    const char* even = "the tokens of o, residual, gate and their gradients must be at a fixed distance";
    if (v[0] != Py_None) {
      const Tensor& g = *c.any(v[0], "grad_x");
      c.need(g.sizes() == o.sizes() && g.scalar_type() == (a.residual_fp32 ? at::kFloat : c.type()), "grad_x must have the shape and type of x");
      c.need(g.size(-1) == 1 || g.stride(-1) == 1, "the last dimension of grad_x must be contiguous");
      a.grad_x = g.data_ptr();
      a.gx_stride = row_stride(c, g, even);
    }
    if (v[1] != Py_None) {
      const Tensor& g = *c.any(v[1], "grad_n");
      c.need(a.pre_weight != nullptr, "grad_n needs pre_weight");
      c.need(g.sizes() == o.sizes() && g.scalar_type() == c.type(), "grad_n must have the shape and type of o");
      c.need(g.size(-1) == 1 || g.stride(-1) == 1, "the last dimension of grad_n must be contiguous");
      a.grad_n = g.data_ptr();
      a.gn_stride = row_stride(c, g, even);
    }
    c.need(a.grad_x || a.grad_n || a.M == 0, "grad_x or grad_n must be given");
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const auto opt = at::TensorOptions().dtype(c.type()).device(dev), f32 = opt.dtype(at::kFloat);
    auto sum = [&](const float* w) { return !w ? Tensor() : a.M ? at::empty({a.D}, f32) : at::zeros({a.D}, f32); };
    const Tensor go = at::empty(o.sizes(), opt), gr = a.residual ? at::empty(o.sizes(), a.residual_fp32 ? f32 : opt) : Tensor();
    const Tensor gg = a.gate ? at::empty(o.sizes(), opt) : Tensor();
    const Tensor g1 = sum(a.post_weight), gb1 = sum(a.post_bias), gsc = sum(a.scale), g2 = sum(a.pre_weight), gb2 = sum(a.pre_bias);
    a.grad_o = go.data_ptr();
    a.grad_residual = ptr(gr);
    a.grad_gate = ptr(gg);
    a.grad_post_weight = fptr(g1);
    a.grad_post_bias = fptr(gb1);
    a.grad_scale = fptr(gsc);
    a.grad_pre_weight = fptr(g2);
    a.grad_pre_bias = fptr(gb2);
    if (a.M > 0) {
      const Tensor scratch = scratch_of(ttt_b200_norm_gate_residual_scratch_bytes(&a), dev);
      give(a, scratch);
      launch(ttt_b200_norm_gate_residual_backward, a, dev);
    }
    return tuple_of({go, gr, gg, g1, gb1, gsc, g2, gb2});
  });
}

// ---- activations in 8 bits ---------------------------------------------------------------------------------------------------
std::vector<int64_t> scales_shape(const Tensor& t, int64_t group) {
  std::vector<int64_t> s(t.sizes().begin(), t.sizes().end());
  if (group) s.back() = (s.back() + group - 1) / group;
  else s.pop_back();
  return s;
}
int64_t group_of(const Call& c, PyObject* o) {
  const int64_t g = integer(o);
  c.need(g == 32 || g == 64 || g == 128, "group must be 32, 64 or 128");
  return g;
}
PyObject* pair_of(const Tensor& a, const Tensor& b) { return tuple_of({a, b}); }

// a list of what `one` makes for each of n
template <class Fn> PyObject* list_of(Py_ssize_t n, Fn one) {
  PyObject* r = PyList_New(n);
  if (!r) throw PythonError();
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o;
    try {
      o = one(i);
    } catch (...) {
      Py_DECREF(r);
      throw;
    }
    PyList_SET_ITEM(r, i, o);
  }
  return r;
}

// pack8(tuple of tensors, group, tuple of a clamp for each or None) -> [(values, scales), ...]
PyObject* pack8(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("pack8", nargs, 3, [&]() -> PyObject* {
    Call c("pack8");
    ttt_b200_pack8_args a = {};
    const Py_ssize_t n = PyTuple_GET_SIZE(v[0]);
    c.need(n >= 1 && n <= TTT_B200_PACK8_TENSORS, "one to four tensors");
    const int64_t group = group_of(c, v[1]);
    const Tensor* first = nullptr;
    for (Py_ssize_t k = 0; k < n; ++k) {
      const Tensor& t = *c.any(PyTuple_GET_ITEM(v[0], k), "a tensor");
      c.need(t.dim() >= 1, "tensors must be [..., D]");
      if (!first) {
        c.first(PyTuple_GET_ITEM(v[0], k), "a tensor", t.dim(), "[..., D]");
        first = &t;
      }
      c.need(t.sizes() == first->sizes() && t.scalar_type() == first->scalar_type(), "tensors of one call must share shape and type");
      c.need(t.size(-1) <= 1 || t.stride(-1) == 1, "the last dimension of a tensor must be contiguous");
      a.stride[k] = row_stride(c, t, "the rows of a tensor must be at a fixed distance");
      a.src[k] = t.data_ptr();
      if (v[2] != Py_None) a.clamp[k] = static_cast<int32_t>(integer(PyTuple_GET_ITEM(v[2], k)));
    }
    c.sized(first->size(-1), "a row");
    c.need(first->size(-1) >= 1, "rows have no values");
    a.D = static_cast<int32_t>(first->size(-1));
    a.M = first->numel() / a.D;
    a.dtype = c.dtype();
    a.group = static_cast<int32_t>(group);
    a.count = static_cast<int32_t>(n);
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const std::vector<int64_t> scaled = scales_shape(*first, group);
    Tensor q[TTT_B200_PACK8_TENSORS], s[TTT_B200_PACK8_TENSORS];
    for (Py_ssize_t k = 0; k < n; ++k) {
      q[k] = fresh(first->sizes(), at::kFloat8_e4m3fn, dev);
      s[k] = fresh(scaled, at::kFloat, dev);
      a.values[k] = q[k].data_ptr();
      a.scales[k] = fptr(s[k]);
    }
    if (a.M > 0) launch(ttt_b200_pack8, a, dev);
    return list_of(n, [&](Py_ssize_t k) { return pair_of(q[k], s[k]); });
  });
}

// unpack8(tuple of (values, scales), dtype code) -> [tensor, ...]
PyObject* unpack8(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("unpack8", nargs, 2, [&]() -> PyObject* {
    Call c("unpack8");
    ttt_b200_pack8_args a = {};
    const Py_ssize_t n = PyTuple_GET_SIZE(v[0]);
    c.need(n >= 1 && n <= TTT_B200_PACK8_TENSORS, "one to four pairs of values and scales");
    a.dtype = static_cast<int32_t>(integer(v[1]));
    const Tensor* first = nullptr;
    int group = -1;
    for (Py_ssize_t k = 0; k < n; ++k) {
      PyObject* o = PyTuple_GET_ITEM(v[0], k);
      c.need(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 2, "what is unpacked must be (values, scales)");
      const Tensor &q = *c.any(PyTuple_GET_ITEM(o, 0), "values"), &s = *c.any(PyTuple_GET_ITEM(o, 1), "scales");
      c.need(q.scalar_type() == at::kFloat8_e4m3fn && q.dim() >= 1 && q.is_contiguous(), "values must be contiguous float8_e4m3fn [..., D]");
      if (!first) first = &q;
      c.need(q.sizes() == first->sizes(), "values of one call must share their shape");
      int found = -1;
      for (const int g : {0, 32, 64, 128})
        if (s.sizes() == at::IntArrayRef(scales_shape(q, g)) && (group < 0 || group == g)) found = g;
      c.need(found >= 0 && s.scalar_type() == at::kFloat && s.is_contiguous(),
             "scales must be contiguous float32 [..., D / group], group 32, 64 or 128, or [...], and the same for all");
      group = found;
      a.values[k] = q.data_ptr();
      a.scales[k] = static_cast<float*>(s.data_ptr());
    }
    c.sized(first->size(-1), "a row");
    c.need(first->size(-1) >= 1, "rows have no values");
    a.D = static_cast<int32_t>(first->size(-1));
    a.M = first->numel() / a.D;
    a.group = group;
    a.count = static_cast<int32_t>(n);
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const at::ScalarType type = a.dtype == TTT_B200_BF16 ? at::kBFloat16 : a.dtype == TTT_B200_FP16 ? at::kHalf : at::kFloat;
    Tensor t[TTT_B200_PACK8_TENSORS];
    for (Py_ssize_t k = 0; k < n; ++k) {
      t[k] = fresh(first->sizes(), type, dev);
      a.dst[k] = t[k].data_ptr();
    }
    if (a.M > 0) launch(ttt_b200_unpack8, a, dev);
    return list_of(n, [&](Py_ssize_t k) { return wrap(t[k]); });
  });
}

// norm8(o, residual, weight, bias, layer, group or 0, eps, want_stats) -> (x, values, scales, stats or None)
PyObject* norm8(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("norm8", nargs, 8, [&]() -> PyObject* {
    Call c("norm_residual_8bit");
    ttt_b200_norm8_args a = {};
    const Tensor& o = *c.any(v[0], "o");
    c.need(o.dim() >= 1, "o must be [..., D]");
    c.first(v[0], "o", o.dim(), "[..., D]");
    c.need(o.size(-1) >= 1 && o.size(-1) <= 8192, "o must have 1 to 8192 values to a token");
    a.D = static_cast<int32_t>(o.size(-1));
    a.M = o.numel() / a.D;
    a.dtype = c.dtype();
    const char* even = "the tokens of o and residual must be at a fixed distance";
    a.o = o.data_ptr();
    a.o_stride = row_stride(c, o, even);
    const bool added = v[1] != Py_None;
    if (added) {
      const Tensor& r = *c.any(v[1], "residual");
      c.need(r.sizes() == o.sizes(), "residual must have the shape of o");
      c.need(r.scalar_type() == c.type() || r.scalar_type() == at::kFloat, "residual must have the type of o, or float32");
      c.need(r.size(-1) == 1 || r.stride(-1) == 1, "the last dimension of residual must be contiguous");
      a.residual_fp32 = r.scalar_type() == at::kFloat && c.type() != at::kFloat;
      a.residual = r.data_ptr();
      a.residual_stride = row_stride(c, r, even);
    }
    a.weight = c.weight(v[2], "weight", {a.D});
    a.bias = c.f32(v[3], "bias", {a.D});
    a.layer = truth(v[4]);
    const int64_t group = integer(v[5]);
    c.need(group == 0 || group == 32 || group == 64 || group == 128, "group must be 32, 64, 128 or None");
    a.group = static_cast<int32_t>(group);
    a.eps = static_cast<float>(PyFloat_AsDouble(v[6]));
    if (PyErr_Occurred()) {
      if (!PyErr_ExceptionMatches(PyExc_TypeError)) throw PythonError();
      PyErr_Clear();
      refuse("norm_residual_8bit: eps must be a number");
    }
    c.need(a.eps >= 0.f, "eps must be >= 0");
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor x = added ? fresh(o.sizes(), a.residual_fp32 ? at::kFloat : c.type(), dev) : o;
    const Tensor q = fresh(o.sizes(), at::kFloat8_e4m3fn, dev), s = fresh(scales_shape(o, group), at::kFloat, dev);
    const Tensor stats = truth(v[7]) ? fresh({a.M, 4}, at::kFloat, dev) : Tensor();
    a.x = added ? x.data_ptr() : nullptr;
    a.values = q.data_ptr();
    a.scales = fptr(s);
    a.stats = fptr(stats);
    if (a.M > 0) launch(ttt_b200_norm_residual_8bit, a, dev);
    return tuple_of({x, q, s, stats});
  });
}

// ---- rows of tables of states --------------------------------------------------------------------------------------------------
// v: a tuple of tables
int64_t tables_of(Call& c, ttt_b200_tables_args& a, PyObject* v) {
  const Py_ssize_t n = PyTuple_GET_SIZE(v);
  c.need(n >= 1 && n <= TTT_B200_TABLES, "1 to 16 tables");
  int64_t rows = -1;
  for (Py_ssize_t k = 0; k < n; ++k) {
    const Tensor& t = *c.any(PyTuple_GET_ITEM(v, k), "a table");
    c.need(t.dim() >= 1 && t.is_contiguous(), "a table must be contiguous and have rows");
    if (rows < 0) rows = t.size(0);
    c.need(t.size(0) == rows, "tables of one call must have as many rows");
    const int64_t bytes = rows ? t.numel() / rows * static_cast<int64_t>(t.element_size()) : 0;
    if (!bytes) continue;
    for (int j = 0; j < a.count; ++j) {
      const char *p = static_cast<char*>(t.data_ptr()), *q = static_cast<char*>(a.table[j]);
      c.need(p + rows * bytes <= q || q + rows * a.row_bytes[j] <= p, "tables of one call must not overlap");
    }
    a.table[a.count] = t.data_ptr();
    a.row_bytes[a.count++] = bytes;
  }
  c.sized(rows, "a table");
  a.rows = static_cast<int32_t>(rows);
  return rows;
}
void changed_tables(PyObject* v) {
  for (Py_ssize_t k = 0; k < PyTuple_GET_SIZE(v); ++k) changed(PyTuple_GET_ITEM(v, k));
}
// What names the rows is read by every block while others write.
void apart(const Call& c, const ttt_b200_tables_args& a, const Tensor& t, const char* name) {
  const char *p = static_cast<char*>(t.data_ptr()), *end = p + t.nbytes();
  for (int j = 0; j < a.count; ++j) {
    const char* q = static_cast<char*>(a.table[j]);
    c.need(end <= q || q + a.rows * a.row_bytes[j] <= p, (std::string(name) + " must not overlap a table").c_str());
  }
}
const int32_t* pairs_of(Call& c, ttt_b200_tables_args& a, PyObject* o, const char* name) {
  const Tensor& t = *c.any(o, name);
  c.need(t.dim() == 1 && t.scalar_type() == at::kInt && t.is_contiguous(), (std::string(name) + " must be contiguous int32 [n]").c_str());
  c.need(t.size(0) <= TTT_B200_TABLE_PAIRS, (std::string("at most 4096 rows in ") + name).c_str());
  a.pairs = static_cast<int32_t>(t.size(0));
  if (a.pairs) apart(c, a, t, name);
  return static_cast<const int32_t*>(t.data_ptr());
}

// copy_rows(tables, source, target)
PyObject* copy_rows(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("copy_rows", nargs, 3, [&]() -> PyObject* {
    Call c("copy_rows");
    ttt_b200_tables_args a = {};
    const int64_t rows = tables_of(c, a, v[0]);
    a.source = pairs_of(c, a, v[1], "source");
    const int32_t n = a.pairs;
    a.target = pairs_of(c, a, v[2], "target");
    c.need(a.pairs == n, "source and target must have as many rows");
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    if (rows && n && a.count) {
      launch(ttt_b200_copy_rows, a, dev);
      changed_tables(v[0]);
    }
    Py_RETURN_NONE;
  });
}

// clear_rows(tables, rows)
PyObject* clear_rows(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("clear_rows", nargs, 2, [&]() -> PyObject* {
    Call c("clear_rows");
    ttt_b200_tables_args a = {};
    const int64_t rows = tables_of(c, a, v[0]);
    a.target = pairs_of(c, a, v[1], "rows");
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    if (rows && a.pairs && a.count) {
      launch(ttt_b200_clear_rows, a, dev);
      changed_tables(v[0]);
    }
    Py_RETURN_NONE;
  });
}

// compact_rows(tables, used) -> place
PyObject* compact_rows(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  return guarded("compact_rows", nargs, 2, [&]() -> PyObject* {
    Call c("compact_rows");
    ttt_b200_tables_args a = {};
    const int64_t rows = tables_of(c, a, v[0]);
    const Tensor& used = *c.shaped(v[1], "used", at::kBool, {rows});
    c.need(used.is_contiguous(), "used must be contiguous");
    c.need(rows <= 8192, "at most 8192 rows");
    apart(c, a, used, "used");
    const c10::Device dev = c.device();
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor place = fresh({rows}, at::kInt, dev);
    a.used = static_cast<const uint8_t*>(used.data_ptr());
    a.place = static_cast<int32_t*>(place.data_ptr());
    if (rows) {
      launch(ttt_b200_compact_rows, a, dev);
      changed_tables(v[0]);
    }
    return wrap(place);
  });
}

#define TTT_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {TTT_METHOD(conv),          TTT_METHOD(conv_backward), TTT_METHOD(conv_step), TTT_METHOD(scan),
                          TTT_METHOD(scan_backward), TTT_METHOD(scan_step),     TTT_METHOD(block),     TTT_METHOD(block_backward),
                          TTT_METHOD(gated),         TTT_METHOD(gated_backward), TTT_METHOD(gated_step),
                          TTT_METHOD(pack8),         TTT_METHOD(unpack8),        TTT_METHOD(norm8),
                          TTT_METHOD(copy_rows),     TTT_METHOD(clear_rows),     TTT_METHOD(compact_rows),
                          {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_ttt_layer_host", "Validation and launch of the layer-side sequence operators.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ttt_layer_host() { return PyModule_Create(&kModule); }
