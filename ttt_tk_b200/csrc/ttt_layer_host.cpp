// Host side of the layer-side sequence operators (`ttt_tk_b200.ssm`, the block end in `ttt_tk_b200.glue`): argument validation,
// the outputs and scratch, the C ABI's argument structs and the launch, in native code: decoding calls them for a token at a time.
//
// Plain CPython functions (METH_FASTCALL, positional arguments); a failed check raises ValueError, a failed launch RuntimeError.
// Shapes and types are checked before devices, so that every refusal but the last is the same without a GPU.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <stdexcept>
#include <string>

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
  static constexpr int kMost = 16;
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
    if (a.B > 0) launch(ttt_b200_short_conv_step, a, dev);
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
    if (a.B > 0) launch(ttt_b200_ssm_scan_step, a, dev);
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

#define TTT_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {TTT_METHOD(conv),          TTT_METHOD(conv_backward), TTT_METHOD(conv_step), TTT_METHOD(scan),
                          TTT_METHOD(scan_backward), TTT_METHOD(scan_step),     TTT_METHOD(block),     TTT_METHOD(block_backward),
                          {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_ttt_layer_host", "Validation and launch of the layer-side sequence operators.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ttt_layer_host() { return PyModule_Create(&kModule); }
