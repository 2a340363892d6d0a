// Torch binding of the 8-bit decoder operators (include/vdexec_kernels.h): the
// Python module verdict_b200._torch_ops behind verdict_b200/ops.py.  Each
// function checks its tensors, allocates its outputs, enqueues one kernel on
// the current stream of the tensors' device and returns.
//
// In C++ because calls on single tokens are bound by the host: checks,
// allocations and the argument list took 6 to 16 us a call from Python, beside
// kernels of 2 to 5 us.

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "vdexec_kernels.h"

namespace {

using at::Tensor;
using at::ScalarType;

struct Refused {  // becomes a ValueError
  std::string what;
};
struct Failed {  // the library refused or failed: verdict_b200._abi.VdError
  int code;
  std::string what;
};
struct Raised {};  // a Python exception is set

[[noreturn]] void refuse(const std::string& what) { throw Refused{what}; }

std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

// Types as bits, to be combined; the codes of the C entries come out of code().
enum Types : unsigned { kF16 = 1, kBF16 = 2, kF32 = 4, kF8 = 8, kI32 = 16, kI64 = 32, kReal = kF16 | kBF16 | kF32 };

unsigned type_of(ScalarType t) {
  switch (t) {
    case ScalarType::Half: return kF16;
    case ScalarType::BFloat16: return kBF16;
    case ScalarType::Float: return kF32;
    case ScalarType::Float8_e4m3fn: return kF8;
    case ScalarType::Int: return kI32;
    case ScalarType::Long: return kI64;
    default: return 0;
  }
}
unsigned type_of(const Tensor& t) { return type_of(t.scalar_type()); }
int code(unsigned type) { return type == kF16 ? VDK_FP16 : type == kBF16 ? VDK_BF16 : type == kF32 ? VDK_FP32 : VDK_FP8; }
ScalarType scalar(int code) {
  return code == VDK_FP16   ? ScalarType::Half
         : code == VDK_BF16 ? ScalarType::BFloat16
         : code == VDK_FP32 ? ScalarType::Float
                            : ScalarType::Float8_e4m3fn;
}

const Tensor* optional(PyObject* o, const char* name) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor, got " + Py_TYPE(o)->tp_name);
  return &THPVariable_Unpack(o);
}
const Tensor& tensor(PyObject* o, const char* name) {
  const Tensor* t = optional(o, name);
  if (!t) refuse(std::string(name) + " must be a tensor, got NoneType");
  return *t;
}

// One argument: on a CUDA device (that of `like`), of one of the types, with
// `dims` dimensions and unit stride along the last (`packed`: contiguous).
void check(const Tensor& t, const char* name, int64_t dims, unsigned types, const Tensor* like = nullptr,
           bool packed = false) {
  const auto say = [&](const std::string& what) { refuse(std::string(name) + what); };
  if (!t.is_cuda()) say(" must be on a CUDA device");
  if (like && t.device() != like->device()) say(" is on " + t.device().str() + ", expected " + like->device().str());
  if (!(type_of(t) & types)) say(std::string(" has unsupported dtype ") + c10::toString(t.scalar_type()));
  if (t.dim() != dims) say(" must have " + std::to_string(dims) + " dimensions, got shape " + shape_of(t));
  if (t.is_neg()) say(" is a negated view: materialise it first (resolve_neg)");
  if (t.requires_grad() && c10::GradMode::is_enabled())
    say(" requires a gradient: this operator has no backward pass");
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined())
    say(" carries a forward-mode tangent: this operator has no derivative");
  if (!t.is_contiguous()) {
    if (packed) say(" must be contiguous");
    if (t.size(-1) > 1 && t.stride(-1) != 1) say(" needs unit stride along its last dimension");
  }
}

void expect(const Tensor& t, const char* name, at::IntArrayRef shape) {
  if (t.sizes() != shape) {
    std::string s;
    for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
    refuse(std::string(name) + " has shape " + shape_of(t) + ", expected (" + s + ")");
  }
}

void distinct_rows(const Tensor& t, const char* name) {
  if (t.size(0) > 1 && t.stride(0) < t.size(1)) refuse(std::string("rows of ") + name + " overlap");
}

int64_t blocks(int64_t n) { return (n + 127) / 128; }
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
// Row stride; a single row's is whatever its width needs (an 8-bit row's rounded up to 16 bytes).
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1); }
int64_t ld16(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : up16(t.size(1)); }

void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

// A tensor of the caller's was written: autograd and views saved for it see that.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor empty(at::IntArrayRef shape, ScalarType type, const Tensor& like) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(like.device()));
}

// An 8-bit matrix whose rows start on 16-byte boundaries, as fp8_linear takes it.
Tensor empty_f8(int64_t rows, int64_t cols, const Tensor& like) {
  const int64_t width = up16(cols);
  Tensor q = empty({rows, width}, ScalarType::Float8_e4m3fn, like);
  return width == cols ? q : q.narrow(1, 0, cols);
}

template <class F>
void run(const Tensor& like, F&& call) {
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != like.device().index()) guard.set_device(like.device());
  char err[512] = "";
  const int rc = call(c10::cuda::getCurrentCUDAStream(like.device().index()).stream(), err, sizeof(err));
  if (rc != VD_OK) throw Failed{rc, err};
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised();
  return v != 0;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* wrap(const Tensor* t) {
  if (t) return THPVariable_Wrap(*t);
  Py_RETURN_NONE;
}
template <class... T>
PyObject* tuple(const T&... t) {
  PyObject* items[] = {wrap(t)...};
  PyObject* r = PyTuple_New(sizeof...(T));
  for (size_t i = 0; i < sizeof...(T); ++i) {
    if (!items[i] || !r) {
      for (size_t j = i; j < sizeof...(T); ++j) Py_XDECREF(items[j]);
      Py_XDECREF(r);
      throw Raised();
    }
    PyTuple_SET_ITEM(r, i, items[i]);
  }
  return r;
}

// --- the operators: positional arguments as ops.py passes them -----------------

PyObject* quantize_fp8(PyObject* const* a) {  // x, gate, act
  const Tensor& x = tensor(a[0], "x");
  check(x, "x", 2, kReal);
  const Tensor* gate = optional(a[1], "gate");
  const int act = static_cast<int>(integer(a[2]));
  const int64_t rows = x.size(0), cols = x.size(1);
  if (gate) {
    check(*gate, "gate", 2, type_of(x), &x);
    expect(*gate, "gate", x.sizes());
  } else if (act != VDK_ACT_NONE) {
    refuse("an activation needs a gate");
  }
  if (cols < 1) refuse("x needs at least one column");
  Tensor q = empty_f8(rows, cols, x), scale = empty({rows, blocks(cols)}, ScalarType::Float, x);
  if (rows)
    run(x, [&](void* s, char* e, size_t n) {
      return vdk_quantize_fp8(ptr(x), ld(x), ptr(gate), gate ? ld(*gate) : 0, act, rows, cols, code(type_of(x)), ptr(q),
                              ld16(q), static_cast<float*>(ptr(scale)), blocks(cols), s, e, n);
    });
  return tuple(q, scale);
}

PyObject* quantize_fp8_weight(PyObject* const* a) {  // w
  const Tensor& w = tensor(a[0], "w");
  check(w, "w", 2, kReal);
  const int64_t rows = w.size(0), cols = w.size(1);
  if (rows < 1 || cols < 1) refuse("w needs at least one row and one column");
  Tensor q = empty_f8(rows, cols, w), scale = empty({blocks(rows), blocks(cols)}, ScalarType::Float, w);
  run(w, [&](void* s, char* e, size_t n) {
    return vdk_quantize_fp8_weight(ptr(w), ld(w), rows, cols, code(type_of(w)), ptr(q), ld16(q),
                                   static_cast<float*>(ptr(scale)), blocks(cols), s, e, n);
  });
  return tuple(q, scale);
}

PyObject* fp8_linear(PyObject* const* p) {  // a, a_scale, w, w_scale, bias, out type, out, status
  const Tensor &a = tensor(p[0], "a"), &sa = tensor(p[1], "a_scale"), &w = tensor(p[2], "w"), &sw = tensor(p[3], "w_scale");
  check(a, "a", 2, kF8);
  check(w, "w", 2, kF8, &a);
  const int64_t m = a.size(0), k = a.size(1), n = w.size(0), kb = blocks(k);
  if (w.size(1) != k) refuse("a has " + std::to_string(k) + " columns and w " + std::to_string(w.size(1)));
  if (k < 1 || n < 1) refuse("a and w need at least one column and w one row");
  check(sa, "a_scale", 2, kF32, &a);
  expect(sa, "a_scale", {m, kb});
  check(sw, "w_scale", 2, kF32, &a);
  expect(sw, "w_scale", {blocks(n), kb});
  const Tensor* bias = optional(p[4], "bias");
  if (bias) {
    check(*bias, "bias", 1, kF32, &a, true);
    expect(*bias, "bias", {n});
  }
  const int out_code = static_cast<int>(integer(p[5]));
  const Tensor* given = optional(p[6], "out");
  if (given) {
    check(*given, "out", 2, type_of(scalar(out_code)), &a);
    expect(*given, "out", {m, n});
    distinct_rows(*given, "out");
  }
  const Tensor out = given ? *given : empty({m, n}, scalar(out_code), a);
  const Tensor& status = tensor(p[7], "status");
  if (m)
    run(a, [&](void* s, char* e, size_t len) {
      return vdk_fp8_linear(ptr(a), ld16(a), static_cast<float*>(ptr(sa)), ld(sa), ptr(w), ld16(w),
                            static_cast<float*>(ptr(sw)), ld(sw), m, n, k, static_cast<float*>(ptr(bias)), ptr(out),
                            ld(out), out_code, static_cast<int*>(ptr(status)), s, e, len);
    });
  if (given) {
    if (m) written(*given);
    Py_INCREF(p[6]);
    return p[6];
  }
  return wrap(out);
}

// y, residual, post_gain, gate, residual_scale, block_scale, pre_gain, eps, plus_one, out type (-1: y's), in_place
PyObject* block_norm(PyObject* const* p) {
  const Tensor *y = optional(p[0], "y"), *h = optional(p[1], "residual"), *post = optional(p[2], "post_gain"),
               *gate = optional(p[3], "gate"), *pre = optional(p[6], "pre_gain");
  const double residual_scale = real(p[4]), block_scale = real(p[5]), eps = real(p[7]);
  const bool plus_one = truth(p[8]), in_place = truth(p[10]);
  int out_code = static_cast<int>(integer(p[9]));
  if (!y && !h) refuse("need y or a residual");
  const Tensor& x = y ? *y : *h;
  check(x, y ? "y" : "residual", 2, kReal);
  const int64_t rows = x.size(0), cols = x.size(1);
  if (cols < 1 || cols > VDK_NORM_MAX_COLS)
    refuse("rows have " + std::to_string(cols) + " columns, supported: 1 to " + std::to_string(VDK_NORM_MAX_COLS));
  if (h) {
    check(*h, "residual", 2, y ? kF32 | type_of(*y) : kReal, &x);
    expect(*h, "residual", x.sizes());
    distinct_rows(*h, "residual");
  } else if (in_place) {
    refuse("in_place needs a residual");
  }
  const unsigned h_type = h ? type_of(*h) : kF32, y_type = y ? type_of(*y) : h_type;
  if (post) {
    check(*post, "post_gain", 1, kF32, &x, true);
    expect(*post, "post_gain", {cols});
  }
  if (pre) {
    check(*pre, "pre_gain", 1, kF32, &x, true);
    expect(*pre, "pre_gain", {cols});
  }
  if (!y && (post || gate)) refuse("post_gain and gate need y");
  int64_t gate_row = 0, gate_col = 0;
  if (gate) {
    if (gate->dim() != 1 && gate->dim() != 2) refuse("gate must be a tensor of 1 or 2 dimensions");
    check(*gate, "gate", gate->dim(), kF32 | y_type, &x);
    const int64_t gr = gate->dim() == 2 ? gate->size(0) : 1, gc = gate->size(-1);
    if ((gr != 1 && gr != rows) || (gc != 1 && gc != cols))
      refuse("gate of shape " + shape_of(*gate) + " does not broadcast to " + shape_of(x));
    gate_row = gr > 1 ? gate->stride(0) : 0;
    gate_col = gc > 1 ? 1 : 0;
  }
  if (!pre && out_code >= 0) refuse("out_dtype needs pre_gain");
  if (out_code < 0) out_code = code(y_type);
  // Without a block output and with nothing to scale, the residual stays as it is.
  const bool keep = !y && h && residual_scale == 1.0;
  const Tensor fresh = keep || in_place ? *h : empty({rows, cols}, scalar(code(h_type)), x);
  Tensor z, scale;
  if (pre) {
    if (out_code == VDK_FP8) {
      z = empty_f8(rows, cols, x);
      scale = empty({rows, blocks(cols)}, ScalarType::Float, x);
    } else {
      z = empty({rows, cols}, scalar(out_code), x);
    }
  }
  if (rows && (pre || !keep))
    run(x, [&](void* s, char* e, size_t n) {
      return vdk_block_norm(ptr(y), y ? ld(*y) : 0, code(y_type), ptr(h), h ? ld(*h) : 0, code(h_type),
                            static_cast<float*>(ptr(post)), ptr(gate), gate ? code(type_of(*gate)) : 0, gate_row, gate_col,
                            static_cast<float>(residual_scale), static_cast<float>(block_scale),
                            static_cast<float*>(ptr(pre)), static_cast<float>(eps), plus_one, rows, cols,
                            keep ? nullptr : ptr(fresh), keep ? 0 : ld(fresh), pre ? ptr(z) : nullptr,
                            !pre ? 0 : out_code == VDK_FP8 ? ld16(z) : ld(z), pre ? out_code : 0,
                            scale.defined() ? static_cast<float*>(ptr(scale)) : nullptr, blocks(cols), s, e, n);
    });
  if (rows && in_place && !keep) written(*h);
  PyObject* residual;
  if (keep || in_place) {
    residual = p[1];
    Py_INCREF(residual);
  } else {
    residual = wrap(fresh);
  }
  PyObject* rest = tuple(z.defined() ? &z : nullptr, scale.defined() ? &scale : nullptr);
  PyObject* r = residual ? PyTuple_Pack(3, residual, PyTuple_GET_ITEM(rest, 0), PyTuple_GET_ITEM(rest, 1)) : nullptr;
  Py_DECREF(rest);
  Py_XDECREF(residual);
  if (!r) throw Raised();
  return r;
}

// q, k, positions, turns, head_dim, rotary_dim, interleaved, factor, inverse, q_out, k_out
PyObject* rotary(PyObject* const* p) {
  const Tensor *q = optional(p[0], "q"), *k = optional(p[1], "k");
  if (!q && !k) refuse("need q or k");
  const Tensor& x = q ? *q : *k;
  check(x, q ? "q" : "k", 3, kReal);
  const int64_t tokens = x.size(0);
  const Tensor& turns = tensor(p[3], "turns");
  if (turns.device() != x.device())
    refuse("the plan is on " + turns.device().str() + ", q and k on " + x.device().str());
  const int64_t head_dim = integer(p[4]), rotary_dim = integer(p[5]);
  const bool interleaved = truth(p[6]), inverse = truth(p[8]);
  const float factor = static_cast<float>(real(p[7]));
  Tensor outs[2];
  vdk_rotary_heads heads[2];
  const Tensor* ins[2] = {q, k};
  const char* names[2] = {"q", "k"};
  const char* out_names[2] = {"q_out", "k_out"};
  for (int i = 0; i < 2; ++i) {
    const Tensor* given = optional(p[9 + i], out_names[i]);
    if (!ins[i]) {
      if (given) refuse(std::string(out_names[i]) + " needs " + names[i]);
      continue;
    }
    const Tensor& t = *ins[i];
    check(t, names[i], 3, type_of(x), &x);
    if (t.size(0) != tokens)
      refuse("q has " + std::to_string(tokens) + " tokens and k " + std::to_string(t.size(0)));
    if (t.size(1) < 1) refuse(std::string(names[i]) + " has no heads");
    if (t.size(2) != head_dim)
      refuse(std::string(names[i]) + " has head_dim " + std::to_string(t.size(2)) + ", the plan " + std::to_string(head_dim));
    if (given) {
      check(*given, out_names[i], 3, type_of(x), &x);
      expect(*given, out_names[i], t.sizes());
    }
    outs[i] = given ? *given : empty(t.sizes(), t.scalar_type(), t);
    heads[i] = {ptr(t), ptr(outs[i]), t.stride(0), t.stride(1), outs[i].stride(0), outs[i].stride(1),
                static_cast<int32_t>(t.size(1))};
  }
  const void* positions = nullptr;
  int bits = 0;
  int64_t first = 0;
  if (PyLong_Check(p[2])) {
    first = integer(p[2]);
  } else {
    const Tensor& pos = tensor(p[2], "positions");
    check(pos, "positions", 1, kI32 | kI64, &x, true);
    if (pos.size(0) != tokens)
      refuse("positions has " + std::to_string(pos.size(0)) + " entries, expected " + std::to_string(tokens));
    positions = ptr(pos);
    bits = type_of(pos) == kI32 ? 32 : 64;
  }
  if (tokens)
    run(x, [&](void* s, char* e, size_t n) {
      return vdk_rotary(q ? &heads[0] : nullptr, k ? &heads[1] : nullptr, tokens, static_cast<int>(head_dim),
                        static_cast<int>(rotary_dim), code(type_of(x)), interleaved, inverse, positions, bits, first,
                        static_cast<const uint64_t*>(ptr(turns)), factor, s, e, n);
    });
  for (int i = 0; i < 2; ++i)
    if (tokens && ins[i] && p[9 + i] != Py_None) written(outs[i]);
  return tuple(q ? &outs[0] : nullptr, k ? &outs[1] : nullptr);
}

PyObject* token_logprobs(PyObject* const* p) {  // logits, ids, top, temperature
  const Tensor& x = tensor(p[0], "logits");
  check(x, "logits", 2, kReal);
  const Tensor* ids = optional(p[1], "ids");
  const int64_t rows = x.size(0), vocab = x.size(1), top = integer(p[2]);
  if (vocab < 1) refuse("logits need at least one column");
  if (top < 0 || top > VDK_LOGPROBS_MAX_TOP) refuse("top must be from 0 to " + std::to_string(VDK_LOGPROBS_MAX_TOP));
  int64_t n = 0;
  Tensor lp, top_ids, top_lp;
  if (ids) {
    if (ids->dim() != 1 && ids->dim() != 2) refuse("ids must be a tensor of 1 or 2 dimensions");
    check(*ids, "ids", ids->dim(), kI64, &x, true);
    if (ids->size(0) != rows)
      refuse("ids has " + std::to_string(ids->size(0)) + " rows, expected " + std::to_string(rows));
    n = ids->dim() == 2 ? ids->size(1) : 1;
    lp = empty(ids->sizes(), ScalarType::Float, x);
  }
  Tensor entropy = empty({rows}, ScalarType::Float, x), lse = empty({rows}, ScalarType::Float, x);
  if (top) {
    top_ids = empty({rows, top}, ScalarType::Int, x);
    top_lp = empty({rows, top}, ScalarType::Float, x);
  }
  const float temperature = static_cast<float>(real(p[3]));
  if (rows)
    run(x, [&](void* s, char* e, size_t len) {
      return vdk_token_logprobs(ptr(x), ld(x), rows, vocab, code(type_of(x)), temperature,
                                n ? static_cast<const int64_t*>(ptr(ids)) : nullptr, n, static_cast<int>(top),
                                n ? static_cast<float*>(ptr(lp)) : nullptr, static_cast<float*>(ptr(entropy)),
                                static_cast<float*>(ptr(lse)), top ? static_cast<int32_t*>(ptr(top_ids)) : nullptr,
                                top ? static_cast<float*>(ptr(top_lp)) : nullptr, s, e, len);
    });
  return tuple(lp.defined() ? &lp : nullptr, &entropy, &lse, top ? &top_ids : nullptr, top ? &top_lp : nullptr);
}

// Calls F with n arguments; nothing but a Python exception leaves it.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) noexcept {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what.c_str());
  } catch (const Failed& e) {
    PyObject* abi = PyImport_ImportModule("verdict_b200._abi");
    PyObject* error = abi ? PyObject_CallMethod(abi, "VdError", "is", e.code, e.what.c_str()) : nullptr;
    if (error) PyErr_SetObject(reinterpret_cast<PyObject*>(Py_TYPE(error)), error);
    Py_XDECREF(error);
    Py_XDECREF(abi);
  } catch (const Raised&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown error");
  }
  return nullptr;
}

#define ENTRY(name, n) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<name, n>)), METH_FASTCALL, nullptr }

PyMethodDef methods[] = {ENTRY(quantize_fp8, 3), ENTRY(quantize_fp8_weight, 1), ENTRY(fp8_linear, 8),
                         ENTRY(block_norm, 11),  ENTRY(rotary, 11),             ENTRY(token_logprobs, 4),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__torch_ops() { return PyModule_Create(&module); }
