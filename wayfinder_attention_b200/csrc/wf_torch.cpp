// fused_linear, layer_norm and token_logprobs as PyTorch calls: argument checks, outputs and
// autograd nodes around the C ABI (include/wayfinder.h), whose functions are looked up in the
// library that the package loads.  A small training step is bound by the host: the same nodes
// in Python took 118 us of host time for a layer norm's forward and backward, against 70 us
// of PyTorch's own.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/wayfinder.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
  decltype(&wf_last_error) last_error;
  decltype(&wf_linear) linear;
  decltype(&wf_linear_workspace_bytes) linear_workspace_bytes;
  decltype(&wf_linear_backward) linear_backward;
  decltype(&wf_linear_backward_workspace_bytes) linear_backward_workspace_bytes;
  decltype(&wf_layer_norm) layer_norm;
  decltype(&wf_layer_norm_backward) layer_norm_backward;
  decltype(&wf_layer_norm_backward_workspace_bytes) layer_norm_backward_workspace_bytes;
  decltype(&wf_max_top_tokens) max_top_tokens;
  decltype(&wf_token_logprobs) token_logprobs;
  decltype(&wf_token_logprobs_backward) token_logprobs_backward;
};
Library wf{};

// ValueError in Python; everything else that is thrown becomes RuntimeError.
struct BadValue : std::runtime_error {
  using std::runtime_error::runtime_error;
};

std::string shape_of(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + (s.size() == 1 ? ",)" : ")");
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return WF_DTYPE_BF16;
    case at::kHalf: return WF_DTYPE_F16;
    case at::kFloat: return WF_DTYPE_F32;
    default:
      throw BadValue(std::string("unsupported dtype ") + c10::toString(t) +
                     "; expected bfloat16, float16 or float32");
  }
}

void check(int rc) {
  if (rc == WF_OK) return;
  const std::string message = wf.last_error();
  if (rc == WF_ERR_INVALID_ARGUMENT || rc == WF_ERR_UNSUPPORTED) throw BadValue(message);
  throw std::runtime_error(message);
}

void check_devices(const Tensor& first, std::initializer_list<const Tensor*> others) {
  auto one = [&](const Tensor& t) {
    if (!t.is_cuda())
      throw std::runtime_error("wayfinder_attention_b200 runs on CUDA tensors only (no CPU fallback); got a tensor on " +
                               t.device().str());
    if (t.device() != first.device())
      throw BadValue("tensors on different devices: " + first.device().str() + " vs " + t.device().str());
  };
  one(first);
  for (const Tensor* t : others)
    if (t->defined()) one(*t);
}

// t as (rows, last axis) with unit-strided rows that do not overlap, copied only if it has to be.
Tensor rows_of(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  if ((r.stride(1) != 1 && r.size(1) > 1) || (r.stride(0) < r.size(1) && r.size(0) > 1)) r = r.contiguous();
  // one row (a transposed column is (1, d) with strides (1, 1)) or none: its stride is never taken
  if (r.size(0) <= 1 && r.stride(0) < r.size(1)) r = r.as_strided(r.sizes(), {r.size(1), 1});
  return r;
}
// What a node saves for rows_of(t): t itself where the rows are a view of it (a view made below the
// AutoDispatchBelowADInplaceOrView guard has a version of its own, and a change of t before the
// backward would go unnoticed), else the copy.  The backward takes the rows of it again.
const Tensor& to_save(const Tensor& t, const Tensor& rows) { return rows.is_alias_of(t) ? t : rows; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool on_16_bytes(const Tensor& rows) {
  return reinterpret_cast<uintptr_t>(rows.data_ptr()) % 16 == 0 && rows.stride(0) * rows.element_size() % 16 == 0;
}
Tensor bytes(size_t n, const Tensor& like) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
// Whether a node is needed.  A forward-mode dual has its tangent whatever it asks of the backward,
// and these operators have no formula for it.
bool wants_grad(std::initializer_list<const Tensor*> all) {
  for (const Tensor* t : all)
    if (t->defined() && t->_fw_grad(0).defined())
      throw std::runtime_error("this operator has no forward-mode derivative; got an input with a tangent");
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : all)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
using Optional = std::optional<Tensor>;
Optional given(const Tensor& t) { return t.defined() ? Optional(t) : std::nullopt; }
Tensor contiguous(const Optional& t) { return t ? t->contiguous() : Tensor(); }
// Whether the backward is asked for an optional input's gradient; an input that was not given
// has no edge, and the edges of the later ones move up: `edge` counts the given ones so far.
bool needs_optional(AutogradContext* ctx, const char* has, size_t& edge) {
  return ctx->saved_data[has].toBool() && ctx->needs_input_grad(edge++);
}
void once_only() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "this operator's backward is not differentiable (create_graph=True)");
}

// ------------------------------------------------------------------ linear
Tensor run_linear(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r, int act, at::IntArrayRef shape,
                  Tensor* z, void* status) {
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  const int code = dtype_code(x.scalar_type());
  Tensor y = at::empty(shape, x.options());
  if (z) *z = at::empty({M, (N + 7) / 8 * 8}, code == WF_DTYPE_F32 ? x.options() : x.options().dtype(at::kHalf));
  const size_t n = wf.linear_workspace_bytes(M, N, K, code, on_16_bytes(x), on_16_bytes(w));
  const Tensor ws = bytes(n, x);
  check(wf.linear(x.data_ptr(), w.data_ptr(), ptr(b), ptr(r), code, M, N, K, x.stride(0), w.stride(0),
                  r.defined() ? r.stride(0) : 0, act, z ? z->data_ptr() : nullptr, y.data_ptr(), ptr(ws), n,
                  static_cast<int32_t*>(status), stream()));
  return y;
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Optional& b, const Optional& r,
                        int64_t act, int64_t status) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto shape = x.sizes().vec();
    shape.back() = w.size(0);
    const Tensor x2 = rows_of(x), w2 = rows_of(w);
    Tensor z;
    Tensor y = run_linear(x2, w2, contiguous(b), r ? rows_of(*r) : Tensor(), (int)act, shape,
                          act ? &z : nullptr, reinterpret_cast<void*>(status));
    ctx->save_for_backward({to_save(x, x2), to_save(w, w2), z});
    ctx->saved_data["bias"] = b.has_value();
    ctx->saved_data["residual"] = r.has_value();
    ctx->saved_data["act"] = act;
    ctx->saved_data["status"] = status;
    ctx->saved_data["shape"] = x.sizes().vec();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once_only();
    const auto saved = ctx->get_saved_variables();
    const Tensor x = rows_of(saved[0]), w = rows_of(saved[1]), &z = saved[2], &dy = grads[0];
    const int64_t act = ctx->saved_data["act"].toInt();
    size_t edge = 2;
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_b = needs_optional(ctx, "bias", edge);
    const bool need_r = needs_optional(ctx, "residual", edge);
    Tensor dx, dw, db;
    if (need_x || need_w || need_b) {
      c10::cuda::CUDAGuard guard(x.device());
      const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
      const int code = dtype_code(x.scalar_type());
      const Tensor g = rows_of(dy);
      if (need_x) dx = at::empty(ctx->saved_data["shape"].toIntVector(), x.options());
      if (need_w) dw = at::empty({N, K}, x.options());
      if (need_b) db = at::empty({N}, x.options());
      const size_t n = wf.linear_backward_workspace_bytes(M, N, K, code, (int)act, on_16_bytes(x), on_16_bytes(w),
                                                          on_16_bytes(g));
      const Tensor ws = bytes(n, x);
      check(wf.linear_backward(x.data_ptr(), w.data_ptr(), ptr(z), g.data_ptr(), code, M, N, K, x.stride(0),
                               w.stride(0), g.stride(0), (int)act, ptr(dx), ptr(dw), ptr(db), ptr(ws), n,
                               reinterpret_cast<int32_t*>(ctx->saved_data["status"].toInt()), stream()));
    }
    return {dx, dw, db, need_r ? dy : Tensor(), Tensor(), Tensor()};
  }
};

Tensor fused_linear(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r, int act, void* status,
                    bool user_status) {
  if (x.dim() < 1 || w.dim() != 2 || x.size(-1) != w.size(1) || w.numel() == 0)
    throw BadValue("expected x (..., d_in) and weight (d_out, d_in) with widths >= 1, got " + shape_of(x.sizes()) +
                   " and " + shape_of(w.sizes()));
  auto shape = x.sizes().vec();
  shape.back() = w.size(0);
  if (b.defined() && (b.dim() != 1 || b.size(0) != w.size(0)))
    throw BadValue("bias " + shape_of(b.sizes()) + " does not match d_out=" + std::to_string(w.size(0)));
  if (r.defined() && r.sizes() != at::IntArrayRef(shape))
    throw BadValue("residual " + shape_of(r.sizes()) + " does not have the output's shape " + shape_of(shape));
  for (const Tensor* t : {&w, &b, &r})
    if (t->defined() && t->scalar_type() != x.scalar_type())
      throw BadValue(std::string("x, weight, bias and residual must have one type, got ") +
                     c10::toString(x.scalar_type()) + " and " + c10::toString(t->scalar_type()));
  check_devices(x, {&w, &b, &r});
  if (wants_grad({&x, &w, &b, &r})) {
    if (user_status) throw BadValue("status is not supported on the differentiable path");
    return LinearFunction::apply(x, w, given(b), given(r), (int64_t)act, reinterpret_cast<int64_t>(status));
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return run_linear(rows_of(x), rows_of(w), b.defined() ? b.contiguous() : b, r.defined() ? rows_of(r) : r, act, shape,
                    nullptr, status);
}

// ------------------------------------------------------------------ layer norm
Tensor run_layer_norm(const Tensor& x, const Tensor& w, const Tensor& b, at::ScalarType param, double eps,
                      at::IntArrayRef shape, Tensor* stats) {
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0), d = x.size(1);
  Tensor y = at::empty(shape, x.options());
  float* at_stats = nullptr;
  if (stats) {
    *stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    at_stats = stats->data_ptr<float>();
  }
  check(wf.layer_norm(x.data_ptr(), dtype_code(x.scalar_type()), rows, d, x.stride(0), ptr(w), ptr(b),
                      dtype_code(param), (float)eps, y.data_ptr(), d, at_stats, stats ? at_stats + rows : nullptr,
                      stream()));
  return y;
}

struct LayerNormFunction : torch::autograd::Function<LayerNormFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Optional& w, const Optional& b, double eps,
                        int64_t param) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor x2 = rows_of(x), w2 = contiguous(w);
    Tensor stats;
    Tensor y = run_layer_norm(x2, w2, contiguous(b), (at::ScalarType)param, eps, x.sizes(), &stats);
    ctx->save_for_backward({to_save(x, x2), w2, stats});
    ctx->saved_data["weight"] = w.has_value();
    ctx->saved_data["bias"] = b.has_value();
    ctx->saved_data["param"] = param;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once_only();
    const auto saved = ctx->get_saved_variables();
    const Tensor x = rows_of(saved[0]), &w = saved[1], &stats = saved[2], &dy = grads[0];
    const auto param = (at::ScalarType)ctx->saved_data["param"].toInt();
    size_t edge = 1;
    const bool need_x = ctx->needs_input_grad(0);
    const bool need_w = needs_optional(ctx, "weight", edge);
    const bool need_b = needs_optional(ctx, "bias", edge);
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t rows = x.size(0), d = x.size(1);
    const int code = dtype_code(x.scalar_type());
    const Tensor g = rows_of(dy);
    Tensor dx, dw, db;
    if (need_x) dx = at::empty(dy.sizes(), x.options());
    if (need_w) dw = at::empty({d}, x.options().dtype(param));
    if (need_b) db = at::empty({d}, x.options().dtype(param));
    const size_t n = need_w || need_b ? wf.layer_norm_backward_workspace_bytes(rows, d, code) : 0;
    const Tensor ws = bytes(n, x);
    const float* s = stats.data_ptr<float>();
    check(wf.layer_norm_backward(x.data_ptr(), g.data_ptr(), code, rows, d, x.stride(0), g.stride(0), ptr(w),
                                 dtype_code(param), s, s + rows, ptr(dx), ptr(dw), ptr(db), ptr(ws), n, stream()));
    return {dx, dw, db, Tensor(), Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const Tensor& w, const Tensor& b, double eps) {
  if (x.dim() < 1 || x.size(-1) < 1) throw BadValue("expected x (..., d) with d >= 1, got " + shape_of(x.sizes()));
  if (!(eps >= 0)) throw BadValue("eps must be >= 0, got " + std::to_string(eps));
  auto param = x.scalar_type();
  bool any = false;
  for (const Tensor* p : {&w, &b}) {
    if (!p->defined()) continue;
    if (p->dim() != 1 || p->size(0) != x.size(-1))
      throw BadValue("weight and bias must be (" + std::to_string(x.size(-1)) + ",), got " + shape_of(p->sizes()));
    const auto t = p->scalar_type();
    if ((t != x.scalar_type() && t != at::kFloat) || (any && t != param))
      throw BadValue(std::string("weight and bias must both be ") + c10::toString(x.scalar_type()) +
                     " or float32, got " + c10::toString(t));
    param = t;
    any = true;
  }
  check_devices(x, {&w, &b});
  dtype_code(x.scalar_type());
  if (wants_grad({&x, &w, &b}))
    return LayerNormFunction::apply(x, given(w), given(b), eps, (int64_t)param);
  at::AutoDispatchBelowADInplaceOrView below;
  return run_layer_norm(rows_of(x), w.defined() ? w.contiguous() : w, b.defined() ? b.contiguous() : b, param, eps,
                        x.sizes(), nullptr);
}

// ------------------------------------------------------------------ token log probabilities
struct Scored {
  Tensor logprob, entropy, top_logprobs, top_tokens;
};
Scored run_token_logprobs(const Tensor& x, const Tensor& tokens, int64_t top_n, int64_t ignore, at::IntArrayRef lead,
                          Tensor* stats, void* status) {
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0);
  const auto f32 = x.options().dtype(at::kFloat);
  auto top = lead.vec();
  top.push_back(top_n);
  Scored r{at::empty(lead, f32), at::empty(lead, f32), at::empty(top, f32), at::empty(top, x.options().dtype(at::kLong))};
  if (stats) *stats = at::empty({2, rows}, f32);
  check(wf.token_logprobs(x.data_ptr(), dtype_code(x.scalar_type()), rows, x.size(1), x.stride(0),
                          tokens.data_ptr<int64_t>(), ignore, (int)top_n, r.logprob.data_ptr<float>(),
                          r.entropy.data_ptr<float>(), stats ? stats->data_ptr<float>() : nullptr,
                          r.top_logprobs.data_ptr<float>(), r.top_tokens.data_ptr<int64_t>(),
                          static_cast<int32_t*>(status), stream()));
  return r;
}

struct TokenLogprobsFunction : torch::autograd::Function<TokenLogprobsFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens,
                               const std::vector<int64_t>& lead, int64_t top_n, int64_t ignore, int64_t status) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor x = rows_of(logits);
    Tensor stats;
    Scored r = run_token_logprobs(x, tokens, top_n, ignore, lead, &stats, reinterpret_cast<void*>(status));
    ctx->save_for_backward({to_save(logits, x), tokens, stats, r.entropy});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["shape"] = logits.sizes().vec();
    ctx->mark_non_differentiable({r.top_logprobs, r.top_tokens});
    ctx->set_materialize_grads(false);
    return {r.logprob, r.entropy, r.top_logprobs, r.top_tokens};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once_only();
    variable_list none(6);
    if (!grads[0].defined() && !grads[1].defined()) return none;
    const auto saved = ctx->get_saved_variables();
    const Tensor x = rows_of(saved[0]), &tokens = saved[1], &stats = saved[2], &entropy = saved[3];
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor gl = grads[0].defined() ? grads[0].contiguous() : Tensor(),
                 gh = grads[1].defined() ? grads[1].contiguous() : Tensor();
    Tensor dx = at::empty(ctx->saved_data["shape"].toIntVector(), x.options());
    check(wf.token_logprobs_backward(x.data_ptr(), dtype_code(x.scalar_type()), x.size(0), x.size(1), x.stride(0),
                                     tokens.data_ptr<int64_t>(), ctx->saved_data["ignore"].toInt(),
                                     stats.data_ptr<float>(), entropy.data_ptr<float>(),
                                     static_cast<const float*>(ptr(gl)), static_cast<const float*>(ptr(gh)),
                                     dx.data_ptr(), stream()));
    none[0] = dx;
    return none;
  }
};

variable_list token_logprobs(const Tensor& logits, const Tensor& tokens, int64_t top_n, int64_t ignore, void* status,
                             bool user_status) {
  if (logits.dim() < 1 || logits.size(-1) < 1)
    throw BadValue("expected logits (..., vocab) with vocab >= 1, got " + shape_of(logits.sizes()));
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  if (tokens.sizes() != lead)
    throw BadValue("tokens " + shape_of(tokens.sizes()) + " do not match logits " + shape_of(logits.sizes()));
  if (tokens.scalar_type() != at::kLong && tokens.scalar_type() != at::kInt)
    throw BadValue(std::string("tokens must be int64 or int32, got ") + c10::toString(tokens.scalar_type()));
  const int64_t most = std::min<int64_t>(logits.size(-1), wf.max_top_tokens());
  if (top_n < 0 || top_n > most)
    throw BadValue("top_n must be in [0, " + std::to_string(most) + "] here, got " + std::to_string(top_n));
  check_devices(logits, {&tokens});
  const Tensor flat = tokens.to(at::kLong).contiguous();
  if (wants_grad({&logits})) {
    if (user_status) throw BadValue("status is not supported on the differentiable path");
    return TokenLogprobsFunction::apply(logits, flat, lead.vec(), top_n, ignore, reinterpret_cast<int64_t>(status));
  }
  at::AutoDispatchBelowADInplaceOrView below;
  Scored r = run_token_logprobs(rows_of(logits), flat, top_n, ignore, lead, nullptr, status);
  return {r.logprob, r.entropy, r.top_logprobs, r.top_tokens};
}

// ------------------------------------------------------------------ Python
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const BadValue& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
Tensor tensor_arg(PyObject* o, const char* name, bool optional = false) {
  if (optional && o == Py_None) return Tensor();
  if (!THPVariable_Check(o)) throw BadValue(std::string(name) + " must be a tensor" + (optional ? " or None" : ""));
  return THPVariable_Unpack(o);
}
int64_t int_arg(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw std::runtime_error("integer expected");
  return v;
}
void count(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) throw std::runtime_error("wrong number of arguments");
}
// The GIL is not held while the host enqueues work.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

PyObject* py_bind(PyObject*, PyObject* path) {
  return guarded([&]() -> PyObject* {
    const char* p = PyUnicode_AsUTF8(path);
    if (!p) throw std::runtime_error("path expected");
    void* lib = dlopen(p, RTLD_NOW | RTLD_LOCAL);
    if (!lib) throw std::runtime_error(dlerror());
    auto find = [&](auto& f, const char* name) {
      f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(dlsym(lib, name));
      if (!f) throw std::runtime_error(std::string("the library lacks ") + name);
    };
    find(wf.last_error, "wf_last_error");
    find(wf.linear, "wf_linear");
    find(wf.linear_workspace_bytes, "wf_linear_workspace_bytes");
    find(wf.linear_backward, "wf_linear_backward");
    find(wf.linear_backward_workspace_bytes, "wf_linear_backward_workspace_bytes");
    find(wf.layer_norm, "wf_layer_norm");
    find(wf.layer_norm_backward, "wf_layer_norm_backward");
    find(wf.layer_norm_backward_workspace_bytes, "wf_layer_norm_backward_workspace_bytes");
    find(wf.max_top_tokens, "wf_max_top_tokens");
    find(wf.token_logprobs, "wf_token_logprobs");
    find(wf.token_logprobs_backward, "wf_token_logprobs_backward");
    Py_RETURN_NONE;
  });
}

// fused_linear(x, weight, bias, residual, activation, status pointer, the status is the user's)
PyObject* py_fused_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    count(n, 7);
    const Tensor x = tensor_arg(a[0], "x"), w = tensor_arg(a[1], "weight"), b = tensor_arg(a[2], "bias", true),
                 r = tensor_arg(a[3], "residual", true);
    const int64_t act = int_arg(a[4]), status = int_arg(a[5]);
    const bool user = a[6] == Py_True;
    Tensor y;
    {
      Unlocked unlocked;
      y = fused_linear(x, w, b, r, (int)act, reinterpret_cast<void*>(status), user);
    }
    return THPVariable_Wrap(std::move(y));
  });
}

// layer_norm(x, weight, bias, eps)
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    count(n, 4);
    const Tensor x = tensor_arg(a[0], "x"), w = tensor_arg(a[1], "weight", true), b = tensor_arg(a[2], "bias", true);
    const double eps = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) throw std::runtime_error("number expected");
    Tensor y;
    {
      Unlocked unlocked;
      y = layer_norm(x, w, b, eps);
    }
    return THPVariable_Wrap(std::move(y));
  });
}

// token_logprobs(logits, tokens, top_n, ignore_index, status pointer, the status is the user's)
PyObject* py_token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 6);
    const Tensor logits = tensor_arg(a[0], "logits"), tokens = tensor_arg(a[1], "tokens");
    const int64_t top_n = int_arg(a[2]), ignore = int_arg(a[3]), status = int_arg(a[4]);
    const bool user = a[5] == Py_True;
    variable_list r;
    {
      Unlocked unlocked;
      r = token_logprobs(logits, tokens, top_n, ignore, reinterpret_cast<void*>(status), user);
    }
    PyObject* out = PyTuple_New((Py_ssize_t)r.size());
    if (!out) return nullptr;
    for (size_t i = 0; i < r.size(); ++i) PyTuple_SET_ITEM(out, (Py_ssize_t)i, THPVariable_Wrap(std::move(r[i])));
    return out;
  });
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_O, "Look the C ABI up in the library at this path."},
    {"fused_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_fused_linear)), METH_FASTCALL, nullptr},
    {"layer_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_layer_norm)), METH_FASTCALL, nullptr},
    {"token_logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_token_logprobs)), METH_FASTCALL,
     nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_wf_torch", "PyTorch calls over the wayfinder C ABI.", -1, methods,
                      nullptr,               nullptr,     nullptr,                                   nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__wf_torch() { return PyModule_Create(&module); }
