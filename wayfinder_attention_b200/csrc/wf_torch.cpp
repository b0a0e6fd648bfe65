// fused_linear, layer_norm, token_logprobs, linear_token_logprobs and token_embedding as PyTorch calls: argument checks, outputs and
// autograd nodes around the C ABI (include/wayfinder.h), whose functions are looked up in the
// library that the package loads.  A small training step is bound by the host: the same nodes
// in Python took 118 us of host time for a layer norm's forward and backward, against 70 us
// of PyTorch's own.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <limits>
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
  decltype(&wf_linear_token_logprobs) linear_token_logprobs;
  decltype(&wf_linear_token_logprobs_workspace_bytes) linear_token_logprobs_workspace_bytes;
  decltype(&wf_linear_token_logprobs_backward) linear_token_logprobs_backward;
  decltype(&wf_linear_token_logprobs_backward_workspace_bytes) linear_token_logprobs_backward_workspace_bytes;
  decltype(&wf_token_embedding) token_embedding;
  decltype(&wf_token_embedding_backward) token_embedding_backward;
  decltype(&wf_token_embedding_backward_workspace_bytes) token_embedding_backward_workspace_bytes;
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
// A gradient goes on on the stream of the node that takes it.  A leaf's node that a graph made outside of a capture keeps
// alive has the default stream, which cannot wait for a capture: the engine's attempt breaks the capture, so
// it is refused before.  A leaf that this pass wants nothing of (autograd.grad for others) is not gone to.
void check_capture() {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (size_t i = 0; i < node->num_outputs(); ++i) {
    if (!node->task_should_compute_output(i)) continue;
    const auto to = node->next_edge(i).function->stream();
    TORCH_CHECK(!to || *to != c10::cuda::getDefaultCUDAStream(to->device_index()).unwrap(),
                "a backward is captured into a CUDA graph while an autograd graph of the same leaves, made on the "
                "default stream, is alive: delete that first");
  }
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

// ------------------------------------------------------------------ log probabilities without logits
Tensor long_ids(const Tensor& t, const char* name) {
  if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)
    throw BadValue(std::string(name) + " must be int64 or int32, got " + c10::toString(t.scalar_type()));
  return t.to(at::kLong).contiguous();
}

std::pair<Tensor, Tensor> run_linear_logprobs(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& tokens,
                                              int64_t ignore, at::IntArrayRef lead, Tensor* stats, void* status) {
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0), d = x.size(1), vocab = w.size(0);
  const int code = dtype_code(x.scalar_type());
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor logprob = at::empty(lead, f32), entropy = at::empty(lead, f32);
  if (stats) *stats = at::empty({2, rows}, f32);
  const size_t n = wf.linear_token_logprobs_workspace_bytes(rows, vocab, d, code, on_16_bytes(x), on_16_bytes(w));
  const Tensor ws = bytes(n, x);
  check(wf.linear_token_logprobs(x.data_ptr(), w.data_ptr(), ptr(b), code, rows, vocab, d, x.stride(0), w.stride(0),
                                 tokens.data_ptr<int64_t>(), ignore, logprob.data_ptr<float>(),
                                 entropy.data_ptr<float>(), stats ? stats->data_ptr<float>() : nullptr, ptr(ws), n,
                                 static_cast<int32_t*>(status), stream()));
  return {logprob, entropy};
}

struct LinearLogprobsFunction : torch::autograd::Function<LinearLogprobsFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Optional& b,
                               const Tensor& tokens, int64_t ignore, int64_t status) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor x2 = rows_of(x), w2 = rows_of(w), b2 = contiguous(b);
    Tensor stats;
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    auto [logprob, entropy] =
        run_linear_logprobs(x2, w2, b2, tokens, ignore, lead, &stats, reinterpret_cast<void*>(status));
    ctx->save_for_backward({to_save(x, x2), to_save(w, w2), b2, tokens, stats, entropy});
    ctx->saved_data["bias"] = b.has_value();
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["status"] = status;
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->set_materialize_grads(false);
    return {logprob, entropy};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once_only();
    check_capture();
    variable_list out(6);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor x = rows_of(saved[0]), w = rows_of(saved[1]), &b = saved[2], &tokens = saved[3], &stats = saved[4],
                 &entropy = saved[5];
    size_t edge = 2;
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_b = needs_optional(ctx, "bias", edge);
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t rows = x.size(0), d = x.size(1), vocab = w.size(0);
    const int code = dtype_code(x.scalar_type());
    const Tensor gl = grads[0].defined() ? grads[0].contiguous() : Tensor(),
                 gh = grads[1].defined() ? grads[1].contiguous() : Tensor();
    if (need_x) out[0] = at::empty(ctx->saved_data["shape"].toIntVector(), x.options());
    if (need_w) out[1] = at::empty({vocab, d}, x.options());
    if (need_b) out[2] = at::empty({vocab}, x.options());
    const size_t n =
        wf.linear_token_logprobs_backward_workspace_bytes(rows, vocab, d, code, on_16_bytes(x), on_16_bytes(w));
    const Tensor ws = bytes(n, x);
    check(wf.linear_token_logprobs_backward(
        x.data_ptr(), w.data_ptr(), ptr(b), code, rows, vocab, d, x.stride(0), w.stride(0), tokens.data_ptr<int64_t>(),
        ctx->saved_data["ignore"].toInt(), stats.data_ptr<float>(), entropy.data_ptr<float>(),
        static_cast<const float*>(ptr(gl)), static_cast<const float*>(ptr(gh)), ptr(out[0]), ptr(out[1]), ptr(out[2]),
        ptr(ws), n, reinterpret_cast<int32_t*>(ctx->saved_data["status"].toInt()), stream()));
    return out;
  }
};

variable_list linear_token_logprobs(const Tensor& x, const Tensor& w, const Tensor& tokens, const Tensor& b,
                                    int64_t ignore, void* status, bool user_status) {
  if (x.dim() < 1 || w.dim() != 2 || x.size(-1) != w.size(1) || w.numel() == 0)
    throw BadValue("expected x (..., d) and weight (vocab, d) with sizes >= 1, got " + shape_of(x.sizes()) + " and " +
                   shape_of(w.sizes()));
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  if (tokens.sizes() != lead)
    throw BadValue("tokens " + shape_of(tokens.sizes()) + " do not match x " + shape_of(x.sizes()));
  if (b.defined() && (b.dim() != 1 || b.size(0) != w.size(0)))
    throw BadValue("bias " + shape_of(b.sizes()) + " does not match vocab=" + std::to_string(w.size(0)));
  for (const Tensor* t : {&w, &b})
    if (t->defined() && t->scalar_type() != x.scalar_type())
      throw BadValue(std::string("x, weight and bias must have one type, got ") + c10::toString(x.scalar_type()) +
                     " and " + c10::toString(t->scalar_type()));
  check_devices(x, {&w, &tokens, &b});
  dtype_code(x.scalar_type());
  const Tensor flat = long_ids(tokens, "tokens");
  if (wants_grad({&x, &w, &b})) {
    if (user_status) throw BadValue("status is not supported on the differentiable path");
    return LinearLogprobsFunction::apply(x, w, given(b), flat, ignore, reinterpret_cast<int64_t>(status));
  }
  at::AutoDispatchBelowADInplaceOrView below;
  auto [logprob, entropy] = run_linear_logprobs(rows_of(x), rows_of(w), b.defined() ? b.contiguous() : b, flat, ignore,
                                                lead, nullptr, status);
  return {logprob, entropy};
}

// ------------------------------------------------------------------ token embedding
Tensor run_embedding(const Tensor& w, const Tensor& pw, const Tensor& tokens, const Tensor& positions, double scale,
                     at::IntArrayRef lead, void* status) {
  c10::cuda::CUDAGuard guard(w.device());
  auto shape = lead.vec();
  const int64_t seq = shape.empty() ? 1 : shape.back();
  shape.push_back(w.size(1));
  Tensor y = at::empty(shape, w.options());
  check(wf.token_embedding(tokens.data_ptr<int64_t>(), tokens.numel(), w.data_ptr(), dtype_code(w.scalar_type()),
                           w.size(0), w.size(1), w.stride(0), (float)scale, ptr(pw), pw.defined() ? pw.size(0) : 0,
                           pw.defined() ? pw.stride(0) : 0,
                           positions.defined() ? positions.data_ptr<int64_t>() : nullptr, std::max<int64_t>(seq, 1),
                           y.data_ptr(), static_cast<int32_t*>(status), stream()));
  return y;
}

struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& w, const Optional& pw, const Tensor& tokens,
                        const Optional& positions, double scale, int64_t padding, const std::vector<int64_t>& lead,
                        int64_t status) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor at = positions ? *positions : Tensor();
    Tensor y = run_embedding(rows_of(w), pw ? rows_of(*pw) : Tensor(), tokens, at, scale, lead,
                             reinterpret_cast<void*>(status));
    ctx->save_for_backward({tokens, at});
    ctx->saved_data["position_weight"] = pw.has_value();
    ctx->saved_data["places"] = pw ? pw->size(0) : 0;
    ctx->saved_data["vocab"] = w.size(0);
    ctx->saved_data["seq"] = lead.empty() ? 1 : lead.back();
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once_only();
    check_capture();
    const auto saved = ctx->get_saved_variables();
    const Tensor &tokens = saved[0], &positions = saved[1];
    size_t edge = 1;
    const bool need_w = ctx->needs_input_grad(0), need_p = needs_optional(ctx, "position_weight", edge);
    c10::cuda::CUDAGuard guard(grads[0].device());
    const Tensor dy = rows_of(grads[0]);
    const int64_t n = tokens.numel(), d = dy.size(1), seq = std::max<int64_t>(1, ctx->saved_data["seq"].toInt());
    const int code = dtype_code(dy.scalar_type());
    const int64_t vocab = ctx->saved_data["vocab"].toInt(), places = ctx->saved_data["places"].toInt();
    variable_list out(8);
    if (need_w) out[0] = at::empty({vocab, d}, dy.options());
    if (need_p) out[1] = at::empty({places, d}, dy.options());
    const size_t size = wf.token_embedding_backward_workspace_bytes(n, need_w ? vocab : 0, need_p ? places : 0, d, code,
                                                                    positions.defined());
    const Tensor ws = bytes(size, dy);
    check(wf.token_embedding_backward(tokens.data_ptr<int64_t>(),
                                      positions.defined() ? positions.data_ptr<int64_t>() : nullptr, n, seq,
                                      dy.data_ptr(), code, d, dy.stride(0), vocab,
                                      (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(),
                                      ptr(out[0]), places, ptr(out[1]), ptr(ws), size, stream()));
    return out;
  }
};

Tensor token_embedding(const Tensor& tokens, const Tensor& w, double scale, const Tensor& pw, const Tensor& positions,
                       int64_t padding, void* status, bool user_status) {
  if (w.dim() != 2 || w.numel() == 0)
    throw BadValue("expected weight (vocab, d) with sizes >= 1, got " + shape_of(w.sizes()));
  if (pw.defined() && (pw.dim() != 2 || pw.numel() == 0 || pw.size(1) != w.size(1)))
    throw BadValue("position_weight " + shape_of(pw.sizes()) + " does not match weight " + shape_of(w.sizes()));
  if (pw.defined() && pw.scalar_type() != w.scalar_type())
    throw BadValue(std::string("weight and position_weight must have one type, got ") + c10::toString(w.scalar_type()) +
                   " and " + c10::toString(pw.scalar_type()));
  if (positions.defined() && !pw.defined()) throw BadValue("positions need a position_weight");
  const auto lead = tokens.sizes();
  if (positions.defined() && positions.sizes() != lead &&
      (positions.dim() != 1 || lead.empty() || positions.size(0) != lead.back()))
    throw BadValue("positions " + shape_of(positions.sizes()) + " are neither of the tokens' shape " + shape_of(lead) +
                   " nor of its last axis");
  if (padding >= w.size(0)) throw BadValue("padding_index must be below vocab=" + std::to_string(w.size(0)));
  if (!(std::abs(scale) <= std::numeric_limits<float>::max())) throw BadValue("scale must be finite in float32");
  check_devices(w, {&tokens, &pw, &positions});
  dtype_code(w.scalar_type());
  const Tensor flat = long_ids(tokens, "tokens"),
               at = positions.defined() ? long_ids(positions.expand(lead), "positions") : Tensor();
  if (wants_grad({&w, &pw})) {
    if (user_status) throw BadValue("status is not supported on the differentiable path");
    return EmbeddingFunction::apply(w, given(pw), flat, given(at), scale, padding, lead.vec(),
                                    reinterpret_cast<int64_t>(status));
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return run_embedding(rows_of(w), pw.defined() ? rows_of(pw) : pw, flat, at, scale, lead, status);
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
    find(wf.linear_token_logprobs, "wf_linear_token_logprobs");
    find(wf.linear_token_logprobs_workspace_bytes, "wf_linear_token_logprobs_workspace_bytes");
    find(wf.linear_token_logprobs_backward, "wf_linear_token_logprobs_backward");
    find(wf.linear_token_logprobs_backward_workspace_bytes, "wf_linear_token_logprobs_backward_workspace_bytes");
    find(wf.token_embedding, "wf_token_embedding");
    find(wf.token_embedding_backward, "wf_token_embedding_backward");
    find(wf.token_embedding_backward_workspace_bytes, "wf_token_embedding_backward_workspace_bytes");
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

// linear_token_logprobs(x, weight, tokens, bias, ignore_index, status pointer, the status is the user's)
PyObject* py_linear_token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 7);
    const Tensor x = tensor_arg(a[0], "x"), w = tensor_arg(a[1], "weight"), tokens = tensor_arg(a[2], "tokens"),
                 b = tensor_arg(a[3], "bias", true);
    const int64_t ignore = int_arg(a[4]), status = int_arg(a[5]);
    const bool user = a[6] == Py_True;
    variable_list r;
    {
      Unlocked unlocked;
      r = linear_token_logprobs(x, w, tokens, b, ignore, reinterpret_cast<void*>(status), user);
    }
    PyObject* out = PyTuple_New(2);
    if (!out) return nullptr;
    for (int i = 0; i < 2; ++i) PyTuple_SET_ITEM(out, i, THPVariable_Wrap(std::move(r[i])));
    return out;
  });
}

// token_embedding(tokens, weight, scale, position_weight, positions, padding_index or -1, status pointer,
// the status is the user's)
PyObject* py_token_embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    count(n, 8);
    const Tensor tokens = tensor_arg(a[0], "tokens"), w = tensor_arg(a[1], "weight"),
                 pw = tensor_arg(a[3], "position_weight", true), positions = tensor_arg(a[4], "positions", true);
    const double scale = PyFloat_AsDouble(a[2]);
    if (PyErr_Occurred()) throw std::runtime_error("number expected");
    const int64_t padding = int_arg(a[5]), status = int_arg(a[6]);
    const bool user = a[7] == Py_True;
    Tensor y;
    {
      Unlocked unlocked;
      y = token_embedding(tokens, w, scale, pw, positions, padding, reinterpret_cast<void*>(status), user);
    }
    return THPVariable_Wrap(std::move(y));
  });
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_O, "Look the C ABI up in the library at this path."},
    {"fused_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_fused_linear)), METH_FASTCALL, nullptr},
    {"layer_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_layer_norm)), METH_FASTCALL, nullptr},
    {"token_logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_token_logprobs)), METH_FASTCALL,
     nullptr},
    {"linear_token_logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_linear_token_logprobs)),
     METH_FASTCALL, nullptr},
    {"token_embedding", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_token_embedding)), METH_FASTCALL,
     nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_wf_torch", "PyTorch calls over the wayfinder C ABI.", -1, methods,
                      nullptr,               nullptr,     nullptr,                                   nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__wf_torch() { return PyModule_Create(&module); }
