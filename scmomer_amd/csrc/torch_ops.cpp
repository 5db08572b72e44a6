// The operators at a model's end (norm.py, logits.py) as torch functions: checks of arguments, allocation of outputs and
// workspaces, calls of the C ABI, autograd nodes.  They are called one by one from eager programs, forward on one thread
// and backward on autograd's, where an interpreted host path costs more than most of the kernels: layer_norm forward and
// backward at launch-bound sizes 165 us through Python functions and ctypes, 109 us with those cut down, 67 us here (an
// elementwise product of torch's own, forward and backward: 47 us; its layer norm 75).
// The library's entry points are handed over as addresses (bind), so this module needs no second copy of it.
#include "../../include/scmomer_hip.h"
#include <torch/extension.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <limits>
#include <tuple>
#include <unordered_set>
#include <vector>

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Api {
  decltype(&scm_last_error) last_error;
  decltype(&scm_norm_fwd) norm_fwd;
  decltype(&scm_norm_bwd) norm_bwd;
  decltype(&scm_norm_bwd_ws_floats) norm_bwd_ws_floats;
  decltype(&scm_score_ws_floats) score_ws_floats;
  decltype(&scm_score_fwd) score_fwd;
  decltype(&scm_score_bwd) score_bwd;
  decltype(&scm_topk_distill_tape_floats) topk_distill_tape_floats;
  decltype(&scm_topk_distill_ws_floats) topk_distill_ws_floats;
  decltype(&scm_topk_distill_fwd) topk_distill_fwd;
  decltype(&scm_topk_distill_bwd) topk_distill_bwd;
  decltype(&scm_topk_distill_step) topk_distill_step;
} api;

constexpr int64_t NORM_MAX_D = 16384, LOGITS_MAX_K = 64, LOGITS_MAX_V = 1 << 30;

void call(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", api.last_error()); }

int type_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return SCM_F32;
    case at::kBFloat16: return SCM_BF16;
    case at::kHalf: return SCM_F16;
    default: TORCH_CHECK_TYPE(false, name, ": expected float32, bfloat16 or float16, got ", t.scalar_type());
  }
}
// A tensor whose memory holds its values: a view that only notes a change of sign (the imaginary part of a conjugate) and
// a gradient that is only noted to be zero get theirs written.
Tensor values(const Tensor& t) {
  if (!t.defined()) return t;
  return t.is_neg() ? t.resolve_neg() : t._is_zerotensor() ? t.clone() : t;
}
// [T, D] form of [..., D]: a view where one row stride describes it (an expanded batch keeps stride 0), else a copy
Tensor rows_of(const Tensor& t_, const char* name) {
  const Tensor t = values(t_);
  type_of(t, name);
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1, name, ": expected [..., D] with D >= 1, got ", t.sizes());
  Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / t.size(-1), t.size(-1)});
  return r.size(1) != 1 && r.stride(1) != 1 ? r.contiguous() : r;
}
void on_device_of(const Tensor& t, const Tensor& o, const char* name) {
  TORCH_CHECK_VALUE(!o.defined() || o.device() == t.device(), name, ": on ", o.device(), ", expected ", t.device());
}
void check_device(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, ": expected a device tensor; scmomer_amd has no CPU path");
}
void* stream_of(const Tensor& t) {   // the tensors' device is the current one here
  return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}
template <typename T = float>
T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }
Tensor floats(const Tensor& like, at::IntArrayRef size) { return at::empty(size, like.options().dtype(at::kFloat)); }
Tensor scratch(const Tensor& like, int64_t n) { return n ? floats(like, {n}) : Tensor(); }
Tensor opt(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
bool needs_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
// one value per row of the logits, contiguous
Tensor row_vector(const Tensor& t, const Tensor& logits, at::ScalarType type, const char* name) {
  if (!t.defined()) return t;
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, ": expected ", type, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.sizes() == logits.sizes().slice(0, logits.dim() - 1), name, ": expected ",
                    logits.sizes().slice(0, logits.dim() - 1), ", got ", t.sizes());
  on_device_of(logits, t, name);
  return values(t).contiguous();
}
// an incoming gradient as n contiguous f32 values (undefined: none)
Tensor grad_rows(const Tensor& g, const Tensor& like, int64_t n) {
  if (!g.defined()) return g;
  TORCH_CHECK_VALUE(g.numel() == n, "incoming gradient: ", g.numel(), " values, expected ", n);
  on_device_of(like, g, "incoming gradient");
  return values(g).to(at::kFloat).contiguous();
}

// The kernels work on addresses: what hands tensors on without values, or follows a call by its torch operations, sees
// nothing of them.  Refused are tensors of forward-mode differentiation (their tangent would be lost), wrappers, which have
// no memory (of subclasses with a dispatch of their own, of torch.func's transforms), and calls under a tracer (it would
// record the allocation of the results only).
void check_followed(std::initializer_list<std::reference_wrapper<const Tensor>> tensors) {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  bool traced = torch::jit::tracer::isTracing();
  if (TorchDispatchModeTLS::any_modes_set())
    for (const auto key : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
      traced = traced || TorchDispatchModeTLS::get_mode(key).has_value();
  TORCH_CHECK_NOT_IMPLEMENTED(!traced, "this operator of scmomer_amd cannot be traced");
  constexpr c10::DispatchKeySet wrappers({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                          c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize});
  for (const Tensor& t : tensors) {
    if (!t.defined()) continue;
    TORCH_CHECK_NOT_IMPLEMENTED(!t.key_set().has_any(wrappers), "this operator of scmomer_amd takes plain tensors, not those of "
                                "torch.func's transforms or of subclasses with a dispatch of their own");
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "this operator of scmomer_amd has no forward-mode derivative");
  }
}

// Gradients that came out of a backward pass under create_graph: they refuse to be differentiated again.
struct FirstOnly : torch::autograd::Function<FirstOnly> {
  static Tensor forward(AutogradContext*, const Tensor& g) { return g.view_as(g); }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "this operator of scmomer_amd has first derivatives only");
  }
};
Tensor once(const Tensor& g) {
  if (!g.defined() || !at::GradMode::is_enabled()) return g;
  return FirstOnly::apply(g.detach().requires_grad_(true));
}

// A leaf's accumulator keeps the stream of the graph that made it for as long as a graph holds it.  Where that is the default
// stream, a backward pass under capture would make that stream wait for a captured event, which no capture allows and
// which ends the process.  Called by the node whose gradients are due, before anything is launched, for all that this
// backward pass reaches from there: the leaves of a whole model.
void check_capture(const Tensor& t) {
  const auto here = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (here.stream() == nullptr) return;   // never under capture
  if (hipStreamIsCapturing(here.stream(), &status) != hipSuccess) {
    (void)hipGetLastError();
    return;
  }
  const auto first = torch::autograd::get_current_node();
  if (status == hipStreamCaptureStatusNone || !first) return;
  std::vector<torch::autograd::Node*> todo{first.get()};
  std::unordered_set<torch::autograd::Node*> seen{first.get()};
  while (!todo.empty()) {
    torch::autograd::Node* const node = todo.back();
    todo.pop_back();
    for (uint32_t i = 0; i < node->num_outputs(); ++i) {
      const auto& e = node->next_edge(i);
      if (!e.function || !node->task_should_compute_output(i) || !seen.insert(e.function.get()).second) continue;
      const auto s = e.function->stream();
      TORCH_CHECK(!s || s->id() != 0, "a backward pass under capture reaches ", e.function->name(), " on the default stream, "
                  "which cannot take part: release the eager graph that holds it (its loss and outputs), or run that graph's "
                  "forward pass on another stream than the default one");
      todo.push_back(e.function.get());
    }
  }
}

// ---------------------------------------------------------------------------- layer norm
// -> y, statistics [2, T] (mean, 1 / standard deviation)
std::tuple<Tensor, Tensor> norm_fwd(const Tensor& x_, const Tensor& w_, const Tensor& b_, double eps,
                                    std::optional<at::ScalarType> out_dtype, bool stats) {
  const Tensor x = rows_of(x_, "x"), w = values(w_), b = values(b_);
  const int64_t t = x.size(0), d = x.size(1);
  const auto out = out_dtype.value_or(x.scalar_type());
  TORCH_CHECK_TYPE(out == x.scalar_type() || (x.scalar_type() == at::kFloat && out == at::kBFloat16), "layer norm: ",
                   x.scalar_type(), " in gives ", x.scalar_type(), " out, or bfloat16 from float32 (asked for ", out, ")");
  TORCH_CHECK_VALUE(d <= NORM_MAX_D, "layer norm: at most ", NORM_MAX_D, " columns (got ", d, ")");
  check_device(x, "x");
  for (const auto& [p, name] : {std::pair<const Tensor&, const char*>(w, "weight"), {b, "bias"}}) {
    if (!p.defined()) continue;
    TORCH_CHECK_TYPE(p.scalar_type() == at::kFloat, name, ": expected float32, got ", p.scalar_type());
    TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == d && p.is_contiguous(), name, ": expected a contiguous [", d, "], got ",
                      p.sizes());
    on_device_of(x, p, name);
  }
  const c10::DeviceGuard guard(x.device());
  Tensor y = at::empty(x_.sizes(), x.options().dtype(out));
  Tensor st = stats ? floats(x, {2, t}) : Tensor();
  if (t)
    call(api.norm_fwd(x.data_ptr(), type_of(x, "x"), x.stride(0), ptr(w), ptr(b), t, (int)d, (float)eps, y.data_ptr(),
                      type_of(y, "y"), ptr(st), stats ? ptr(st) + t : nullptr, stream_of(x)), "scm_norm_fwd");
  return {y, st};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w_, const OptTensor& b_, double eps,
                        std::optional<at::ScalarType> out_dtype) {
    const Tensor w = opt(w_), b = opt(b_);
    auto [y, st] = norm_fwd(x, w, b, eps, out_dtype, true);
    ctx->save_for_backward({x, w, st});
    ctx->saved_data["bias"] = b.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_followed({grads[0]});
    const auto saved = ctx->get_saved_variables();
    check_capture(saved[0]);
    const Tensor &x_ = saved[0], &st = saved[2];
    const Tensor x = rows_of(x_, "x"), w = values(saved[1]), dy = rows_of(grads[0], "dy");
    on_device_of(x, dy, "dy");
    const int64_t t = x.size(0), d = x.size(1);
    // edges count the tensors that were given
    const bool want_x = ctx->needs_input_grad(0), want_w = w.defined() && ctx->needs_input_grad(1);
    const bool want_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(w.defined() ? 2 : 1);
    const c10::DeviceGuard guard(x.device());
    Tensor dx = want_x ? at::empty(x_.sizes(), x.options()) : Tensor();
    auto sum = [&](bool want) {   // no rows: the sums are empty
      return !want ? Tensor() : t ? floats(x, {d}) : at::zeros({d}, x.options().dtype(at::kFloat));
    };
    Tensor dw = sum(want_w), db = sum(want_b);
    if (t && (want_x || want_w || want_b)) {
      const Tensor ws = want_w || want_b ? floats(x, {api.norm_bwd_ws_floats(t, (int)d)}) : Tensor();
      call(api.norm_bwd(dy.data_ptr(), type_of(dy, "dy"), dy.stride(0), x.data_ptr(), type_of(x, "x"), x.stride(0), ptr(st),
                        ptr(st) + t, ptr(w), t, (int)d, ptr<void>(dx), ptr(ws), ptr(dw), ptr(db), stream_of(x)),
           "scm_norm_bwd");
    }
    return {once(dx), once(dw), once(db), Tensor(), Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps,
                  std::optional<at::ScalarType> out_dtype) {
  const Tensor w = opt(weight), b = opt(bias);
  check_followed({x, w, b});
  if (at::GradMode::is_enabled() && (needs_grad(x) || needs_grad(w) || needs_grad(b)))
    return LayerNorm::apply(x, weight, bias, eps, out_dtype);
  return std::get<0>(norm_fwd(x, w, b, eps, out_dtype, false));
}

// ---------------------------------------------------------------------------- rows of logits
Tensor logits_rows(const Tensor& logits, double temperature, int64_t k) {
  Tensor x = rows_of(logits, "logits");
  TORCH_CHECK_VALUE(x.size(1) <= LOGITS_MAX_V, "logits: at most 2^30 classes (got ", x.size(1), ")");
  TORCH_CHECK_VALUE((float)temperature > 0.f && std::isnormal((float)temperature),   // smaller: 1 / temperature overflows
                    "temperature must be positive, finite and at least 2^-126, got ", temperature);
  TORCH_CHECK_VALUE(k >= 0 && k <= LOGITS_MAX_K, "at most ", LOGITS_MAX_K, " entries per row (got ", k, ")");
  check_device(x, "logits");
  return x;
}
at::DimVector row_shape(const Tensor& logits) {
  const auto s = logits.sizes();
  return at::DimVector(s.begin(), s.end() - 1);
}

struct Score { Tensor logprob, entropy, lse, top_logprob, top_index, tape; };
Score score_fwd(const Tensor& logits, const Tensor& targets_, int64_t k, double temperature, int64_t ignore, bool entropy,
                bool tape) {
  const Tensor x = logits_rows(logits, temperature, k);
  const int64_t t = x.size(0), v = x.size(1);
  TORCH_CHECK_VALUE(k <= v, k, " alternatives of ", v, " classes");
  const Tensor targets = row_vector(targets_, logits, at::kLong, "targets");
  const c10::DeviceGuard guard(x.device());
  at::DimVector shape = row_shape(logits);
  Score o;
  o.lse = floats(x, shape);
  if (targets.defined()) o.logprob = floats(x, shape);
  if (entropy) o.entropy = floats(x, shape);
  if (k) {
    shape.push_back(k);
    o.top_logprob = floats(x, shape);
    o.top_index = at::empty(shape, x.options().dtype(at::kLong));
  }
  if (tape) o.tape = floats(x, {t, 2});
  if (t) {
    const Tensor ws = scratch(x, api.score_ws_floats(t, (int)v, (int)k));
    call(api.score_fwd(x.data_ptr(), type_of(x, "logits"), x.stride(0), t, (int)v, (float)temperature, ptr<int64_t>(targets),
                       ignore, (int)k, ptr(o.logprob), ptr(o.lse), ptr(o.entropy), ptr(o.top_logprob),
                       ptr<int64_t>(o.top_index), ptr(o.tape), ptr(ws), stream_of(x)), "scm_score_fwd");
  }
  return o;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  // the outputs that there are, in the order of Score
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& targets_, int64_t k,
                               double temperature, int64_t ignore, bool entropy) {
    const Tensor targets = opt(targets_);
    Score o = score_fwd(logits, targets, k, temperature, ignore, entropy, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, targets, o.entropy, o.top_index, o.tape});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore"] = ignore;
    variable_list out;
    for (const Tensor& t : {o.logprob, o.entropy, o.lse, o.top_logprob, o.top_index})
      if (t.defined()) out.push_back(t);
    if (k) ctx->mark_non_differentiable({o.top_index});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    for (const Tensor& g : grads) check_followed({g});
    const auto saved = ctx->get_saved_variables();
    check_capture(saved[0]);
    const Tensor &logits = saved[0], &entropy = saved[2], &top_index = saved[3], &tape = saved[4];
    const double temperature = ctx->saved_data["temperature"].toDouble();
    const int64_t k = top_index.defined() ? top_index.size(-1) : 0;
    const Tensor x = rows_of(logits, "logits");
    const Tensor targets = saved[1].defined() ? values(saved[1]).contiguous() : saved[1];
    const int64_t t = x.size(0), v = x.size(1);
    size_t i = 0;
    const Tensor none;
    const Tensor g_lp = grad_rows(targets.defined() ? grads[i++] : none, x, t);
    const Tensor g_ent = grad_rows(entropy.defined() ? grads[i++] : none, x, t);
    const Tensor g_lse = grad_rows(grads[i++], x, t);
    const Tensor g_top = grad_rows(k ? grads[i++] : none, x, t * k);
    const c10::DeviceGuard guard(x.device());
    Tensor dx = at::empty(logits.sizes(), x.options());
    if (t)
      call(api.score_bwd(x.data_ptr(), type_of(x, "logits"), x.stride(0), t, (int)v, (float)temperature,
                         ptr<int64_t>(targets), ctx->saved_data["ignore"].toInt(), (int)k, ptr(tape), ptr(entropy),
                         ptr<int64_t>(top_index), ptr(g_lp), ptr(g_lse), ptr(g_ent), ptr(g_top), dx.data_ptr(),
                         stream_of(x)), "scm_score_bwd");
    return {once(dx), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<OptTensor, OptTensor, Tensor, OptTensor, OptTensor> token_logprobs(const Tensor& logits, const OptTensor& targets_,
                                                                            int64_t k, double temperature, int64_t ignore,
                                                                            bool entropy) {
  const Tensor targets = opt(targets_);
  check_followed({logits, targets});
  auto maybe = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
  if (!(at::GradMode::is_enabled() && logits.requires_grad())) {
    const Score o = score_fwd(logits, targets, k, temperature, ignore, entropy, false);
    return {maybe(o.logprob), maybe(o.entropy), o.lse, maybe(o.top_logprob), maybe(o.top_index)};
  }
  const variable_list out = TokenLogprobs::apply(logits, targets_, k, temperature, ignore, entropy);
  size_t i = 0;
  const OptTensor lp = targets.defined() ? OptTensor(out[i++]) : OptTensor();
  const OptTensor ent = entropy ? OptTensor(out[i++]) : OptTensor();
  const Tensor lse = out[i++];
  return {lp, ent, lse, k ? OptTensor(out[i]) : OptTensor(), k ? OptTensor(out[i + 1]) : OptTensor()};
}

// ---------------------------------------------------------------------------- distillation from top log probabilities
enum Reduction : int64_t { MEAN, SUM, NONE };
Reduction reduction_of(const std::string& r) {
  TORCH_CHECK_VALUE(r == "mean" || r == "sum" || r == "none", "reduction must be 'mean', 'sum' or 'none', got '", r, "'");
  return r == "mean" ? MEAN : r == "sum" ? SUM : NONE;
}
// the operands of one call, contiguous where the kernels want them so
struct Distill {
  Tensor x, index, lp, weight;
  int64_t t, v, k;
  double temperature;
  bool tail;
  Reduction red;

  // checked: the operands of a forward, in its backward
  Distill(const Tensor& logits, const Tensor& index_, const Tensor& lp_, const Tensor& weight_, double temperature_,
          bool tail_, Reduction red_, bool checked)
      : temperature(temperature_), tail(tail_), red(red_) {
    if (!checked) {
      TORCH_CHECK_VALUE(index_.dim() == logits.dim() && logits.dim() >= 1 && index_.sizes() == lp_.sizes() &&
                            index_.sizes().slice(0, logits.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
                        "teacher entries ", index_.sizes(), " and ", lp_.sizes(), " for logits ", logits.sizes());
      TORCH_CHECK_VALUE(index_.size(-1) >= 1, "no teacher entries");
      TORCH_CHECK_TYPE(index_.scalar_type() == at::kLong, "top_index: expected int64, got ", index_.scalar_type());
      TORCH_CHECK_TYPE(lp_.scalar_type() == at::kFloat, "top_logprob: expected float32, got ", lp_.scalar_type());
      TORCH_CHECK_VALUE(!lp_.requires_grad() && !needs_grad(weight_),
                        "the teacher's log probabilities and the weights take no gradient: detach them");
    }
    k = index_.size(-1);
    x = checked ? rows_of(logits, "logits") : logits_rows(logits, temperature, k);
    on_device_of(x, index_, "top_index");
    on_device_of(x, lp_, "top_logprob");
    index = values(index_).contiguous();
    lp = values(lp_).contiguous();
    weight = row_vector(weight_, logits, at::kFloat, "weight");
    t = x.size(0);
    v = x.size(1);
  }
  template <typename F, typename... A>
  int with(F f, A... a) const {
    return f(x.data_ptr(), type_of(x, "logits"), x.stride(0), t, (int)v, (float)temperature, ptr<int64_t>(index), ptr(lp),
             (int)k, (int)tail, ptr(weight), (int)(red == MEAN), a...);
  }
  Tensor no_rows() const {   // an empty sum; its mean is 0 / 0
    return at::full({}, red == MEAN ? std::numeric_limits<double>::quiet_NaN() : 0.0, x.options().dtype(at::kFloat));
  }
  // -> the loss (or the rows' losses, shaped as the logits' rows), what the backward reads: the weights' sum, the tape
  std::tuple<Tensor, Tensor> forward(const Tensor& logits, bool backward_follows) const {
    const c10::DeviceGuard guard(x.device());
    const Tensor out = floats(x, red == NONE ? row_shape(logits) : at::DimVector());
    if (!t) return {red == NONE ? out : no_rows(), Tensor()};
    Tensor keep;
    if (backward_follows) keep = floats(x, {1 + api.topk_distill_tape_floats(t, (int)v, (int)k)});
    const int64_t nws = api.topk_distill_ws_floats(t, (int)v);
    const Tensor ws = scratch(x, nws + (red == NONE ? 0 : t));   // workspace (8-byte aligned), the rows' losses
    float* const rows = red == NONE ? ptr(out) : ptr(ws) + nws;
    call(with(api.topk_distill_fwd, rows, red == NONE ? nullptr : ptr(out), red == NONE ? nullptr : ptr(keep),
              keep.defined() ? ptr(keep) + 1 : nullptr, ptr(ws), stream_of(x)), "scm_topk_distill_fwd");
    return {out, keep};
  }
};

struct TopkDistillation : torch::autograd::Function<TopkDistillation> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& index, const Tensor& lp,
                        const OptTensor& weight_, double temperature, bool tail, int64_t red) {
    const Tensor weight = opt(weight_);
    const Distill op(logits, index, lp, weight, temperature, tail, (Reduction)red, false);
    auto [loss, keep] = op.forward(logits, true);
    ctx->save_for_backward({logits, index, lp, weight, keep});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["opts"] = (int64_t)tail + 2 * red;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_followed({grads[0]});
    const auto saved = ctx->get_saved_variables();
    check_capture(saved[0]);
    const int64_t opts = ctx->saved_data["opts"].toInt();
    const Distill op(saved[0], saved[1], saved[2], saved[3], ctx->saved_data["temperature"].toDouble(), opts & 1,
                     (Reduction)(opts >> 1), true);
    const c10::DeviceGuard guard(op.x.device());
    Tensor dx = at::empty(saved[0].sizes(), op.x.options());
    if (op.t) {
      const bool per_row = op.red == NONE;
      const Tensor g = grad_rows(grads[0], op.x, per_row ? op.t : 1);
      float* const keep = ptr(saved[4]);
      call(op.with(api.topk_distill_bwd, keep, ptr(g), (int)per_row, keep + 1, dx.data_ptr(), stream_of(op.x)),
           "scm_topk_distill_bwd");
    }
    return {once(dx), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor topk_distillation(const Tensor& logits, const Tensor& index, const Tensor& lp, double temperature, bool tail,
                         const OptTensor& weight, const std::string& reduction) {
  const Reduction red = reduction_of(reduction);
  const Tensor w = opt(weight);
  check_followed({logits, index, lp, w});
  if (at::GradMode::is_enabled() && logits.requires_grad())
    return TopkDistillation::apply(logits, index, lp, weight, temperature, tail, (int64_t)red);
  return std::get<0>(Distill(logits, index, lp, w, temperature, tail, red, false).forward(logits, false));
}

std::tuple<Tensor, Tensor> topk_distillation_grad(const Tensor& logits, const Tensor& index, const Tensor& lp,
                                                  double temperature, bool tail, const OptTensor& weight,
                                                  const std::string& reduction, double scale) {
  const Reduction red = reduction_of(reduction);
  TORCH_CHECK_VALUE(red != NONE, "topk_distillation_grad: reduction must be 'mean' or 'sum'");
  const at::NoGradGuard no_grad;
  const Tensor w = opt(weight);
  check_followed({logits, index, lp, w});
  const Distill op(logits, index, lp, w, temperature, tail, red, false);
  const c10::DeviceGuard guard(op.x.device());
  Tensor dx = at::empty(logits.sizes(), op.x.options());
  if (!op.t) return {op.no_rows(), dx};
  Tensor loss = floats(op.x, {});
  // one piece of scratch memory: workspace (8-byte aligned), tape, the rows' losses, the sum of the weights
  const int64_t nws = api.topk_distill_ws_floats(op.t, (int)op.v);
  const int64_t ntape = api.topk_distill_tape_floats(op.t, (int)op.v, (int)op.k);
  const Tensor buf = floats(op.x, {nws + ntape + op.t + 1});
  float* const ws = ptr(buf);
  float* const rows = ws + nws + ntape;
  call(op.with(api.topk_distill_step, (float)scale, rows, ptr(loss), rows + op.t, ws + nws, ws, dx.data_ptr(),
               stream_of(op.x)), "scm_topk_distill_step");
  return {loss, dx};
}

// address(name) -> the entry point's address in the loaded library
void bind(const py::function& address) {
#define SCM_BIND(f) api.f = reinterpret_cast<decltype(api.f)>(address("scm_" #f).cast<uintptr_t>())
  SCM_BIND(last_error);
  SCM_BIND(norm_fwd);
  SCM_BIND(norm_bwd);
  SCM_BIND(norm_bwd_ws_floats);
  SCM_BIND(score_ws_floats);
  SCM_BIND(score_fwd);
  SCM_BIND(score_bwd);
  SCM_BIND(topk_distill_tape_floats);
  SCM_BIND(topk_distill_ws_floats);
  SCM_BIND(topk_distill_fwd);
  SCM_BIND(topk_distill_bwd);
  SCM_BIND(topk_distill_step);
#undef SCM_BIND
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  py::register_local_exception_translator([](std::exception_ptr p) {   // the package's kinds of errors, without a C++ trace
    try {
      if (p) std::rethrow_exception(p);
    } catch (const c10::TypeError& e) {
      PyErr_SetString(PyExc_TypeError, e.what_without_backtrace());
    } catch (const c10::ValueError& e) {
      PyErr_SetString(PyExc_ValueError, e.what_without_backtrace());
    } catch (const c10::NotImplementedError& e) {
      PyErr_SetString(PyExc_NotImplementedError, e.what_without_backtrace());
    }
  });
  m.def("bind", &bind);
  const auto free = py::call_guard<py::gil_scoped_release>();
  m.def("layer_norm", &layer_norm, free, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"),
        py::arg("out_dtype"));
  m.def("token_logprobs", &token_logprobs, free);
  m.def("topk_distillation", &topk_distillation, free);
  m.def("topk_distillation_grad", &topk_distillation_grad, free);
}
