// Autograd functions of the token-wise operators over the C ABI (include/vg_api.h), as the extension module
// vae_gan_amd/_vgtorch.so.  In C++ because these operators are called many times a step on small tensors: a Python autograd
// function costs some 20 us of host time forward and 45 backward around kernels of 5 to 20 us, these 6 and 12.
// Each checks its arguments, allocates its outputs and workspaces from torch's allocator and enqueues on the current stream
// of its tensors' device.  None differentiates twice, carries forward-mode tangents or can be traced: each refuses.
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "../../include/vg_api.h"

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

namespace {

int vg_dtype(const char* what, const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return VG_BF16;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, what, ": unsupported activation dtype ", t.scalar_type());
  return VG_F32;
}
void on_device(const char* what, const Tensor& x, std::initializer_list<const Tensor*> others) {
  TORCH_CHECK(x.is_cuda(), what, ": the HIP path needs a tensor on an MI355X device (got ", x.device(), "); there is no CPU fallback");
  for (const Tensor* t : others)
    TORCH_CHECK(!t->defined() || t->device() == x.device(), what, ": tensors on ", x.device(), " and ", t->device());
}
void ok(int rc, const char* what) { TORCH_CHECK(rc == VG_OK, "libvg_hip ", what, " failed (rc=", rc, "): ", vg_last_error()); }
void* stream() { return (void*)c10::hip::getCurrentHIPStream().stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor bytes(size_t n, const Tensor& like) { return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor(); }
void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": cannot be differentiated twice (create_graph=True)");
}
// What launches kernels on memory cannot pass on a tangent (a result without one reads as a derivative of zero), and a trace of it
// would hold the allocation of its result alone.
void eager_only(const char* what, std::initializer_list<const Tensor*> ts) {
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), what, ": cannot be traced (torch.jit.trace)");
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what, ": has no forward-mode derivative (torch.autograd.forward_ad)");
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// t as rows of its last dimension, contiguous within a row, with one row stride; a copy only where no single stride does
struct Rows {
  Tensor t;
  int64_t n, ld;
};
Rows rows_of(const Tensor& t) {
  const int64_t c = t.size(-1);
  if (t.is_contiguous()) return {t, t.numel() / c, c};
  Tensor r = t.reshape({-1, c});
  if ((c > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < c)) r = r.contiguous();
  return {r, r.size(0), r.size(0) > 1 ? r.stride(0) : c};
}

// ---- layer norm -------------------------------------------------------------------------------------------------------
Tensor layer_norm_run(const Rows& x, const Tensor& like, const Tensor& w, const Tensor& b, double eps, int64_t c, const Tensor& stats) {
  Tensor y = at::empty(like.sizes(), like.options());
  const int64_t cs = like.size(-1);
  ok(vg_layer_norm_fwd(ptr(x.t), x.ld, (const float*)ptr(w), (const float*)ptr(b), ptr(y), cs, (float*)ptr(stats), x.n, (int)c, (int)cs,
                       (float)eps, vg_dtype("layer_norm", like), stream()),
     "layer_norm_fwd");
  return y;
}
struct LayerNorm : Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, int64_t c) {
    const Rows r = rows_of(x);
    const Tensor w = weight.contiguous(), b = bias.contiguous();
    const Tensor stats = at::empty({r.n, 2}, x.options().dtype(at::kFloat));
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["c"] = c;
    return layer_norm_run(r, x, w, b, eps, c, stats);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("layer_norm");
    eager_only("layer_norm", {&g[0]});
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    const c10::DeviceGuard guard(x.device());
    const int64_t c = ctx->saved_data["c"].toInt(), cs = x.size(-1);
    const Rows r = rows_of(x), d = rows_of(g[0]);
    Tensor dx, dw, db, ws;
    if (ctx->needs_input_grad(0)) dx = at::empty(x.sizes(), x.options());
    if (ctx->needs_input_grad(1)) dw = at::empty({c}, w.options());
    if (ctx->needs_input_grad(2)) db = at::empty({c}, w.options());
    if (r.n == 0) {
      if (dw.defined()) dw.zero_();
      if (db.defined()) db.zero_();
      return {dx, dw, db, Tensor(), Tensor()};
    }
    if (dw.defined() || db.defined()) ws = bytes(vg_layer_norm_bwd_ws_bytes(r.n, (int)c), x);
    ok(vg_layer_norm_bwd(ptr(r.t), r.ld, ptr(d.t), d.ld, (const float*)ptr(w), (const float*)ptr(stats), ptr(dx), cs, (float*)ptr(dw),
                         (float*)ptr(db), ptr(ws), r.n, (int)c, (int)cs, vg_dtype("layer_norm", x), stream()),
       "layer_norm_bwd");
    return {dx, dw, db, Tensor(), Tensor()};
  }
};
Tensor layer_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, std::optional<int64_t> columns) {
  eager_only("layer_norm", {&x, &weight, &bias});
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "layer_norm: no columns in a tensor of shape ", x.sizes());
  TORCH_CHECK(x.size(-1) <= (1 << 24), "layer_norm: ", x.size(-1), " columns in a row");
  const int64_t c = columns.value_or(x.size(-1));
  TORCH_CHECK(c >= 1 && c <= x.size(-1), "layer_norm: c = ", c, " of ", x.size(-1), " columns");
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"weight", weight}, {"bias", bias}})
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == c, "layer_norm: ", name, " must be float32 [", c, "], got ",
                t.scalar_type(), " ", t.sizes());
  TORCH_CHECK_VALUE(eps >= 0, "layer_norm: eps = ", eps);
  vg_dtype("layer_norm", x);
  on_device("layer_norm", x, {&weight, &bias});
  const c10::DeviceGuard guard(x.device());
  if (!wants_grad({&x, &weight, &bias})) return layer_norm_run(rows_of(x), x, weight.contiguous(), bias.contiguous(), eps, c, Tensor());
  return LayerNorm::apply(x, weight, bias, eps, c);
}

// ---- product with bias, activation and residual --------------------------------------------------------------------------
Tensor linear_act_run(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& residual, int64_t act, Tensor* slope) {
  const int dt = vg_dtype("linear_act", x), wdt = vg_dtype("linear_act", w);
  const Rows r = rows_of(x);
  const int64_t n = w.size(0), k = w.size(1);
  auto sizes = x.sizes().vec();
  sizes.back() = n;
  Tensor y = at::empty(sizes, x.options());
  if (r.n == 0) return y;
  const Tensor b = bias.defined() ? bias.contiguous() : bias;
  const Rows res = residual.defined() ? rows_of(residual) : Rows{Tensor(), 0, 0};
  if (slope) *slope = at::empty({r.n, n}, x.options().dtype(dt == VG_BF16 ? at::kHalf : at::kFloat));
  const Tensor ws = bytes(vg_linear_act_fwd_ws_bytes(ptr(r.t), r.ld, ptr(w), wdt, r.n, n, k, dt), x);
  ok(vg_linear_act_fwd(ptr(r.t), r.ld, ptr(w), wdt, ptr(b), b.defined() ? vg_dtype("linear_act", b) : 0, ptr(res.t), res.ld, ptr(y),
                       slope ? ptr(*slope) : nullptr, ptr(ws), r.n, n, k, (int)act, dt, stream()),
     "linear_act_fwd");
  return y;
}
struct LinearAct : Function<LinearAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_,
                        const std::optional<Tensor>& residual_, int64_t act, bool slopes) {
    const Tensor bias = bias_.value_or(Tensor()), residual = residual_.value_or(Tensor());
    const Tensor w = weight.contiguous();
    Tensor slope;
    Tensor y = linear_act_run(x, w, bias, residual, act, slopes ? &slope : nullptr);
    ctx->save_for_backward({x, w, slope});
    ctx->saved_data["bias"] = (int64_t)(!bias.defined() ? 0 : bias.scalar_type() == at::kFloat ? 2 : 1);
    ctx->saved_data["residual"] = residual.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gs) {
    once("linear_act");
    eager_only("linear_act", {&gs[0]});
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &slope = saved[2];
    const c10::DeviceGuard guard(x.device());
    const int dt = vg_dtype("linear_act", x), wdt = vg_dtype("linear_act", w);
    const int64_t has_b = ctx->saved_data["bias"].toInt();       // absent tensors have no edge of their own
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(2);
    const bool f32b = has_b == 2;
    const int64_t n = w.size(0), k = w.size(1);
    const Rows r = rows_of(x);
    const int64_t m = r.n;
    Tensor dx, dw, db, dres;
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(has_b ? 3 : 2)) dres = gs[0];
    if (need_x) dx = at::empty(x.sizes(), x.options());
    if (need_w) dw = at::empty({n, k}, w.options());
    if (need_b) db = at::empty({n}, x.options().dtype(f32b ? at::kFloat : x.scalar_type()));
    if (m == 0) {
      if (need_w) dw.zero_();
      if (need_b) db.zero_();
      return {dx, dw, db, dres, Tensor(), Tensor()};
    }
    const Tensor g = gs[0].contiguous();
    Tensor dz = g;
    const bool sloped = slope.defined() && (need_x || need_w || need_b);
    if (sloped) dz = at::empty({m, n}, x.options());
    // one workspace for the three calls: they follow each other on the stream
    size_t need = need_b ? vg_linear_act_dz_ws_bytes(m, n) : 0;
    if (need_x) need = std::max(need, vg_linear_act_dgrad_ws_bytes(ptr(dz), ptr(w), wdt, m, n, k, dt));
    if (need_w) need = std::max(need, vg_linear_act_wgrad_ws_bytes(ptr(dz), ptr(r.t), r.ld, m, n, k, dt));
    const Tensor ws = bytes(need, x);
    if (sloped || need_b)
      ok(vg_linear_act_dz(ptr(g), ptr(slope), ptr(dz), ptr(db), f32b ? VG_F32 : dt, ptr(ws), m, n, dt, stream()), "linear_act_dz");
    if (need_x) ok(vg_linear_act_dgrad(ptr(dz), ptr(w), wdt, ptr(dx), ptr(ws), m, n, k, dt, stream()), "linear_act_dgrad");
    if (need_w) ok(vg_linear_act_wgrad(ptr(dz), ptr(r.t), r.ld, ptr(dw), wdt, ptr(ws), m, n, k, dt, stream()), "linear_act_wgrad");
    return {dx, dw, db, dres, Tensor(), Tensor()};
  }
};
Tensor linear_act(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_, int64_t act, const std::optional<Tensor>& residual_) {
  const Tensor bias = bias_.value_or(Tensor()), residual = residual_.value_or(Tensor());
  eager_only("linear_act", {&x, &weight, &bias, &residual});
  TORCH_CHECK(x.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x.size(-1) && weight.numel() > 0,
              "linear_act: mat1 and mat2 shapes cannot be multiplied (", x.sizes(), " and ", weight.sizes(), " transposed)");
  vg_dtype("linear_act", x);
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"weight", weight}, {"bias", bias}})
    TORCH_CHECK_TYPE(!t.defined() || t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, "linear_act: ", name, " is ",
                     t.scalar_type(), ", x is ", x.scalar_type(), " (the same or float32 is supported)");
  const int64_t n = weight.size(0);
  TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == n), "linear_act: bias of shape ", bias.sizes(), " for ", n, " outputs");
  if (residual.defined()) {
    auto want = x.sizes().vec();
    want.back() = n;
    TORCH_CHECK(residual.scalar_type() == x.scalar_type() && residual.sizes() == want, "linear_act: residual is ", residual.scalar_type(), " ",
                residual.sizes(), ", the result ", x.scalar_type(), " ", want);
  }
  TORCH_CHECK_VALUE(act >= VG_ACT_NONE && act <= VG_ACT_SILU, "linear_act: activation ", act);
  on_device("linear_act", x, {&weight, &bias, &residual});
  const c10::DeviceGuard guard(x.device());
  if (!wants_grad({&x, &weight, &bias, &residual})) return linear_act_run(x, weight.contiguous(), bias, residual, act, nullptr);
  return LinearAct::apply(x, weight, bias_, residual_, act, act != VG_ACT_NONE && wants_grad({&x, &weight, &bias}));
}

// ---- log probabilities of tokens -------------------------------------------------------------------------------------------
variable_list token_logprobs_run(const Tensor& logits, const Tensor& tokens, int64_t top, int64_t ignore, const Tensor& lse) {
  const Rows r = rows_of(logits);
  const int64_t vocab = logits.size(-1);
  const auto lead = tokens.sizes();
  const auto f32 = logits.options().dtype(at::kFloat);
  Tensor logp = at::empty(lead, f32), entropy = at::empty(lead, f32), top_logp, top_at;
  if (top) {
    auto s = lead.vec();
    s.push_back(top);
    top_logp = at::empty(s, f32);
    top_at = at::empty(s, f32.dtype(at::kLong));
  }
  if (r.n) {
    const Tensor ws = bytes(vg_token_logprobs_ws_bytes(r.n, (int)vocab, (int)top), logits);
    ok(vg_token_logprobs_fwd(ptr(r.t), r.ld, (const int64_t*)ptr(tokens), ignore, r.n, (int)vocab, (int)top, (float*)ptr(logp),
                             (float*)ptr(entropy), (float*)ptr(lse), (float*)ptr(top_logp), (int64_t*)ptr(top_at), ptr(ws),
                             vg_dtype("token_logprobs", logits), stream()),
       "token_logprobs_fwd");
  }
  if (top) return {logp, entropy, top_logp, top_at};
  return {logp, entropy};
}
struct TokenLogprobs : Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, int64_t top, int64_t ignore) {
    ctx->set_materialize_grads(false);
    const Tensor lse = at::empty({tokens.numel(), 2}, logits.options().dtype(at::kFloat));
    variable_list out = token_logprobs_run(logits, tokens, top, ignore, lse);
    ctx->save_for_backward({logits, tokens, lse, out[1]});
    ctx->saved_data["ignore"] = ignore;
    if (top) ctx->mark_non_differentiable({out[2], out[3]});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("token_logprobs");
    eager_only("token_logprobs", {&g[0], &g[1]});
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &tokens = saved[1], &lse = saved[2], &entropy = saved[3];
    const c10::DeviceGuard guard(logits.device());
    const Rows r = rows_of(logits);
    const int64_t vocab = logits.size(-1);
    if (!g[0].defined() && !g[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    // rows laid out like the logits' own: the two are then aligned alike
    const int64_t ld = r.ld <= vocab + 256 ? r.ld : vocab;
    Tensor dx;
    if (ld == vocab) dx = at::empty(logits.sizes(), logits.options());
    else dx = at::empty({r.n, ld}, logits.options()).narrow(1, 0, vocab).unflatten(0, tokens.sizes());
    if (r.n) {
      const Tensor a = g[0].defined() ? g[0].to(at::kFloat).contiguous() : Tensor(), b = g[1].defined() ? g[1].to(at::kFloat).contiguous() : Tensor();
      ok(vg_token_logprobs_bwd(ptr(r.t), r.ld, (const int64_t*)ptr(tokens), ctx->saved_data["ignore"].toInt(), (const float*)ptr(lse),
                               (const float*)ptr(entropy), (const float*)ptr(a), (const float*)ptr(b), ptr(dx), ld, r.n, (int)vocab,
                               vg_dtype("token_logprobs", logits), stream()),
         "token_logprobs_bwd");
    }
    return {dx, Tensor(), Tensor(), Tensor()};
  }
};
variable_list token_logprobs(const Tensor& logits, const Tensor& tokens, int64_t top, int64_t ignore) {
  constexpr int64_t most = 32;
  eager_only("token_logprobs", {&logits});
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1, "token_logprobs: no logits in a tensor of shape ", logits.sizes());
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK(tokens.scalar_type() == at::kLong && tokens.sizes() == lead, "token_logprobs: tokens must be int64 ", lead, ", got ",
              tokens.scalar_type(), " ", tokens.sizes());
  TORCH_CHECK_VALUE(top >= 0 && top <= std::min(most, logits.size(-1)), "token_logprobs: top = ", top, " of ", logits.size(-1),
                    " logits (at most ", most, ")");
  TORCH_CHECK(logits.size(-1) <= (1 << 30), "token_logprobs: ", logits.size(-1), " logits in a row");
  vg_dtype("token_logprobs", logits);
  on_device("token_logprobs", logits, {&tokens});
  const c10::DeviceGuard guard(logits.device());
  const Tensor t = tokens.contiguous();
  if (!wants_grad({&logits})) return token_logprobs_run(logits, t, top, ignore, Tensor());
  return TokenLogprobs::apply(logits, t, top, ignore);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
  m.def("linear_act", &linear_act, py::call_guard<py::gil_scoped_release>());
  m.def("token_logprobs", &token_logprobs, py::call_guard<py::gil_scoped_release>());
}
