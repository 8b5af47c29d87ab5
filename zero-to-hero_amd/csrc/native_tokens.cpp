// The token operators' host path in ppo_amd._native: tokens.py's functions for
// the ordinary call (plain contiguous tensors on one GPU), and their autograd
// nodes, so that neither direction runs in the interpreter.  Any other call
// returns None and takes tokens.py's checks.
//
// Measured on MI355X, us a call among others, through Python and here: log-probabilities
// of 256 x 18 18 and 5.5, the policy loss of 528 x 500 with its gradient 167 and 67 (of
// which torch's engine takes half), the preference loss of 248 x 1000 160 and 61.
#include "native.hpp"

#include <c10/core/DeviceGuard.h>
#include <hip/hip_runtime.h>

#include <cmath>

#include "ppo_tokens.h"

namespace ppo_native {
namespace {

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return PPO_DTYPE_F32;
    case at::kBFloat16: return PPO_DTYPE_BF16;
    case at::kHalf: return PPO_DTYPE_F16;
    default: return -1;
  }
}

at::ScalarType type_of(PyObject* o) {
  need(THPVariable_CheckExact(o));
  return THPVariable_Unpack(o).scalar_type();
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const float* floats(const Tensor& t) { return static_cast<const float*>(ptr(t)); }

Tensor bytes(size_t n, const at::Device& device) {
  if (!n) return {};
  return at::empty({(int64_t)n}, at::TensorOptions().dtype(at::kByte).device(device));
}

// The capture that a device's current stream is in, 0 if none.
int64_t capture_of(const at::Device& device) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  const hipError_t e = hipStreamGetCaptureInfo(
      c10::hip::getCurrentHIPStream(device.index()).stream(), &status, &id);
  TORCH_CHECK(e == hipSuccess, "hipStreamGetCaptureInfo: ", hipGetErrorString(e));
  return status == hipStreamCaptureStatusNone ? 0 : (int64_t)id;
}

PyObject* capture_id(PyObject*, PyObject* index) {
  const long device = PyLong_AsLong(index);
  if (device == -1 && PyErr_Occurred()) return nullptr;
  try {
    return PyLong_FromLongLong(capture_of(at::Device(at::kCUDA, (c10::DeviceIndex)device)));
  } catch (const std::exception&) {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

// An operand that has no gradient here: where it asks for one, tokens.py refuses it.
const Tensor& constant(const Tensor& t) {
  need(!t._fw_grad(0).defined() && !(at::GradMode::is_enabled() && t.requires_grad()));
  return t;
}

// Logits and what every row of them has: actions (int32 or int64; undefined for a
// distilled row) and a mask (bool or uint8; undefined: every row counts).
struct Rows {
  Tensor logits, actions, mask;
  double tau = 1.0;

  Rows() = default;
  Rows(PyObject* x, PyObject* a, PyObject* m, PyObject* temperature) {
    const at::ScalarType type = type_of(x);
    need(dtype_code(type) >= 0);
    logits = plain(x, type);
    need(logits.dim() >= 1 && logits.numel() > 0);
    need(!logits._fw_grad(0).defined());
    if (a) {
      const at::ScalarType t = type_of(a);
      need(t == at::kInt || t == at::kLong);
      actions = row_tensor(a, t);
    }
    if (m != Py_None) {
      const at::ScalarType t = type_of(m);
      need(t == at::kBool || t == at::kByte);
      mask = row_tensor(m, t);
    }
    tau = number(temperature);
    need(tau > 0.0 && std::isfinite(tau));
  }
  at::Device device() const { return logits.device(); }
  at::IntArrayRef shape() const { return logits.sizes().slice(0, logits.dim() - 1); }
  int64_t A() const { return logits.size(-1); }
  int64_t n() const { return logits.numel() / A(); }
  int64_t tokens() const { return logits.dim() >= 2 ? logits.size(-2) : 1; }
  int64_t sequences() const { return n() / tokens(); }
  int dtype() const { return dtype_code(logits.scalar_type()); }
  at::TensorOptions f32() const { return logits.options().dtype(at::kFloat); }
  Tensor row_tensor(PyObject* o, at::ScalarType t) const {
    const Tensor& r = plain(o, t, device());
    need(r.sizes() == shape());
    return r;
  }
  Tensor row_constants(PyObject* o) const { return constant(row_tensor(o, at::kFloat)); }
  ppo_token_rows c() const {
    return {logits.const_data_ptr(), ptr(actions), static_cast<const uint8_t*>(ptr(mask)),
            sequences(), tokens(), A(), dtype(),
            actions.defined() && actions.scalar_type() == at::kLong, tau};
  }
  Tensor scratch() const {
    return bytes(ppo_token_workspace_bytes(sequences(), tokens(), A(), dtype()), device());
  }
  Tensor saved() const { return at::empty({n(), PPO_TOKEN_SAVED}, f32()); }
  bool differentiable() const { return at::GradMode::is_enabled() && logits.requires_grad(); }
};

// What a backward pass got back or was handed: as the forward had it, or a clear
// error (a saved-tensor hook may return anything).
Tensor like_forward(const Tensor& t, at::ScalarType type, at::IntArrayRef shape,
                    const at::Device& device, const char* what) {
  TORCH_CHECK(t.device() == device && t.scalar_type() == type && t.sizes() == shape &&
                  t.layout() == at::kStrided && !t.key_set().has_any(kWrapped),
              what, ": a saved tensor came back as ", t.scalar_type(), " ", t.sizes(), " on ",
              t.device(), ", expected ", type, " ", shape, " on ", device);
  return t.contiguous();
}

void save_rows(AutogradContext* ctx, const Rows& r, std::initializer_list<Tensor> more) {
  variable_list v = {r.logits, r.actions, r.mask};
  v.insert(v.end(), more.begin(), more.end());
  ctx->save_for_backward(std::move(v));
  ctx->set_materialize_grads(false);
  ctx->saved_data["tau"] = r.tau;
  ctx->saved_data["shape"] = r.logits.sizes().vec();
  ctx->saved_data["type"] = (int64_t)r.logits.scalar_type();
  ctx->saved_data["device"] = (int64_t)r.device().index();
}

Rows saved_rows(AutogradContext* ctx, const variable_list& v, const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what,
              " can be differentiated once: its backward pass has no create_graph");
  Rows r;
  const at::Device device(at::kCUDA, (c10::DeviceIndex)ctx->saved_data["device"].toInt());
  const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
  const at::IntArrayRef rows = at::IntArrayRef(shape).slice(0, shape.size() - 1);
  r.tau = ctx->saved_data["tau"].toDouble();
  r.logits = like_forward(v[0], (at::ScalarType)ctx->saved_data["type"].toInt(), shape, device, what);
  if (v[1].defined()) {
    TORCH_CHECK(v[1].scalar_type() == at::kInt || v[1].scalar_type() == at::kLong, what,
                ": the saved actions came back as ", v[1].scalar_type());
    r.actions = like_forward(v[1], v[1].scalar_type(), rows, device, what);
  }
  if (v[2].defined()) {
    TORCH_CHECK(v[2].scalar_type() == at::kBool || v[2].scalar_type() == at::kByte, what,
                ": the saved mask came back as ", v[2].scalar_type());
    r.mask = like_forward(v[2], v[2].scalar_type(), rows, device, what);
  }
  return r;
}

// An incoming gradient in fp32.
Tensor incoming(const Tensor& g, at::IntArrayRef shape, const at::Device& device,
                const char* what) {
  TORCH_CHECK(g.device() == device && g.sizes() == shape && g.layout() == at::kStrided &&
                  !g.key_set().has_any(kWrapped),
              what, ": the incoming gradient is ", g.sizes(), " on ", g.device(), ", expected ",
              shape, " on ", device);
  return g.to(at::kFloat).contiguous();
}

// A gradient that the forward pass formed for an incoming gradient of `value`
// (tokens._Held): the first backward pass outside other captures may take it.
void hold(AutogradContext* ctx, const Tensor& grad, double value) {
  ctx->saved_data["held"] = grad;
  ctx->saved_data["value"] = value;
  ctx->saved_data["capture"] = capture_of(grad.device());
}
Tensor take_held(AutogradContext* ctx, const at::Device& device) {
  const auto it = ctx->saved_data.find("held");
  if (it == ctx->saved_data.end()) return {};
  Tensor grad = it->second.toTensor();
  ctx->saved_data.erase(it);
  return capture_of(device) == ctx->saved_data["capture"].toInt() ? grad : Tensor();
}

// --- log-probabilities -----------------------------------------------------------------

int log_probs(const Rows& r, const Tensor& minus, Tensor& lp, Tensor* H, Tensor* saved) {
  const c10::DeviceGuard guard(r.device());
  lp = at::empty(r.shape(), r.f32());
  if (H) *H = at::empty(r.shape(), r.f32());
  if (saved) *saved = r.saved();
  const Tensor ws = r.scratch();
  const ppo_token_rows c = r.c();
  return ppo_token_log_probs(&c, floats(minus), lp.data_ptr<float>(),
                             H ? H->data_ptr<float>() : nullptr,
                             saved ? saved->data_ptr<float>() : nullptr, ptr(ws), ws.numel(),
                             current_stream(r.device()));
}

Tensor log_probs_backward(const Rows& r, const Tensor& saved, const float* dlp, const float* dH,
                          const Tensor& scale, const Tensor& held, double value) {
  const c10::DeviceGuard guard(r.device());
  const Tensor d = held.defined() ? held : at::empty_like(r.logits);
  const ppo_token_rows c = r.c();
  const int code = ppo_token_log_probs_backward(&c, floats(saved), dlp, dH, floats(scale),
                                                held.defined() ? value : 0.0, d.data_ptr(),
                                                current_stream(r.device()));
  check_in_node("ppo_token_log_probs_backward", code, r.device(), current_stream(r.device()));
  return d;
}

struct LogProbsNode : public torch::autograd::Function<LogProbsNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor&, const Rows* r, bool entropy) {
    Tensor lp, H, saved;
    check_in_node("ppo_token_log_probs",
                  log_probs(*r, Tensor(), lp, entropy ? &H : nullptr, &saved), r->device(),
                  current_stream(r->device()));
    save_rows(ctx, *r, {saved});
    if (!entropy) return {lp};
    return {lp, H};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    constexpr const char* what = "token_log_probs";
    const variable_list v = ctx->get_saved_variables();
    const Rows r = saved_rows(ctx, v, what);
    Tensor dlp, dH;
    if (g[0].defined()) dlp = incoming(g[0], r.shape(), r.device(), what);
    if (g.size() > 1 && g[1].defined()) dH = incoming(g[1], r.shape(), r.device(), what);
    if (!dlp.defined() && !dH.defined()) return variable_list(3);
    const Tensor saved = like_forward(v[3], at::kFloat, {r.n(), PPO_TOKEN_SAVED}, r.device(), what);
    return {log_probs_backward(r, saved, floats(dlp), floats(dH), Tensor(), Tensor(), 0.0),
            Tensor(), Tensor()};
  }
};

PyObject* token_log_probs(PyObject* const* a) {  // logits, actions, mask, temperature, entropy
  const Rows r(a[0], a[1], a[2], a[3]);
  need(PyBool_Check(a[4]));
  const bool entropy = a[4] == Py_True;
  if (r.differentiable()) {
    variable_list out;
    unlocked([&] { return out = LogProbsNode::apply(r.logits, &r, entropy), 0; });
    return entropy ? tuple_of({out[0], out[1]}) : wrap(out[0]);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor lp, H;
  const int code =
      unlocked([&] { return log_probs(r, Tensor(), lp, entropy ? &H : nullptr, nullptr); });
  check("ppo_token_log_probs", code, r.device(), current_stream(r.device()));
  return entropy ? tuple_of({lp, H}) : wrap(lp);
}

// --- losses ------------------------------------------------------------------------------

// Element i of a 1-D fp32 tensor as a 0-d tensor on the same storage (no autograd
// view).
Tensor element(const Tensor& t, int64_t i) {
  auto impl =
      c10::make_intrusive<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
  impl->set_sizes_contiguous(at::IntArrayRef{});
  impl->set_storage_offset(t.storage_offset() + i);
  return Tensor(std::move(impl));
}

PyObject* pair(const Tensor& first, PyObject* second) {
  py::object rest = py::reinterpret_steal<py::object>(second);
  py::tuple r(2);
  PyTuple_SET_ITEM(r.ptr(), 0, wrap(first));
  PyTuple_SET_ITEM(r.ptr(), 1, rest.release().ptr());
  return r.release().ptr();
}

double held(PyObject* o) {
  const double x = number(o);
  need(x >= PPO_TOKEN_LEAST && x <= PPO_TOKEN_MOST);
  return x;
}
double finite(PyObject* o) {
  const double x = number(o);
  need(std::isfinite(x));
  return x;
}
double coefficient(PyObject* o) {
  const double x = number(o);
  need(std::isfinite((float)x));
  return x;
}

// reduction, denominator, grad_scale
void weights_of(PyObject* const* a, ppo_token_loss& l) {
  l.reduction = (int)integer(a[0]);
  l.denominator = a[1] == Py_None ? 0.0 : held(a[1]);
  l.grad_scale = held(a[2]);
}

struct Policy {
  Rows r;
  Tensor old, adv, ref;
  ppo_token_loss l = {};
};

int policy(const Policy& p, Tensor& scalars, Tensor* saved, Tensor* coef, Tensor* d) {
  const c10::DeviceGuard guard(p.r.device());
  scalars = at::empty({PPO_TOKEN_SCALARS}, p.r.f32());
  if (saved) {
    *saved = p.r.saved();
    *coef = at::empty({2, p.r.n()}, p.r.f32());
    *d = at::empty_like(p.r.logits);
  }
  const Tensor ws = p.r.scratch();
  const ppo_token_rows c = p.r.c();
  return ppo_token_policy_loss(&c, floats(p.old), floats(p.adv), floats(p.ref), &p.l,
                               scalars.data_ptr<float>(), saved ? saved->data_ptr<float>() : nullptr,
                               saved ? coef->data_ptr<float>() : nullptr,
                               saved ? d->data_ptr() : nullptr, ptr(ws), ws.numel(),
                               current_stream(p.r.device()));
}

struct PolicyNode : public torch::autograd::Function<PolicyNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor&, const Policy* p, Tensor* scalars) {
    Tensor saved, coef, d;
    check_in_node("ppo_token_policy_loss", policy(*p, *scalars, &saved, &coef, &d), p->r.device(),
                  current_stream(p->r.device()));
    save_rows(ctx, p->r, {saved, coef});
    hold(ctx, d, p->l.grad_scale);
    return element(*scalars, PPO_TOKEN_SCALAR_LOSS);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    constexpr const char* what = "token_policy_loss";
    const variable_list v = ctx->get_saved_variables();
    const Rows r = saved_rows(ctx, v, what);
    if (!g[0].defined()) return variable_list(3);
    const Tensor scale = incoming(g[0], {}, r.device(), what);
    const Tensor saved = like_forward(v[3], at::kFloat, {r.n(), PPO_TOKEN_SAVED}, r.device(), what),
                 coef = like_forward(v[4], at::kFloat, {2, r.n()}, r.device(), what);
    const float* c = floats(coef);
    const Tensor held = take_held(ctx, r.device());
    return {log_probs_backward(r, saved, c, c + r.n(), scale, held,
                               ctx->saved_data["value"].toDouble()),
            Tensor(), Tensor()};
  }
};

// logits, actions, old, adv, ref, mask, clip_low, clip_high, kl_coef, entropy_coef,
// temperature, reduction, denominator, grad_scale -> (loss, the scalars)
PyObject* token_policy_loss(PyObject* const* a) {
  Policy p;
  p.r = Rows(a[0], a[1], a[5], a[10]);
  p.old = p.r.row_constants(a[2]);
  p.adv = constant(plain(a[3], at::kFloat, p.r.device()));
  const at::IntArrayRef rows = p.r.shape();
  p.l.advantages_per_sequence =
      !rows.empty() && p.adv.sizes() == rows.slice(0, rows.size() - 1);
  need(p.l.advantages_per_sequence || p.adv.sizes() == rows);
  if (a[4] != Py_None) p.ref = p.r.row_constants(a[4]);
  p.l.clip_low = number(a[6]);
  p.l.clip_high = number(a[7]);
  p.l.kl_coef = coefficient(a[8]);
  p.l.entropy_coef = coefficient(a[9]);
  need(p.l.clip_low >= 0.0 && p.l.clip_high >= 0.0);
  need(p.l.kl_coef == 0.0 || p.ref.defined());
  weights_of(a + 11, p.l);
  Tensor scalars, loss;
  if (p.r.differentiable()) {
    unlocked([&] { return loss = PolicyNode::apply(p.r.logits, &p, &scalars), 0; });
  } else {
    at::AutoDispatchBelowADInplaceOrView below;
    const int code = unlocked([&] { return policy(p, scalars, nullptr, nullptr, nullptr); });
    check("ppo_token_policy_loss", code, p.r.device(), current_stream(p.r.device()));
    loss = element(scalars, PPO_TOKEN_SCALAR_LOSS);
  }
  static_assert(PPO_TOKEN_SCALARS == 6, "");
  return pair(loss, tuple_of({element(scalars, 0), element(scalars, 1), element(scalars, 2),
                              element(scalars, 3), element(scalars, 4), element(scalars, 5)}));
}

struct Preference {
  Rows r;
  Tensor ref;
  double beta, smoothing, margin;
  bool average;
};

int preference(const Preference& p, Tensor& loss, Tensor& rewards, Tensor& coef, Tensor* saved) {
  const c10::DeviceGuard guard(p.r.device());
  void* stream = current_stream(p.r.device());
  Tensor relative;
  if (const int code = log_probs(p.r, p.ref, relative, nullptr, saved)) return code;
  const int64_t S = p.r.sequences();
  loss = at::empty({}, p.r.f32());
  rewards = at::empty({S}, p.r.f32());
  coef = at::empty(p.r.shape(), p.r.f32());
  const size_t n = ppo_token_preference_workspace_bytes(S);
  const Tensor ws = bytes(n, p.r.device());
  return ppo_token_preference(floats(relative), static_cast<const uint8_t*>(ptr(p.r.mask)), S,
                              p.r.tokens(), p.beta, p.margin, p.smoothing, p.average,
                              loss.data_ptr<float>(), rewards.data_ptr<float>(),
                              coef.data_ptr<float>(), ptr(ws), n, stream);
}

struct PreferenceNode : public torch::autograd::Function<PreferenceNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor&, const Preference* p, Tensor* rewards) {
    Tensor loss, coef, saved;
    check_in_node("ppo_token_preference", preference(*p, loss, *rewards, coef, &saved),
                  p->r.device(), current_stream(p->r.device()));
    save_rows(ctx, p->r, {saved, coef});
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    constexpr const char* what = "preference_loss";
    const variable_list v = ctx->get_saved_variables();
    const Rows r = saved_rows(ctx, v, what);
    if (!g[0].defined()) return variable_list(3);
    const Tensor scale = incoming(g[0], {}, r.device(), what);
    const Tensor saved = like_forward(v[3], at::kFloat, {r.n(), PPO_TOKEN_SAVED}, r.device(), what),
                 coef = like_forward(v[4], at::kFloat, r.shape(), r.device(), what);
    return {log_probs_backward(r, saved, floats(coef), nullptr, scale, Tensor(), 0.0), Tensor(),
            Tensor()};
  }
};

// logits, actions, ref, mask, beta, label_smoothing, margin, average, temperature
// -> (loss, (chosen, rejected))
PyObject* preference_loss(PyObject* const* a) {
  Preference p;
  p.r = Rows(a[0], a[1], a[3], a[8]);
  need(p.r.logits.dim() == 3 && p.r.logits.size(0) % 2 == 0);
  if (a[2] != Py_None) p.ref = p.r.row_constants(a[2]);
  p.beta = finite(a[4]);
  p.smoothing = number(a[5]);
  need(p.smoothing >= 0.0 && p.smoothing <= 1.0);
  p.margin = finite(a[6]);
  need(PyBool_Check(a[7]));
  p.average = a[7] == Py_True;
  Tensor loss, rewards;
  if (p.r.differentiable()) {
    unlocked([&] { return loss = PreferenceNode::apply(p.r.logits, &p, &rewards), 0; });
  } else {
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor coef;
    const int code = unlocked([&] { return preference(p, loss, rewards, coef, nullptr); });
    check("ppo_token_preference", code, p.r.device(), current_stream(p.r.device()));
  }
  at::AutoDispatchBelowADInplaceOrView below;
  const int64_t P = p.r.sequences() / 2;
  return pair(loss, tuple_of({rewards.narrow(0, 0, P), rewards.narrow(0, P, P)}));
}

struct Distill {
  Rows r;
  Tensor teacher, ids;
  ppo_token_loss l = {};
  int64_t K() const { return ids.size(-1); }
};

int distill(const Distill& p, Tensor& loss, Tensor* saved, Tensor* d) {
  const c10::DeviceGuard guard(p.r.device());
  loss = at::empty({}, p.r.f32());
  if (saved) {
    *saved = p.r.saved();
    *d = at::empty_like(p.r.logits);
  }
  const Tensor ws = p.r.scratch();
  const ppo_token_rows c = p.r.c();
  return ppo_token_distillation(&c, p.teacher.const_data_ptr(),
                                dtype_code(p.teacher.scalar_type()), p.ids.const_data_ptr(),
                                p.ids.scalar_type() == at::kLong, p.K(), &p.l,
                                loss.data_ptr<float>(), saved ? saved->data_ptr<float>() : nullptr,
                                saved ? d->data_ptr() : nullptr, ptr(ws), ws.numel(),
                                current_stream(p.r.device()));
}

struct DistillNode : public torch::autograd::Function<DistillNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor&, const Distill* p) {
    Tensor loss, saved, d;
    check_in_node("ppo_token_distillation", distill(*p, loss, &saved, &d), p->r.device(),
                  current_stream(p->r.device()));
    save_rows(ctx, p->r, {saved, p->teacher, p->ids});
    ctx->saved_data["K"] = p->K();
    hold(ctx, d, p->l.grad_scale);
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    constexpr const char* what = "distillation_loss";
    const variable_list v = ctx->get_saved_variables();
    const Rows r = saved_rows(ctx, v, what);
    if (!g[0].defined()) return variable_list(2);
    const at::Device dev = r.device();
    const Tensor scale = incoming(g[0], {}, dev, what);
    const Tensor saved = like_forward(v[3], at::kFloat, {r.n(), PPO_TOKEN_SAVED}, dev, what);
    std::vector<int64_t> shape = r.shape().vec();
    const int64_t K = ctx->saved_data["K"].toInt();
    shape.push_back(K);
    TORCH_CHECK(dtype_code(v[4].scalar_type()) >= 0 &&
                    (v[5].scalar_type() == at::kInt || v[5].scalar_type() == at::kLong),
                what, ": the saved teacher came back as ", v[4].scalar_type(), " and ",
                v[5].scalar_type());
    const Tensor teacher = like_forward(v[4], v[4].scalar_type(), shape, dev, what),
                 ids = like_forward(v[5], v[5].scalar_type(), shape, dev, what);
    const Tensor held = take_held(ctx, dev);
    const c10::DeviceGuard guard(dev);
    const Tensor d = held.defined() ? held : at::empty_like(r.logits);
    const ppo_token_rows c = r.c();
    const int code = ppo_token_distillation_backward(
        &c, teacher.const_data_ptr(), dtype_code(teacher.scalar_type()), ids.const_data_ptr(),
        ids.scalar_type() == at::kLong, K, floats(saved), floats(scale),
        held.defined() ? ctx->saved_data["value"].toDouble() : 0.0, d.data_ptr(),
        current_stream(dev));
    check_in_node("ppo_token_distillation_backward", code, dev, current_stream(dev));
    return {d, Tensor()};
  }
};

// logits, teacher, ids, mask, temperature, reduction, denominator, grad_scale
PyObject* distillation_loss(PyObject* const* a) {
  Distill p;
  p.r = Rows(a[0], nullptr, a[3], a[4]);
  const at::ScalarType tt = type_of(a[1]), it = type_of(a[2]);
  need(dtype_code(tt) >= 0 && (it == at::kInt || it == at::kLong));
  p.teacher = constant(plain(a[1], tt, p.r.device()));
  p.ids = plain(a[2], it, p.r.device());
  const int64_t dim = p.r.logits.dim();
  need(p.teacher.dim() == dim && p.teacher.sizes() == p.ids.sizes() && p.teacher.size(-1) > 0 &&
       p.teacher.sizes().slice(0, dim - 1) == p.r.shape());
  weights_of(a + 5, p.l);
  Tensor loss;
  if (p.r.differentiable()) {
    unlocked([&] { return loss = DistillNode::apply(p.r.logits, &p), 0; });
    return wrap(loss);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  const int code = unlocked([&] { return distill(p, loss, nullptr, nullptr); });
  check("ppo_token_distillation", code, p.r.device(), current_stream(p.r.device()));
  return wrap(loss);
}

// --- top logits ----------------------------------------------------------------------------

PyObject* top_logits(PyObject* const* a) {  // logits, k
  const at::ScalarType type = type_of(a[0]);
  need(dtype_code(type) >= 0);
  const Tensor& x = plain(a[0], type);
  need(x.dim() >= 1 && x.numel() > 0 && PyLong_CheckExact(a[1]));
  const int64_t A = x.size(-1), n = x.numel() / A, k = integer(a[1]);
  need(k >= 1 && k <= A && k <= PPO_TOKEN_MAX_K);
  const at::Device dev = x.device();
  void* stream = current_stream(dev);
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor values, ids;
  const int code = unlocked([&] {
    const c10::DeviceGuard guard(dev);
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = k;
    values = at::empty(shape, x.options());
    ids = at::empty(shape, x.options().dtype(at::kLong));
    const int dtype = dtype_code(type);
    const size_t nbytes = ppo_token_top_workspace_bytes(n, A, k, dtype);
    const Tensor ws = bytes(nbytes, dev);
    return ppo_token_top(x.const_data_ptr(), dtype, n, A, k, values.data_ptr(),
                         ids.data_ptr<int64_t>(), ptr(ws), nbytes, stream);
  });
  check("ppo_token_top", code, dev, stream);
  return tuple_of({values, ids});
}

}  // namespace

PyMethodDef kTokenMethods[] = {{"capture_id", capture_id, METH_O, nullptr},
                               PPO_ENTRY("token_log_probs", token_log_probs, 5),
                               PPO_ENTRY("token_policy_loss", token_policy_loss, 14),
                               PPO_ENTRY("preference_loss", preference_loss, 9),
                               PPO_ENTRY("distillation_loss", distillation_loss, 8),
                               PPO_ENTRY("top_logits", top_logits, 2),
                               {nullptr, nullptr, 0, nullptr}};

}  // namespace ppo_native
