// The layer operators' host path in ppo_amd._native: layers.py's functions for
// the ordinary call (plain contiguous tensors of one type on one GPU), and the
// autograd nodes of the two that have a gradient, so that neither direction
// runs in the interpreter.  Any other call returns None and takes layers.py's
// checks.
//
// Measured on MI355X, us a call among others, through Python and here: dropout
// of 128 x 128 with its gradient 48 and 28 (of which torch's engine takes 18), the
// gated block of 256 x 128 -> 256 with its gradients 86 and 54, int8_linear of one
// row 14 and 7 (another host takes up to twice that in every figure).
#include "native.hpp"

#include <c10/core/DeviceGuard.h>

#include "ppo_layers.h"

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

// A plain tensor of one of the three types, with at least one dimension.
const Tensor& plain_layer(PyObject* o) {
  const at::ScalarType type = type_of(o);
  need(dtype_code(type) >= 0);
  const Tensor& t = plain(o, type);
  need(t.dim() >= 1);
  return t;
}

Tensor scratch(size_t nbytes, const at::Device& device) {
  if (!nbytes) return {};
  return at::empty({(int64_t)nbytes}, at::TensorOptions().dtype(at::kByte).device(device));
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// PPO_LAYER_ALIGNED where the operands start at multiples of 16 bytes: no room
// for aligned copies of them is needed then.
int aligned_flag(std::initializer_list<const Tensor*> operands) {
  for (const Tensor* t : operands)
    if ((uintptr_t)t->const_data_ptr() & 15) return 0;
  return PPO_LAYER_ALIGNED;
}

std::vector<int64_t> with_last(const Tensor& x, int64_t last) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = last;
  return s;
}

// dropout's arguments p, seed, rows from a[0], for M rows on `device`.
struct Drop {
  double p = 0.0;
  uint64_t seed = 0;
  Tensor seed_at, rows;

  Drop() = default;
  Drop(PyObject* const* a, const at::Device& device, int64_t M) {
    p = number(a[0]);
    need(p >= 0.0 && p <= 1.0);
    if (PyLong_CheckExact(a[1])) {
      seed = PyLong_AsUnsignedLongLongMask(a[1]);
      need(!PyErr_Occurred());
    } else {
      seed_at = plain(a[1], at::kLong, device);
      need(seed_at.numel() == 1);
    }
    if (a[2] != Py_None) {
      rows = plain(a[2], at::kLong, device);
      need(rows.dim() == 1 && rows.size(0) == M);
    }
  }
  ppo_dropout c() const {
    return {p, seed, static_cast<const uint64_t*>(ptr(seed_at)),
            static_cast<const int64_t*>(ptr(rows))};
  }
};

bool needs_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

void need_no_tangent(const Tensor& t) { need(!t.defined() || !t._fw_grad(0).defined()); }

// What a backward pass got back or was handed: as the forward had it, or a
// clear error (a saved-tensor hook may return anything).
Tensor like_forward(const Tensor& t, at::ScalarType type, const at::Device& device) {
  TORCH_CHECK(t.device() == device && t.scalar_type() == type && t.layout() == at::kStrided &&
                  !t.key_set().has_any(kWrapped),
              "a layer's backward pass needs ", type, " tensors of their own on ", device);
  return t.contiguous();
}

// dropout's arguments as a node saved them, for M rows.
Drop saved_drop(AutogradContext* ctx, const Tensor& seed_at, const Tensor& rows,
                const at::Device& device, int64_t M) {
  Drop d;
  d.p = ctx->saved_data["p"].toDouble();
  d.seed = (uint64_t)ctx->saved_data["seed"].toInt();
  if (seed_at.defined()) d.seed_at = like_forward(seed_at, at::kLong, device);
  if (rows.defined()) d.rows = like_forward(rows, at::kLong, device);
  TORCH_CHECK(!seed_at.defined() || d.seed_at.numel() == 1,
              "dropout's saved seed has changed its shape");
  TORCH_CHECK(!rows.defined() || (d.rows.dim() == 1 && d.rows.numel() == M),
              "dropout's saved rows have changed their shape");
  return d;
}

// --- dropout ---------------------------------------------------------------------------

int dropout_into(const Tensor& x, const Tensor& y, const Drop& d) {
  if (x.numel() == 0) return PPO_OK;
  const c10::DeviceGuard guard(x.device());
  const ppo_dropout c = d.c();
  return ppo_layer_dropout(x.const_data_ptr(), y.data_ptr(), dtype_code(x.scalar_type()),
                           x.numel() / x.size(-1), x.size(-1), &c, current_stream(x.device()));
}

struct DropoutNode : public torch::autograd::Function<DropoutNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Drop* d) {
    ctx->save_for_backward({d->seed_at, d->rows});
    ctx->saved_data["p"] = d->p;
    ctx->saved_data["seed"] = (int64_t)d->seed;
    const Tensor y = at::empty_like(x);
    check_in_node("ppo_layer_dropout", dropout_into(x, y, *d), x.device(),
                  current_stream(x.device()));
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list saved = ctx->get_saved_variables();
    if (!g[0].defined()) return {Tensor(), Tensor()};
    TORCH_CHECK(dtype_code(g[0].scalar_type()) >= 0, "dropout's gradient is ", g[0].scalar_type());
    const Tensor dy = like_forward(g[0], g[0].scalar_type(), g[0].device());
    const Drop d = saved_drop(ctx, saved[0], saved[1], dy.device(), dy.numel() / dy.size(-1));
    // linear in x: its derivative is the same mask (create_graph comes again)
    return {apply(dy, &d), Tensor()};
  }
};

PyObject* dropout(PyObject* const* a) {  // x, p, seed, rows
  const Tensor& x = plain_layer(a[0]);
  need(x.numel() > 0);
  const Drop d(a + 1, x.device(), x.numel() / x.size(-1));
  if (needs_grad({&x})) {
    need_no_tangent(x);
    Tensor y;
    unlocked([&] { return y = DropoutNode::apply(x, &d), 0; });
    return wrap(y);
  }
  need_no_tangent(x);
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor y;
  const int code = unlocked([&] {
    y = at::empty_like(x);
    return dropout_into(x, y, d);
  });
  check("ppo_layer_dropout", code, x.device(), current_stream(x.device()));
  return wrap(y);
}

// --- gated feed-forward block ------------------------------------------------------------

struct Gated {
  Tensor x, wg, wu, bg, bu;
  int act;
  Drop drop;
  int64_t M, D, F;
  at::Device device() const { return x.device(); }
};

int gated_forward(const Gated& l, Tensor& h, Tensor* saved) {
  const c10::DeviceGuard guard(l.device());
  const int dtype = dtype_code(l.x.scalar_type()) | aligned_flag({&l.x, &l.wg, &l.wu});
  h = at::empty(with_last(l.x, l.F), l.x.options());
  if (saved) *saved = at::empty({2, l.M, (l.F + 3) / 4 * 4}, l.x.options().dtype(at::kFloat));
  const size_t nbytes = ppo_layer_gated_workspace_bytes(dtype, l.M, l.D, l.F);
  const Tensor ws = scratch(nbytes, l.device());
  const ppo_dropout c = l.drop.c();
  return ppo_layer_gated_forward(l.x.const_data_ptr(), l.wg.const_data_ptr(),
                                 l.wu.const_data_ptr(), ptr(l.bg), ptr(l.bu), dtype, l.M, l.D, l.F,
                                 l.act, &c, h.data_ptr(),
                                 saved ? saved->data_ptr<float>() : nullptr, ptr(ws), nbytes,
                                 current_stream(l.device()));
}

struct GatedNode : public torch::autograd::Function<GatedNode> {
  static Tensor forward(AutogradContext* ctx, at::TensorList, const Gated* l) {
    Tensor h, saved;
    check_in_node("ppo_layer_gated_forward", gated_forward(*l, h, &saved), l->device(),
                  current_stream(l->device()));
    ctx->save_for_backward({l->x, l->wg, l->wu, saved, l->drop.seed_at, l->drop.rows});
    ctx->saved_data["act"] = (int64_t)l->act;
    ctx->saved_data["p"] = l->drop.p;
    ctx->saved_data["seed"] = (int64_t)l->drop.seed;
    ctx->saved_data["bias"] = l->bg.defined();
    return h;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "gated_ffn can be differentiated once: its backward pass has no create_graph");
    const variable_list saved = ctx->get_saved_variables();
    const bool bias = ctx->saved_data["bias"].toBool();
    const int n = bias ? 5 : 3;
    variable_list out(n + 1);
    if (!g[0].defined()) return out;
    const at::Device dev = g[0].device();
    const at::ScalarType type = g[0].scalar_type();
    TORCH_CHECK(dtype_code(type) >= 0, "gated_ffn's gradient is ", type);
    const Tensor dh = like_forward(g[0], type, dev), x = like_forward(saved[0], type, dev),
                 wg = like_forward(saved[1], type, dev), wu = like_forward(saved[2], type, dev),
                 gu = like_forward(saved[3], at::kFloat, dev);
    TORCH_CHECK(x.dim() >= 1 && x.numel() > 0 && wg.dim() == 2 && wg.size(0) > 0 &&
                    wg.size(1) == x.size(-1) && wu.sizes() == wg.sizes(),
                "gated_ffn's saved tensors have changed their shapes");
    const int64_t D = x.size(-1), F = wg.size(0), M = x.numel() / D;
    TORCH_CHECK(dh.numel() == M * F && gu.numel() == 2 * M * ((F + 3) / 4 * 4),
                "gated_ffn's saved tensors have changed their shapes");
    const Drop d = saved_drop(ctx, saved[4], saved[5], dev, M);
    const c10::DeviceGuard guard(dev);
    if (ctx->needs_input_grad(0)) out[0] = at::empty_like(x);
    if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2)) {
      out[1] = at::empty({F, D}, x.options());
      out[2] = at::empty({F, D}, x.options());
    }
    if (bias && (ctx->needs_input_grad(3) || ctx->needs_input_grad(4))) {
      out[3] = at::empty({F}, x.options());
      out[4] = at::empty({F}, x.options());
    }
    const int dtype = dtype_code(type) | aligned_flag({&x, &wg, &wu});
    const size_t nbytes = ppo_layer_gated_backward_workspace_bytes(dtype, M, D, F);
    const Tensor ws = scratch(nbytes, dev);
    const ppo_dropout c = d.c();
    const int code = ppo_layer_gated_backward(
        dh.const_data_ptr(), x.const_data_ptr(), wg.const_data_ptr(), wu.const_data_ptr(),
        gu.const_data_ptr<float>(), dtype, M, D, F, (int)ctx->saved_data["act"].toInt(), &c,
        ptr(out[0]), ptr(out[1]), ptr(out[2]), bias ? ptr(out[3]) : nullptr,
        bias ? ptr(out[4]) : nullptr, ptr(ws), nbytes, current_stream(dev));
    check_in_node("ppo_layer_gated_backward", code, dev, current_stream(dev));
    for (int k = 0; k < n; ++k)
      if (!ctx->needs_input_grad(k)) out[k] = Tensor();
    return out;
  }
};

PyObject* gated_ffn(PyObject* const* a) {  // x, wg, wu, bg, bu, act, p, seed, rows
  Gated l;
  l.x = plain_layer(a[0]);
  const at::ScalarType type = l.x.scalar_type();
  const at::Device dev = l.x.device();
  need(l.x.numel() > 0);
  l.D = l.x.size(-1);
  l.M = l.x.numel() / l.D;
  l.wg = plain(a[1], type, dev);
  l.wu = plain(a[2], type, dev);
  need(l.wg.dim() == 2 && l.wg.size(1) == l.D && l.wg.size(0) > 0 && l.wu.sizes() == l.wg.sizes());
  l.F = l.wg.size(0);
  need((a[3] == Py_None) == (a[4] == Py_None));
  if (a[3] != Py_None) {
    l.bg = plain(a[3], type, dev);
    l.bu = plain(a[4], type, dev);
    need(l.bg.dim() == 1 && l.bg.size(0) == l.F && l.bu.sizes() == l.bg.sizes());
  }
  l.act = (int)integer(a[5]);
  l.drop = Drop(a + 6, dev, l.M);
  for (const Tensor* t : {&l.x, &l.wg, &l.wu, &l.bg, &l.bu}) need_no_tangent(*t);
  Tensor h;
  if (needs_grad({&l.x, &l.wg, &l.wu, &l.bg, &l.bu})) {
    variable_list leaves = {l.x, l.wg, l.wu};
    if (l.bg.defined()) leaves.insert(leaves.end(), {l.bg, l.bu});
    unlocked([&] { return h = GatedNode::apply(at::TensorList(leaves), &l), 0; });
    return wrap(h);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  const int code = unlocked([&] { return gated_forward(l, h, nullptr); });
  check("ppo_layer_gated_forward", code, dev, current_stream(dev));
  return wrap(h);
}

// --- 8 bits ------------------------------------------------------------------------------

PyObject* quantize_rows(PyObject* const* a) {  // x
  const Tensor& x = plain_layer(a[0]);
  need(x.numel() > 0);
  const at::Device dev = x.device();
  void* stream = current_stream(dev);
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor q, scale;
  const int code = unlocked([&] {
    const c10::DeviceGuard guard(dev);
    q = at::empty(x.sizes(), x.options().dtype(at::kChar));
    scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    return ppo_layer_quantize_rows(x.const_data_ptr(), dtype_code(x.scalar_type()),
                                   x.numel() / x.size(-1), x.size(-1), q.data_ptr<int8_t>(),
                                   scale.data_ptr<float>(), stream);
  });
  check("ppo_layer_quantize_rows", code, dev, stream);
  return tuple_of({q, scale});
}

PyObject* int8_linear(PyObject* const* a) {  // x, weight, weight_scale, bias, x_scale, out dtype
  const bool eight = type_of(a[0]) == at::kChar;
  const Tensor& x = eight ? plain(a[0], at::kChar) : plain_layer(a[0]);
  const at::Device dev = x.device();
  need(x.dim() >= 1 && x.numel() > 0);
  const int64_t K = x.size(-1), M = x.numel() / K;
  const Tensor& w = plain(a[1], at::kChar, dev);
  need(w.dim() == 2 && w.size(1) == K && w.size(0) > 0);
  const int64_t N = w.size(0);
  const Tensor& ws = plain_rows(a[2], dev, N);
  need(eight == (a[4] != Py_None));
  at::ScalarType type = x.scalar_type();
  if (a[5] != Py_None) {
    need(THPDtype_Check(a[5]));
    type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  }
  need(dtype_code(type) >= 0 && (eight || type == x.scalar_type()));
  Tensor bias, xs;
  if (a[3] != Py_None) {
    bias = plain(a[3], type, dev);
    need(bias.dim() == 1 && bias.size(0) == N);
  }
  if (eight) {
    xs = plain(a[4], at::kFloat, dev);
    need(xs.sizes() == x.sizes().slice(0, x.dim() - 1));
  }
  need(!needs_grad({&x, &ws, &bias, &xs}));
  for (const Tensor* t : std::initializer_list<const Tensor*>{&x, &ws, &bias, &xs})
    need_no_tangent(*t);
  void* stream = current_stream(dev);
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor out;
  const int code = unlocked([&] {
    const c10::DeviceGuard guard(dev);
    out = at::empty(with_last(x, N), x.options().dtype(type));
    const int flag = eight ? aligned_flag({&x, &w}) : aligned_flag({&w});
    const size_t nbytes = ppo_layer_int8_linear_workspace_bytes(M, N, K, (eight ? 0 : 1) | flag);
    const Tensor work = scratch(nbytes, dev);
    return ppo_layer_int8_linear(eight ? nullptr : x.const_data_ptr(),
                                 eight ? x.const_data_ptr<int8_t>() : nullptr,
                                 static_cast<const float*>(ptr(xs)), w.const_data_ptr<int8_t>(),
                                 in(ws), ptr(bias), dtype_code(type) | flag, M, N, K, out.data_ptr(),
                                 ptr(work), nbytes, stream);
  });
  check("ppo_layer_int8_linear", code, dev, stream);
  return wrap(out);
}

}  // namespace

PyMethodDef kLayerMethods[] = {PPO_ENTRY("layer_dropout", dropout, 4),
                               PPO_ENTRY("layer_gated_ffn", gated_ffn, 9),
                               PPO_ENTRY("layer_quantize_rows", quantize_rows, 1),
                               PPO_ENTRY("layer_int8_linear", int8_linear, 6),
                               {nullptr, nullptr, 0, nullptr}};

}  // namespace ppo_native
