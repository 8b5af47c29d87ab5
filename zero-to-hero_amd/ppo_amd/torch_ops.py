"""The hot path as registered torch operators: torch.ops.ppo_amd.*.

Each operator runs the same HIP kernels as the functions in ops.py (it calls
them), but through torch's dispatcher, so it is visible to torch.compile
(with the fake implementations below, a compiled function traces through it
without a graph break), to torch.library.opcheck and to the profiler's op
view.  The implementations are registered for CUDA (HIP) tensors only: a CPU
tensor raises NotImplementedError, as there is no CPU fallback.

  ppo_amd::gae(rewards, values, dones, last_value?, gamma, lam) -> (adv, ret)
      PPOAgent._advantages + returns (rl/deep/agents/ppo.py:123-124, 173-193)
  ppo_amd::gae_normalize(rewards, values, dones, last_value?, gamma, lam, eps)
      -> (adv, ret, adv_n, stats[2])        ... plus ppo.py:126-127, fused
  ppo_amd::normalize_advantages(adv, eps) -> adv_n      (ppo.py:126-127)
  ppo_amd::ppo_loss_discrete(logits, actions, old_log_probs, advantages,
      returns, values, old_values?, clip_ratio, vf_clip?, value_coef,
      entropy_coef) -> (scalars[6], dlogits, dvalues)   (ppo.py:150-169)
  ppo_amd::ppo_loss_gaussian(mu, log_std, actions, old_log_probs, advantages,
      returns, values, old_values?, clip_ratio, vf_clip?, value_coef,
      entropy_coef) -> (scalars[6], dmu, dlog_std, dvalues)

  ppo_amd::dropout(x, p, seed, seed_at?, rows?) -> y
  ppo_amd::gated_ffn(x, w_gate, w_up, b_gate?, b_up?, activation, dropout_p,
      seed, seed_at?, rows?) -> (h, saved), saved what the backward pass reads
  ppo_amd::gated_ffn_backward(dh, x, w_gate, w_up, saved, bias, activation,
      dropout_p, seed, seed_at?, rows?) -> (dx, dw_gate, dw_up, db_gate, db_up)
  ppo_amd::quantize_rows(x) -> (q, scale)
  ppo_amd::int8_linear(x, weight, weight_scale, bias?, x_scale?, out_dtype?) -> y
      the layers of layers.py; a seed that changes from call to call goes
      into `seed_at` (int64 [1] on the device), which `seed` stands back for

  ppo_amd::token_log_probs(logits, actions, mask?, temperature)
      -> (log_probs, entropy, saved), saved what the backward pass reads
  ppo_amd::token_policy_loss(logits, actions, old_log_probs, advantages,
      ref_log_probs?, mask?, clip_low, clip_high, kl_coef, entropy_coef,
      temperature, reduction, denominator?) -> (scalars[6], saved, coef)
  ppo_amd::preference_loss(logits, actions, ref_log_probs?, mask?, beta,
      label_smoothing, margin, average, temperature)
      -> (loss, rewards, saved, coef)
  ppo_amd::token_log_probs_backward(logits, actions, mask?, temperature, saved,
      d_log_probs, d_entropy?, scale?) -> dlogits
      the backward pass of these three: a loss's coef is its gradient in the
      log-probabilities (and entropies), scale its incoming gradient
  ppo_amd::distillation_loss(logits, teacher_logits, teacher_ids, mask?,
      temperature, reduction, denominator?) -> (loss, saved), and
  ppo_amd::distillation_loss_backward(logits, teacher_logits, teacher_ids,
      mask?, temperature, saved, scale) -> dlogits
  ppo_amd::top_logits(logits, k) -> (values, ids)
      the token policies of tokens.py; the losses form their gradient in the
      backward pass here, from the logits

The loss operators are differentiable in their first output: backward of
scalars[0] (the total loss; the other scalars are reported values) scales the
fused kernel's gradients by the incoming gradient, as ops.ppo_loss_discrete
does.  Their gradient outputs are marked non-differentiable.
"""

from typing import Optional

import torch
from torch import Tensor

from . import _lib, layers, ops, tokens

_NS = "ppo_amd"


def _scalars_like(t: Tensor) -> Tensor:
    return torch.empty(_lib.PPO_NUM_SCALARS, dtype=torch.float32, device=t.device)


# ---------------------------------------------------------------------------
# GAE and normalisation
# ---------------------------------------------------------------------------
@torch.library.custom_op(f"{_NS}::gae", mutates_args=(), device_types="cuda")
def gae(rewards: Tensor, values: Tensor, dones: Tensor, last_value: Optional[Tensor],
        gamma: float, lam: float) -> tuple[Tensor, Tensor]:
    adv, ret = ops.gae(rewards, values, dones, last_value, gamma, lam)
    return adv, ret


@gae.register_fake
def _gae_fake(rewards, values, dones, last_value, gamma, lam):
    return torch.empty_like(rewards), torch.empty_like(rewards)


@torch.library.custom_op(f"{_NS}::gae_normalize", mutates_args=(), device_types="cuda")
def gae_normalize(rewards: Tensor, values: Tensor, dones: Tensor, last_value: Optional[Tensor],
                  gamma: float, lam: float, eps: float) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    adv, ret, adv_n, stats = ops.gae_normalize(rewards, values, dones, last_value, gamma, lam,
                                               eps, return_stats=True)
    return adv, ret, adv_n, stats


@gae_normalize.register_fake
def _gae_normalize_fake(rewards, values, dones, last_value, gamma, lam, eps):
    return (torch.empty_like(rewards), torch.empty_like(rewards), torch.empty_like(rewards),
            torch.empty(2, dtype=torch.float32, device=rewards.device))


@torch.library.custom_op(f"{_NS}::normalize_advantages", mutates_args=(), device_types="cuda")
def normalize_advantages(advantages: Tensor, eps: float) -> Tensor:
    return ops.normalize_advantages(advantages, eps)


@normalize_advantages.register_fake
def _normalize_advantages_fake(advantages, eps):
    return torch.empty_like(advantages)


# ---------------------------------------------------------------------------
# Fused PPO losses (forward + backward in one launch)
# ---------------------------------------------------------------------------
@torch.library.custom_op(f"{_NS}::ppo_loss_discrete", mutates_args=(), device_types="cuda")
def ppo_loss_discrete(logits: Tensor, actions: Tensor, old_log_probs: Tensor, advantages: Tensor,
                      returns: Tensor, values: Tensor, old_values: Optional[Tensor],
                      clip_ratio: float, vf_clip: Optional[float], value_coef: float,
                      entropy_coef: float) -> tuple[Tensor, Tensor, Tensor]:
    return ops.ppo_loss_discrete_fused(logits, actions, old_log_probs, advantages, returns,
                                       values, old_values, clip_ratio, vf_clip, value_coef,
                                       entropy_coef)


@ppo_loss_discrete.register_fake
def _ppo_loss_discrete_fake(logits, actions, old_log_probs, advantages, returns, values,
                            old_values, clip_ratio, vf_clip, value_coef, entropy_coef):
    return _scalars_like(logits), torch.empty_like(logits), torch.empty_like(values)


def _discrete_setup(ctx, inputs, output):
    _, dlogits, dvalues = output
    ctx.mark_non_differentiable(dlogits, dvalues)
    ctx.save_for_backward(dlogits, dvalues)


def _discrete_backward(ctx, grad_scalars, grad_dlogits, grad_dvalues):
    dlogits, dvalues = ctx.saved_tensors
    g = grad_scalars[0]
    return dlogits * g, None, None, None, None, dvalues * g, None, None, None, None, None


ppo_loss_discrete.register_autograd(_discrete_backward, setup_context=_discrete_setup)


@torch.library.custom_op(f"{_NS}::ppo_loss_gaussian", mutates_args=(), device_types="cuda")
def ppo_loss_gaussian(mu: Tensor, log_std: Tensor, actions: Tensor, old_log_probs: Tensor,
                      advantages: Tensor, returns: Tensor, values: Tensor,
                      old_values: Optional[Tensor], clip_ratio: float, vf_clip: Optional[float],
                      value_coef: float, entropy_coef: float
                      ) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    return ops.ppo_loss_gaussian_fused(mu, log_std, actions, old_log_probs, advantages, returns,
                                       values, old_values, clip_ratio, vf_clip, value_coef,
                                       entropy_coef)


@ppo_loss_gaussian.register_fake
def _ppo_loss_gaussian_fake(mu, log_std, actions, old_log_probs, advantages, returns, values,
                            old_values, clip_ratio, vf_clip, value_coef, entropy_coef):
    return (_scalars_like(mu), torch.empty_like(mu), torch.empty_like(log_std),
            torch.empty_like(values))


def _gaussian_setup(ctx, inputs, output):
    _, dmu, dlog_std, dvalues = output
    ctx.mark_non_differentiable(dmu, dlog_std, dvalues)
    ctx.save_for_backward(dmu, dlog_std, dvalues)


def _gaussian_backward(ctx, grad_scalars, grad_dmu, grad_dlog_std, grad_dvalues):
    dmu, dlog_std, dvalues = ctx.saved_tensors
    g = grad_scalars[0]
    return (dmu * g, dlog_std * g, None, None, None, None, dvalues * g, None, None, None, None,
            None)


ppo_loss_gaussian.register_autograd(_gaussian_backward, setup_context=_gaussian_setup)


# ---------------------------------------------------------------------------
# Feed-forward layers
# ---------------------------------------------------------------------------
def _seed(seed: int, seed_at: Optional[Tensor]):
    return seed if seed_at is None else seed_at


@torch.library.custom_op(f"{_NS}::dropout", mutates_args=(), device_types="cuda")
def dropout(x: Tensor, p: float, seed: int, seed_at: Optional[Tensor],
            rows: Optional[Tensor]) -> Tensor:
    return layers.dropout(x, p, _seed(seed, seed_at), rows)


@dropout.register_fake
def _dropout_fake(x, p, seed, seed_at, rows):
    return torch.empty_like(x)


def _dropout_setup(ctx, inputs, output):
    _, ctx.p, ctx.seed, seed_at, rows = inputs
    ctx.save_for_backward(seed_at, rows)


def _dropout_backward(ctx, dy):
    seed_at, rows = ctx.saved_tensors
    return dropout(dy.contiguous(), ctx.p, ctx.seed, seed_at, rows), None, None, None, None


dropout.register_autograd(_dropout_backward, setup_context=_dropout_setup)


@torch.library.custom_op(f"{_NS}::gated_ffn", mutates_args=(), device_types="cuda")
def gated_ffn(x: Tensor, w_gate: Tensor, w_up: Tensor, b_gate: Optional[Tensor],
              b_up: Optional[Tensor], activation: str, dropout_p: float, seed: int,
              seed_at: Optional[Tensor], rows: Optional[Tensor]) -> tuple[Tensor, Tensor]:
    s = _seed(seed, seed_at)
    act = layers._check_gated(x, w_gate, w_up, b_gate, b_up, activation, dropout_p, s, rows)
    return layers._gated_forward(x, w_gate, w_up, b_gate, b_up, act, dropout_p, s, rows, True)


@gated_ffn.register_fake
def _gated_ffn_fake(x, w_gate, w_up, b_gate, b_up, activation, dropout_p, seed, seed_at, rows):
    F = w_gate.shape[0]
    M = 1
    for n in x.shape[:-1]:
        M = M * n
    return (x.new_empty((*x.shape[:-1], F)),
            x.new_empty((2, M, (F + 3) // 4 * 4), dtype=torch.float32))


@torch.library.custom_op(f"{_NS}::gated_ffn_backward", mutates_args=(), device_types="cuda")
def gated_ffn_backward(dh: Tensor, x: Tensor, w_gate: Tensor, w_up: Tensor, saved: Tensor,
                       bias: bool, activation: str, dropout_p: float, seed: int,
                       seed_at: Optional[Tensor], rows: Optional[Tensor]
                       ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    act, s = layers._check_activation(activation), _seed(seed, seed_at)
    layers._check_gated_backward(dh, x, w_gate, w_up, saved, dropout_p, s, rows)
    need = (True, True, True, bias, bias)
    dx, dwg, dwu, dbg, dbu = layers._gated_backward(dh, x, w_gate, w_up, saved, act, dropout_p, s,
                                                    rows, need)
    return (dx, dwg, dwu, x.new_empty(0) if dbg is None else dbg,
            x.new_empty(0) if dbu is None else dbu)


@gated_ffn_backward.register_fake
def _gated_ffn_backward_fake(dh, x, w_gate, w_up, saved, bias, activation, dropout_p, seed,
                             seed_at, rows):
    F = w_gate.shape[0] if bias else 0
    return (torch.empty_like(x), torch.empty_like(w_gate), torch.empty_like(w_up),
            x.new_empty(F), x.new_empty(F))


def _gated_setup(ctx, inputs, output):
    x, w_gate, w_up, b_gate, _, ctx.activation, ctx.p, ctx.seed, seed_at, rows = inputs
    ctx.bias = b_gate is not None
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(x, w_gate, w_up, output[1], seed_at, rows)


def _gated_backward(ctx, dh, _):
    x, w_gate, w_up, saved, seed_at, rows = ctx.saved_tensors
    dx, dwg, dwu, dbg, dbu = gated_ffn_backward(dh.contiguous(), x, w_gate, w_up, saved, ctx.bias,
                                                ctx.activation, ctx.p, ctx.seed, seed_at, rows)
    return (dx, dwg, dwu, dbg if ctx.bias else None, dbu if ctx.bias else None, None, None, None,
            None, None)


gated_ffn.register_autograd(_gated_backward, setup_context=_gated_setup)


@torch.library.custom_op(f"{_NS}::quantize_rows", mutates_args=(), device_types="cuda")
def quantize_rows(x: Tensor) -> tuple[Tensor, Tensor]:
    return layers.quantize_rows(x)


@quantize_rows.register_fake
def _quantize_rows_fake(x):
    return (x.new_empty(x.shape, dtype=torch.int8),
            x.new_empty(x.shape[:-1], dtype=torch.float32))


@torch.library.custom_op(f"{_NS}::int8_linear", mutates_args=(), device_types="cuda")
def int8_linear(x: Tensor, weight: Tensor, weight_scale: Tensor, bias: Optional[Tensor],
                x_scale: Optional[Tensor], out_dtype: Optional[torch.dtype]) -> Tensor:
    return layers.int8_linear(x, weight, weight_scale, bias, x_scale, out_dtype)


@int8_linear.register_fake
def _int8_linear_fake(x, weight, weight_scale, bias, x_scale, out_dtype):
    return x.new_empty((*x.shape[:-1], weight.shape[0]),
                       dtype=x.dtype if out_dtype is None else out_dtype)


# ---------------------------------------------------------------------------
# Token policies
# ---------------------------------------------------------------------------
def _row_floats(logits: Tensor) -> Tensor:
    return logits.new_empty(logits.shape[:-1], dtype=torch.float32)


def _row_count(logits: Tensor):
    n = 1
    for k in logits.shape[:-1]:
        n = n * k
    return n


def _saved_like(logits: Tensor) -> Tensor:
    return logits.new_empty((_row_count(logits), _lib.PPO_TOKEN_SAVED), dtype=torch.float32)


def _check_saved(logits: Tensor, saved: Tensor) -> None:
    tokens._require(saved, "saved", (torch.float32,), logits.device)
    if saved.shape != (_row_count(logits), _lib.PPO_TOKEN_SAVED):
        raise ValueError(f"saved must be {(_row_count(logits), _lib.PPO_TOKEN_SAVED)}, got "
                         f"{tuple(saved.shape)}")


def _check_scalar(logits: Tensor, scale: Optional[Tensor]) -> None:
    if scale is not None:
        tokens._require(scale, "scale", (torch.float32,), logits.device)
        if scale.numel() != 1:
            raise ValueError(f"scale must hold one value, got {scale.numel()}")


def _refuse_gradients(ctx, what: str, inputs: dict) -> None:
    """Inputs (index: name) that ask for a gradient which the operator does not form."""
    for index, name in inputs.items():
        if ctx.needs_input_grad[index]:
            raise RuntimeError(f"{what} has no gradient in {name}: detach it")


@torch.library.custom_op(f"{_NS}::token_log_probs", mutates_args=(), device_types="cuda")
def token_log_probs(logits: Tensor, actions: Tensor, mask: Optional[Tensor], temperature: float
                    ) -> tuple[Tensor, Tensor, Tensor]:
    tokens._check_logits(logits, temperature)
    tokens._check_actions(logits, actions, mask)
    return tokens._log_probs(logits, actions, mask, temperature, None, True, True)


@token_log_probs.register_fake
def _token_log_probs_fake(logits, actions, mask, temperature):
    return _row_floats(logits), _row_floats(logits), _saved_like(logits)


@torch.library.custom_op(f"{_NS}::token_log_probs_backward", mutates_args=(), device_types="cuda")
def token_log_probs_backward(logits: Tensor, actions: Tensor, mask: Optional[Tensor],
                             temperature: float, saved: Tensor, d_log_probs: Tensor,
                             d_entropy: Optional[Tensor], scale: Optional[Tensor]) -> Tensor:
    tokens._check_logits(logits, temperature)
    tokens._check_actions(logits, actions, mask)
    _check_saved(logits, saved)
    _check_scalar(logits, scale)
    tokens._check_rows(logits, d_log_probs, "d_log_probs", (torch.float32,))
    if d_entropy is not None:
        tokens._check_rows(logits, d_entropy, "d_entropy", (torch.float32,))
    return tokens._log_probs_backward(logits, actions, mask, temperature, saved, d_log_probs,
                                      d_entropy, scale)


@token_log_probs_backward.register_fake
def _token_log_probs_backward_fake(logits, actions, mask, temperature, saved, d_log_probs,
                                   d_entropy, scale):
    return torch.empty_like(logits)


def _token_log_probs_setup(ctx, inputs, output):
    logits, actions, mask, ctx.temperature = inputs
    ctx.mark_non_differentiable(output[2])
    ctx.save_for_backward(logits, actions, mask, output[2])


def _token_log_probs_grad(ctx, dlp, dH, _):
    logits, actions, mask, saved = ctx.saved_tensors
    d = token_log_probs_backward(logits, actions, mask, ctx.temperature, saved, dlp.contiguous(),
                                 dH.contiguous(), None)
    return d, None, None, None


token_log_probs.register_autograd(_token_log_probs_grad, setup_context=_token_log_probs_setup)


@torch.library.custom_op(f"{_NS}::token_policy_loss", mutates_args=(), device_types="cuda")
def token_policy_loss(logits: Tensor, actions: Tensor, old_log_probs: Tensor, advantages: Tensor,
                      ref_log_probs: Optional[Tensor], mask: Optional[Tensor], clip_low: float,
                      clip_high: float, kl_coef: float, entropy_coef: float, temperature: float,
                      reduction: str, denominator: Optional[float]
                      ) -> tuple[Tensor, Tensor, Tensor]:
    per_sequence = tokens._check_policy(logits, actions, old_log_probs, advantages, ref_log_probs,
                                        mask, clip_low, clip_high, kl_coef, entropy_coef,
                                        temperature)
    tokens._check_weights(reduction, denominator, 1.0)
    loss = tokens._loss(reduction, denominator, 1.0, clip_low, clip_high, kl_coef, entropy_coef,
                        per_sequence)
    scalars, saved, coef, _ = tokens._policy(logits, actions, old_log_probs, advantages,
                                             ref_log_probs, mask, temperature, loss, True, False)
    return scalars, saved, coef.view(2, *logits.shape[:-1])


@token_policy_loss.register_fake
def _token_policy_loss_fake(logits, actions, old_log_probs, advantages, ref_log_probs, mask,
                            clip_low, clip_high, kl_coef, entropy_coef, temperature, reduction,
                            denominator):
    return (logits.new_empty(_lib.PPO_TOKEN_SCALARS, dtype=torch.float32), _saved_like(logits),
            logits.new_empty((2, *logits.shape[:-1]), dtype=torch.float32))


def _token_policy_setup(ctx, inputs, output):
    _refuse_gradients(ctx, "token_policy_loss",
                      {2: "old_log_probs", 3: "advantages", 4: "ref_log_probs"})
    logits, actions, mask, ctx.temperature = inputs[0], inputs[1], inputs[5], inputs[10]
    ctx.mark_non_differentiable(output[1], output[2])
    ctx.save_for_backward(logits, actions, mask, output[1], output[2])


def _token_policy_grad(ctx, d_scalars, *_):
    logits, actions, mask, saved, coef = ctx.saved_tensors
    d = token_log_probs_backward(logits, actions, mask, ctx.temperature, saved, coef[0], coef[1],
                                 d_scalars[0].clone())
    return (d,) + (None,) * 12


token_policy_loss.register_autograd(_token_policy_grad, setup_context=_token_policy_setup)


@torch.library.custom_op(f"{_NS}::preference_loss", mutates_args=(), device_types="cuda")
def preference_loss(logits: Tensor, actions: Tensor, ref_log_probs: Optional[Tensor],
                    mask: Optional[Tensor], beta: float, label_smoothing: float, margin: float,
                    average: bool, temperature: float) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    tokens._check_preference(logits, actions, ref_log_probs, mask, beta, label_smoothing, margin,
                             temperature)
    relative, _, saved = tokens._log_probs(logits, actions, mask, temperature, ref_log_probs, False,
                                           True)
    loss, rewards, coef = tokens._preference(relative, mask, beta, margin, label_smoothing, average)
    return loss, rewards, saved, coef


@preference_loss.register_fake
def _preference_loss_fake(logits, actions, ref_log_probs, mask, beta, label_smoothing, margin,
                          average, temperature):
    return (logits.new_empty((), dtype=torch.float32),
            logits.new_empty(logits.shape[0], dtype=torch.float32), _saved_like(logits),
            _row_floats(logits))


def _preference_setup(ctx, inputs, output):
    _refuse_gradients(ctx, "preference_loss", {2: "ref_log_probs"})
    logits, actions, mask, ctx.temperature = inputs[0], inputs[1], inputs[3], inputs[8]
    ctx.mark_non_differentiable(*output[1:])
    ctx.save_for_backward(logits, actions, mask, output[2], output[3])


def _preference_grad(ctx, d_loss, *_):
    logits, actions, mask, saved, coef = ctx.saved_tensors
    d = token_log_probs_backward(logits, actions, mask, ctx.temperature, saved, coef, None,
                                 d_loss.contiguous())
    return (d,) + (None,) * 8


preference_loss.register_autograd(_preference_grad, setup_context=_preference_setup)


@torch.library.custom_op(f"{_NS}::distillation_loss", mutates_args=(), device_types="cuda")
def distillation_loss(logits: Tensor, teacher_logits: Tensor, teacher_ids: Tensor,
                      mask: Optional[Tensor], temperature: float, reduction: str,
                      denominator: Optional[float]) -> tuple[Tensor, Tensor]:
    tokens._check_distillation(logits, teacher_logits, teacher_ids, mask, temperature)
    tokens._check_weights(reduction, denominator, 1.0)
    loss = tokens._loss(reduction, denominator, 1.0)
    out, saved, _ = tokens._distill(logits, teacher_logits, teacher_ids, mask, temperature, loss,
                                    True, False)
    return out, saved


@distillation_loss.register_fake
def _distillation_loss_fake(logits, teacher_logits, teacher_ids, mask, temperature, reduction,
                            denominator):
    return logits.new_empty((), dtype=torch.float32), _saved_like(logits)


@torch.library.custom_op(f"{_NS}::distillation_loss_backward", mutates_args=(),
                         device_types="cuda")
def distillation_loss_backward(logits: Tensor, teacher_logits: Tensor, teacher_ids: Tensor,
                               mask: Optional[Tensor], temperature: float, saved: Tensor,
                               scale: Tensor) -> Tensor:
    tokens._check_distillation(logits, teacher_logits, teacher_ids, mask, temperature)
    _check_saved(logits, saved)
    _check_scalar(logits, scale)
    return tokens._distill_backward(logits, teacher_logits, teacher_ids, mask, temperature, saved,
                                    scale)


@distillation_loss_backward.register_fake
def _distillation_loss_backward_fake(logits, teacher_logits, teacher_ids, mask, temperature, saved,
                                     scale):
    return torch.empty_like(logits)


def _distillation_setup(ctx, inputs, output):
    _refuse_gradients(ctx, "distillation_loss", {1: "teacher_logits"})
    logits, teacher, ids, mask, ctx.temperature = inputs[:5]
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(logits, teacher, ids, mask, output[1])


def _distillation_grad(ctx, d_loss, _):
    logits, teacher, ids, mask, saved = ctx.saved_tensors
    d = distillation_loss_backward(logits, teacher, ids, mask, ctx.temperature, saved,
                                   d_loss.contiguous())
    return (d,) + (None,) * 6


distillation_loss.register_autograd(_distillation_grad, setup_context=_distillation_setup)


@torch.library.custom_op(f"{_NS}::top_logits", mutates_args=(), device_types="cuda")
def top_logits(logits: Tensor, k: int) -> tuple[Tensor, Tensor]:
    return tokens.top_logits(logits, k)


@top_logits.register_fake
def _top_logits_fake(logits, k):
    shape = (*logits.shape[:-1], k)
    return logits.new_empty(shape), logits.new_empty(shape, dtype=torch.int64)
