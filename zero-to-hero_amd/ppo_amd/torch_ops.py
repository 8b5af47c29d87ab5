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

The loss operators are differentiable in their first output: backward of
scalars[0] (the total loss; the other scalars are reported values) scales the
fused kernel's gradients by the incoming gradient, as ops.ppo_loss_discrete
does.  Their gradient outputs are marked non-differentiable.
"""

from typing import Optional

import torch
from torch import Tensor

from . import _lib, layers, ops

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
