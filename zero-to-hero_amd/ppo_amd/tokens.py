"""Token policies over libppo_tokens (HIP, gfx950): policies that pick one of up
to a vocabulary of actions at every step of a sequence, trained from their
logits.

Next to the reference's PPO loss over a few actions
(rl/deep/agents/ppo.py:141-171), which ops.ppo_loss_discrete runs in fp32,
these are the pieces of wide ones, with no counterpart in the reference:

  token_log_probs    log-probabilities and entropies of the taken actions, and
                     their gradients
  token_policy_loss  the clipped policy loss with a KL term to a reference
                     policy, over masked sequences
  preference_loss    of preferred over rejected sequences, by their log ratios
                     to a reference policy
  distillation_loss  from a teacher's top logits
  top_logits         those: the K largest of each row, in order

Logits are [..., T, A] (fp32, bf16 or fp16): T tokens of each sequence, one
action of A at each.  Where a mask is False a token does not count: nothing of
it is read, and its gradients are 0.  Argument checks, streams and errors
follow ops.py: tensors are contiguous and on one GPU, work is enqueued on
torch's current stream of that device, nothing synchronises, and there is no
CPU fallback.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from .layers import DTYPES, _on, _wants_gradient, _workspace
from .ops import _native, _ptr, _require, _stream

__all__ = ["token_log_probs", "token_policy_loss", "preference_loss", "distillation_loss",
           "top_logits", "TokenStats", "PreferenceStats"]


class TokenStats(dict):
    """token_policy_loss's scalars as 0-d fp32 device tensors: loss, policy, kl,
    entropy, approx_kl, clipfrac (views of one [6] tensor, whose first element
    the returned loss is as well; no host sync)."""


class PreferenceStats(dict):
    """preference_loss's rewards, beta times the sequences' log ratios: chosen
    and rejected, fp32 [P] on the device."""


def _call(name: str, *args) -> None:
    _lib.check(name, getattr(_lib.load_tokens(), name)(*args))


# ---------------------------------------------------------------------------
# Arguments
# ---------------------------------------------------------------------------
def _check_logits(logits, temperature) -> None:
    _require(logits, "logits", tuple(DTYPES))
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"logits must be [..., A] with A > 0, got {tuple(logits.shape)}")
    if not 0.0 < temperature < math.inf:
        raise ValueError(f"temperature must be > 0 and finite, got {temperature}")


def _check_rows(logits, t, name, dtypes) -> None:
    _require(t, name, dtypes, logits.device)
    if t.shape != logits.shape[:-1]:
        raise ValueError(f"{name} must be {tuple(logits.shape[:-1])}, got {tuple(t.shape)}")


def _check_actions(logits, actions, mask) -> None:
    _check_rows(logits, actions, "actions", (torch.int32, torch.int64))
    _check_mask(logits, mask)


def _check_mask(logits, mask) -> None:
    if mask is not None:
        _check_rows(logits, mask, "mask", (torch.bool, torch.uint8))


def _check_weights(reduction, denominator, grad_scale) -> None:
    if reduction not in _lib.TOKEN_REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_lib.TOKEN_REDUCTIONS)}, "
                         f"got {reduction!r}")
    for value, name in ((1.0 if denominator is None else denominator, "denominator"),
                        (grad_scale, "grad_scale")):
        if not _lib.PPO_TOKEN_LEAST <= value <= _lib.PPO_TOKEN_MOST:
            raise ValueError(f"{name} must be in [{_lib.PPO_TOKEN_LEAST}, "
                             f"{_lib.PPO_TOKEN_MOST}], got {value}")


def _sizes(logits) -> tuple[int, int, int]:
    """(sequences, tokens, A)."""
    shape = (1, 1, *logits.shape)
    return math.prod(shape[:-2]), shape[-2], shape[-1]


def _rows(logits, actions, mask, temperature) -> _lib.TokenRows:
    return _lib.TokenRows(logits.data_ptr(), _ptr(actions), _ptr(mask), *_sizes(logits),
                          DTYPES[logits.dtype],
                          int(actions is not None and actions.dtype == torch.int64),
                          float(temperature))


def _loss(reduction, denominator, grad_scale, clip_low=0.0, clip_high=0.0, kl_coef=0.0,
          entropy_coef=0.0, per_sequence=False) -> _lib.TokenLoss:
    return _lib.TokenLoss(float(clip_low), float(clip_high), float(kl_coef), float(entropy_coef),
                          0.0 if denominator is None else float(denominator), float(grad_scale),
                          _lib.TOKEN_REDUCTIONS[reduction], int(per_sequence))


def _scratch(logits):
    nbytes = _lib.load_tokens().ppo_token_workspace_bytes(*_sizes(logits), DTYPES[logits.dtype])
    # (a loss over no rows still takes some)
    return _workspace(max(nbytes, 1 << 20 if logits.numel() == 0 else 0), logits.device)


def _saved(logits) -> torch.Tensor:
    S, T, _ = _sizes(logits)
    return torch.empty((S * T, _lib.PPO_TOKEN_SAVED), dtype=torch.float32, device=logits.device)


def _like_forward(t, dtype, shape, device, what) -> torch.Tensor:
    """What a saved-tensor hook hands back, as the forward pass had it."""
    if t.dtype != dtype or t.shape != shape or t.device != device:
        raise RuntimeError(f"{what}: a saved tensor came back as {t.dtype} {tuple(t.shape)} on "
                           f"{t.device}, expected {dtype} {tuple(shape)} on {device}")
    return t.contiguous()


def _like(logits, actions, mask):
    """What the tensors of every row are, for _saved_rows."""
    return (logits.shape, logits.device, logits.dtype, *(None if t is None else t.dtype
                                                         for t in (actions, mask)))


def _check_constants(what: str, **tensors) -> None:
    """Refuses operands that ask for a gradient which `what` does not form."""
    for name, t in tensors.items():
        if _wants_gradient(t):
            raise RuntimeError(f"{what} has no gradient in {name}: detach it")


def _once(what: str) -> None:
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} can be differentiated once: its backward pass has no "
                           "create_graph")


# ---------------------------------------------------------------------------
# Launches
# ---------------------------------------------------------------------------
def _log_probs(logits, actions, mask, temperature, minus, entropy, save):
    """(log_probs - minus, entropy or None, saved or None)."""
    new = dict(dtype=torch.float32, device=logits.device)
    lp = torch.empty(logits.shape[:-1], **new)
    H = torch.empty(logits.shape[:-1], **new) if entropy else None
    saved = _saved(logits) if save else None
    if lp.numel():
        with _on(logits.device):
            ws = _scratch(logits)
            _call("ppo_token_log_probs", ctypes.byref(_rows(logits, actions, mask, temperature)),
                  _ptr(minus), lp.data_ptr(), _ptr(H), _ptr(saved), ws.data_ptr(), ws.numel(),
                  _stream(logits.device))
    return lp, H, saved


def _log_probs_backward(logits, actions, mask, temperature, saved, dlp, dH, scale=None,
                        held=None, held_for=0.0):
    """dlogits; in `held`, which is left as it is where *scale equals held_for."""
    d = torch.empty_like(logits) if held is None else held
    if d.numel():
        with _on(logits.device):
            _call("ppo_token_log_probs_backward",
                  ctypes.byref(_rows(logits, actions, mask, temperature)), saved.data_ptr(),
                  _ptr(dlp), _ptr(dH), _ptr(scale), 0.0 if held is None else float(held_for),
                  d.data_ptr(), _stream(logits.device))
    return d


def _policy(logits, actions, old, adv, ref, mask, temperature, loss, save, grad):
    """(scalars, saved, coef, dlogits), those not asked for None."""
    new = dict(dtype=torch.float32, device=logits.device)
    scalars = torch.empty(_lib.PPO_TOKEN_SCALARS, **new)
    saved = _saved(logits) if save else None
    coef = torch.empty((2, saved.shape[0]), **new) if save else None
    d = torch.empty_like(logits) if grad else None
    with _on(logits.device):
        ws = _scratch(logits)
        _call("ppo_token_policy_loss", ctypes.byref(_rows(logits, actions, mask, temperature)),
              old.data_ptr(), adv.data_ptr(), _ptr(ref), ctypes.byref(loss), scalars.data_ptr(),
              _ptr(saved), _ptr(coef), _ptr(d), ws.data_ptr(), ws.numel(),
              _stream(logits.device))
    return scalars, saved, coef, d


def _preference(relative, mask, beta, margin, smoothing, average):
    """(loss, rewards [S], coef) of relative [S,T]."""
    S, T = relative.shape
    new = dict(dtype=torch.float32, device=relative.device)
    loss, rewards, coef = torch.empty((), **new), torch.empty(S, **new), torch.empty((S, T), **new)
    with _on(relative.device):
        nbytes = _lib.load_tokens().ppo_token_preference_workspace_bytes(S)
        ws = _workspace(nbytes, relative.device)
        _call("ppo_token_preference", relative.data_ptr(), _ptr(mask), S, T, float(beta),
              float(margin), float(smoothing), int(average), loss.data_ptr(), rewards.data_ptr(),
              coef.data_ptr(), ws.data_ptr(), nbytes, _stream(relative.device))
    return loss, rewards, coef


def _distill(logits, teacher, ids, mask, temperature, loss, save, grad):
    """(loss, saved, dlogits), those not asked for None."""
    out = torch.empty((), dtype=torch.float32, device=logits.device)
    saved = _saved(logits) if save else None
    d = torch.empty_like(logits) if grad else None
    with _on(logits.device):
        ws = _scratch(logits)
        _call("ppo_token_distillation", ctypes.byref(_rows(logits, None, mask, temperature)),
              teacher.data_ptr(), DTYPES[teacher.dtype], ids.data_ptr(),
              int(ids.dtype == torch.int64), ids.shape[-1], ctypes.byref(loss), out.data_ptr(),
              _ptr(saved), _ptr(d), ws.data_ptr(), ws.numel(), _stream(logits.device))
    return out, saved, d


def _distill_backward(logits, teacher, ids, mask, temperature, saved, scale, held=None,
                      held_for=0.0):
    d = torch.empty_like(logits) if held is None else held
    if d.numel():
        with _on(logits.device):
            _call("ppo_token_distillation_backward",
                  ctypes.byref(_rows(logits, None, mask, temperature)), teacher.data_ptr(),
                  DTYPES[teacher.dtype], ids.data_ptr(), int(ids.dtype == torch.int64),
                  ids.shape[-1], saved.data_ptr(), scale.data_ptr(),
                  0.0 if held is None else float(held_for), d.data_ptr(),
                  _stream(logits.device))
    return d


class _Held:
    """A gradient that the forward pass formed for the incoming gradient `value`.
    The first backward pass may take it; a later one, or one that a graph
    replays without that forward pass, forms the gradient anew from the
    logits."""

    def __init__(self, grad, value: float) -> None:
        self.grad, self.value = grad, value
        self.capture = _native().capture_id(grad.device.index)

    def take(self):
        grad, self.grad = self.grad, None
        if grad is not None and _native().capture_id(grad.device.index) != self.capture:
            grad = None
        return grad


def _scale(grad_loss: torch.Tensor) -> torch.Tensor:
    return grad_loss.to(torch.float32).contiguous()


# ---------------------------------------------------------------------------
# Autograd
# ---------------------------------------------------------------------------
class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, mask, temperature, entropy):
        lp, H, saved = _log_probs(logits, actions, mask, temperature, None, entropy, True)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, actions, mask, saved)
        ctx.like = _like(logits, actions, mask)
        return lp, H

    @staticmethod
    def backward(ctx, dlp, dH):
        _once("token_log_probs")
        if dlp is None and dH is None:
            return (None,) * 5
        logits, actions, mask, saved = _saved_rows(ctx, "token_log_probs")
        dlp, dH = (None if g is None else _scale(g) for g in (dlp, dH))
        return (_log_probs_backward(logits, actions, mask, ctx.temperature, saved, dlp, dH),
                None, None, None, None)


def _saved_rows(ctx, what):
    """logits, actions, mask, saved and what else a node saved, checked."""
    shape, device, dtype, actions_dtype, mask_dtype = ctx.like
    logits, actions, mask, saved, *more = ctx.saved_tensors
    rows = shape[:-1]
    return (_like_forward(logits, dtype, shape, device, what),
            None if actions is None else _like_forward(actions, actions_dtype, rows, device, what),
            None if mask is None else _like_forward(mask, mask_dtype, rows, device, what),
            _like_forward(saved, torch.float32, (math.prod(rows), _lib.PPO_TOKEN_SAVED), device,
                          what),
            *more)


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, old, adv, ref, mask, temperature, loss):
        scalars, saved, coef, d = _policy(logits, actions, old, adv, ref, mask, temperature, loss,
                                          True, True)
        ctx.temperature, ctx.held = temperature, _Held(d, loss.grad_scale)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(scalars)
        ctx.save_for_backward(logits, actions, mask, saved, coef)
        ctx.like = _like(logits, actions, mask)
        total = torch.empty(0, dtype=torch.float32, device=logits.device)
        total.set_(scalars.untyped_storage(), scalars.storage_offset(), ())
        return total, scalars

    @staticmethod
    def backward(ctx, grad_loss, _):
        _once("token_policy_loss")
        if grad_loss is None:
            return (None,) * 8
        logits, actions, mask, saved, coef = _saved_rows(ctx, "token_policy_loss")
        coef = _like_forward(coef, torch.float32, (2, saved.shape[0]), saved.device,
                             "token_policy_loss")
        d = _log_probs_backward(logits, actions, mask, ctx.temperature, saved, coef[0], coef[1],
                                _scale(grad_loss), ctx.held.take(), ctx.held.value)
        return (d,) + (None,) * 7


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, ref, mask, temperature, beta, margin, smoothing, average):
        relative, _, saved = _log_probs(logits, actions, mask, temperature, ref, False, True)
        loss, rewards, coef = _preference(relative, mask, beta, margin, smoothing, average)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(rewards)
        ctx.save_for_backward(logits, actions, mask, saved, coef)
        ctx.like = _like(logits, actions, mask)
        return loss, rewards

    @staticmethod
    def backward(ctx, grad_loss, _):
        _once("preference_loss")
        if grad_loss is None:
            return (None,) * 9
        logits, actions, mask, saved, coef = _saved_rows(ctx, "preference_loss")
        coef = _like_forward(coef, torch.float32, logits.shape[:-1], logits.device,
                             "preference_loss")
        d = _log_probs_backward(logits, actions, mask, ctx.temperature, saved, coef, None,
                                _scale(grad_loss))
        return (d,) + (None,) * 8


class _DistillationLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, ids, mask, temperature, loss):
        out, saved, d = _distill(logits, teacher, ids, mask, temperature, loss, True, True)
        ctx.temperature, ctx.held = temperature, _Held(d, loss.grad_scale)
        ctx.save_for_backward(logits, None, mask, saved, teacher, ids)
        ctx.like = _like(logits, None, mask)
        ctx.top = teacher.shape, teacher.dtype, ids.dtype
        return out

    @staticmethod
    def backward(ctx, grad_loss):
        _once("distillation_loss")
        logits, _, mask, saved, teacher, ids = _saved_rows(ctx, "distillation_loss")
        shape, dtype, ids_dtype = ctx.top
        teacher = _like_forward(teacher, dtype, shape, logits.device, "distillation_loss")
        ids = _like_forward(ids, ids_dtype, shape, logits.device, "distillation_loss")
        d = _distill_backward(logits, teacher, ids, mask, ctx.temperature, saved,
                              _scale(grad_loss), ctx.held.take(), ctx.held.value)
        return (d,) + (None,) * 5


# ---------------------------------------------------------------------------
# Functions
# ---------------------------------------------------------------------------
def token_log_probs(
    logits: torch.Tensor,
    actions: torch.Tensor,
    mask: Optional[torch.Tensor] = None,
    temperature: float = 1.0,
    entropy: bool = False,
):
    """log p[action] of each row of logits [..., A] (fp32, bf16 or fp16), p =
    softmax(logits / temperature): fp32 [...], or with `entropy` the pair of
    them and the entropies -sum p log p.

    actions [...] is int32 or int64; one outside [0, A) gives NaN (and is never
    dereferenced).  mask [...] (bool or uint8): where it is False, both are 0,
    and nothing of the row is read.  A logit of -inf is an action that cannot
    be taken.  Both results are differentiable once in the logits
    (create_graph raises)."""
    got = _native().token_log_probs(logits, actions, mask, temperature, entropy)
    if got is not None:
        return got
    _check_logits(logits, temperature)
    _check_actions(logits, actions, mask)
    if _wants_gradient(logits):
        lp, H = _LogProbs.apply(logits, actions, mask, float(temperature), bool(entropy))
    else:
        lp, H, _ = _log_probs(logits, actions, mask, temperature, None, entropy, False)
    return (lp, H) if entropy else lp


def _check_policy(logits, actions, old_log_probs, advantages, ref_log_probs, mask, clip_low,
                  clip_high, kl_coef, entropy_coef, temperature) -> bool:
    """Refuses what the kernels do not take; whether advantages are one a sequence."""
    _check_logits(logits, temperature)
    _check_actions(logits, actions, mask)
    _check_rows(logits, old_log_probs, "old_log_probs", (torch.float32,))
    _require(advantages, "advantages", (torch.float32,), logits.device)
    per_sequence = logits.dim() >= 2 and advantages.shape == logits.shape[:-2]
    if advantages.shape != logits.shape[:-1] and not per_sequence:
        raise ValueError(f"advantages must be {tuple(logits.shape[:-1])} or "
                         f"{tuple(logits.shape[:-2])}, got {tuple(advantages.shape)}")
    if ref_log_probs is not None:
        _check_rows(logits, ref_log_probs, "ref_log_probs", (torch.float32,))
    if not clip_low >= 0.0 or not clip_high >= 0.0:
        raise ValueError(f"clip_low and clip_high must be >= 0, got {clip_low}, {clip_high}")
    for value, name in ((kl_coef, "kl_coef"), (entropy_coef, "entropy_coef")):
        if not abs(value) <= torch.finfo(torch.float32).max:
            raise ValueError(f"{name} must be finite in fp32, got {value}")
    if kl_coef != 0.0 and ref_log_probs is None:
        raise ValueError("kl_coef needs ref_log_probs")
    return per_sequence


def token_policy_loss(
    logits: torch.Tensor,
    actions: torch.Tensor,
    old_log_probs: torch.Tensor,
    advantages: torch.Tensor,
    ref_log_probs: Optional[torch.Tensor] = None,
    mask: Optional[torch.Tensor] = None,
    clip_low: float = 0.2,
    clip_high: Optional[float] = None,
    kl_coef: float = 0.0,
    entropy_coef: float = 0.0,
    temperature: float = 1.0,
    reduction: str = "token",
    denominator: Optional[float] = None,
    grad_scale: float = 1.0,
) -> tuple[torch.Tensor, TokenStats]:
    """Differentiable clipped policy loss over sequences of tokens, with a KL
    term to a reference policy.

    With ratio = exp(log p[action] - old_log_probs) and d = ref_log_probs -
    log p[action], a token's loss is
      -min(ratio adv, clip(ratio, 1 - clip_low, 1 + clip_high) adv)
      + kl_coef (exp(d) - d - 1) - entropy_coef H
    (clip_high None: clip_low), and the loss their mean over the tokens that
    the mask counts (reduction "token"), or over the sequences that have any,
    of their means ("sequence"); `denominator` takes the place of the number of
    those tokens or sequences, for a batch in several calls or ranks (it and
    grad_scale lie in [1e-30, 1e30]).
    logits [..., T, A]; actions, old_log_probs, ref_log_probs and mask [..., T];
    advantages [..., T], or [...] for one a sequence; those three are constants, and
    refused where they require a gradient.  Over no tokens the loss is 0.

    Returns (loss, stats): `loss` is a 0-d tensor to differentiate once in the
    logits, `stats` the same means of the terms, reported values.  The forward
    pass forms the gradient as well, times grad_scale, in its one pass over the
    logits; the backward pass hands it out if the incoming gradient is
    grad_scale (1 for loss.backward(); the scale of a loss scaler otherwise),
    and forms it anew from the logits if not, which costs another pass and
    gives the same: either is rounded once."""
    clip_high = clip_low if clip_high is None else clip_high
    got = _native().token_policy_loss(
        logits, actions, old_log_probs, advantages, ref_log_probs, mask, clip_low, clip_high,
        kl_coef, entropy_coef, temperature, _lib.TOKEN_REDUCTIONS.get(reduction), denominator,
        grad_scale)
    if got is not None:
        return got[0], TokenStats(zip(_lib.TOKEN_SCALAR_NAMES, got[1]))
    per_sequence = _check_policy(logits, actions, old_log_probs, advantages, ref_log_probs, mask,
                                 clip_low, clip_high, kl_coef, entropy_coef, temperature)
    _check_weights(reduction, denominator, grad_scale)
    _check_constants("token_policy_loss", old_log_probs=old_log_probs, advantages=advantages,
                     ref_log_probs=ref_log_probs)
    loss = _loss(reduction, denominator, grad_scale, clip_low, clip_high, kl_coef, entropy_coef,
                 per_sequence)
    args = (logits, actions, old_log_probs, advantages, ref_log_probs, mask, float(temperature),
            loss)
    if _wants_gradient(logits):
        total, scalars = _PolicyLoss.apply(*args)
    else:
        scalars = _policy(*args, False, False)[0]
        total = scalars[0]
    return total, TokenStats({name: scalars.detach()[i]
                              for i, name in enumerate(_lib.TOKEN_SCALAR_NAMES)})


def _check_preference(logits, actions, ref_log_probs, mask, beta, label_smoothing, margin,
                      temperature) -> None:
    _check_logits(logits, temperature)
    if logits.dim() != 3 or logits.shape[0] == 0 or logits.shape[0] % 2:
        raise ValueError("logits must be [2 P, T, A] with P > 0, the chosen sequences first, got "
                         f"{tuple(logits.shape)}")
    _check_actions(logits, actions, mask)
    if ref_log_probs is not None:
        _check_rows(logits, ref_log_probs, "ref_log_probs", (torch.float32,))
    if not math.isfinite(beta) or not math.isfinite(margin):
        raise ValueError(f"beta and margin must be finite, got {beta}, {margin}")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must be in [0, 1], got {label_smoothing}")


def preference_loss(
    logits: torch.Tensor,
    actions: torch.Tensor,
    ref_log_probs: Optional[torch.Tensor] = None,
    mask: Optional[torch.Tensor] = None,
    beta: float = 0.1,
    label_smoothing: float = 0.0,
    margin: float = 0.0,
    average: bool = False,
    temperature: float = 1.0,
) -> tuple[torch.Tensor, PreferenceStats]:
    """Differentiable loss of preferred over rejected sequences.

    logits [2 P, T, A]: the P chosen sequences, then in the same order the P
    rejected ones; actions, ref_log_probs and mask [2 P, T].  A sequence's log
    ratio is the sum (the mean with `average`) of log p[action] - ref_log_probs
    over the tokens that the mask counts, 0 over none; without ref_log_probs
    (constants, refused where they require a gradient) they count as 0.  The loss is the mean over pairs of
      -(1 - label_smoothing) log sigmoid(m) - label_smoothing log sigmoid(-m),
      m = beta (chosen ratio - rejected ratio) - margin.

    Returns (loss, stats): `loss` to differentiate once in the logits, `stats`
    the rewards beta times the log ratios, reported values.  Sums over tokens
    are formed in 64 bits from differences rounded once, so the policy may lie
    close to its reference."""
    got = _native().preference_loss(logits, actions, ref_log_probs, mask, beta, label_smoothing,
                                    margin, average, temperature)
    if got is not None:
        return got[0], PreferenceStats(zip(("chosen", "rejected"), got[1]))
    _check_preference(logits, actions, ref_log_probs, mask, beta, label_smoothing, margin,
                      temperature)
    _check_constants("preference_loss", ref_log_probs=ref_log_probs)
    if _wants_gradient(logits):
        loss, rewards = _PreferenceLoss.apply(logits, actions, ref_log_probs, mask,
                                              float(temperature), beta, margin, label_smoothing,
                                              average)
    else:
        relative = _log_probs(logits, actions, mask, temperature, ref_log_probs, False, False)[0]
        loss, rewards, _ = _preference(relative, mask, beta, margin, label_smoothing, average)
    P = logits.shape[0] // 2
    return loss, PreferenceStats(chosen=rewards[:P], rejected=rewards[P:])


def _check_distillation(logits, teacher_logits, teacher_ids, mask, temperature) -> None:
    _check_logits(logits, temperature)
    _check_mask(logits, mask)
    _require(teacher_logits, "teacher_logits", tuple(DTYPES), logits.device)
    _require(teacher_ids, "teacher_ids", (torch.int32, torch.int64), logits.device)
    if (teacher_logits.dim() != logits.dim() or teacher_logits.shape[:-1] != logits.shape[:-1]
            or teacher_logits.shape[-1] == 0):
        raise ValueError(f"teacher_logits must be {(*logits.shape[:-1], 'K')} with K > 0, got "
                         f"{tuple(teacher_logits.shape)}")
    if teacher_ids.shape != teacher_logits.shape:
        raise ValueError(f"teacher_ids must be {tuple(teacher_logits.shape)}, got "
                         f"{tuple(teacher_ids.shape)}")


def distillation_loss(
    logits: torch.Tensor,
    teacher_logits: torch.Tensor,
    teacher_ids: torch.Tensor,
    mask: Optional[torch.Tensor] = None,
    temperature: float = 1.0,
    reduction: str = "token",
    denominator: Optional[float] = None,
    grad_scale: float = 1.0,
) -> torch.Tensor:
    """Differentiable distillation from a teacher's K top logits (top_logits):
    temperature^2 times the mean of sum_k q_k (log q_k - log p[id_k]), q the
    softmax of teacher_logits / temperature over the row's K entries, p that of
    the student's whole row of logits [..., A].

    teacher_logits [..., K] (fp32, bf16 or fp16, K up to 256) and teacher_ids
    [..., K] (int32 or int64).  An entry with a negative id is none; entries of
    one id add up; an id from A on gives NaN; a row without entries, or with
    none but -inf, adds 0 to the loss, has no gradient and counts.  mask, reduction, denominator and grad_scale are
    token_policy_loss's.  Differentiable once in the student's logits alone."""
    got = _native().distillation_loss(logits, teacher_logits, teacher_ids, mask, temperature,
                                      _lib.TOKEN_REDUCTIONS.get(reduction), denominator,
                                      grad_scale)
    if got is not None:
        return got
    _check_distillation(logits, teacher_logits, teacher_ids, mask, temperature)
    _check_weights(reduction, denominator, grad_scale)
    if _wants_gradient(teacher_logits):
        raise RuntimeError("distillation_loss has no gradient in the teacher's logits: detach them")
    loss = _loss(reduction, denominator, grad_scale)
    args = (logits, teacher_logits, teacher_ids, mask, float(temperature), loss)
    if _wants_gradient(logits):
        return _DistillationLoss.apply(*args)
    return _distill(*args, False, False)[0]


def top_logits(logits: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(values [..., k], ids int64 [..., k]): the k largest of each row of logits
    [..., A] (fp32, bf16 or fp16) in falling order and their columns, k up to
    256.  Equal logits come in the order of their columns (0 and -0 are equal),
    NaN before everything, as torch.sort(descending=True, stable=True) puts
    them.  A up to 2^22.  Not differentiable."""
    got = _native().top_logits(logits, k)
    if got is not None:
        return got
    _check_logits(logits, 1.0)
    A = logits.shape[-1]
    if not isinstance(k, int) or isinstance(k, bool):
        raise TypeError(f"k must be an int, got {type(k).__name__}")
    if not 1 <= k <= min(A, _lib.PPO_TOKEN_MAX_K):
        raise ValueError(f"k must be in [1, {min(A, _lib.PPO_TOKEN_MAX_K)}], got {k}")
    device = logits.device
    values = torch.empty((*logits.shape[:-1], k), dtype=logits.dtype, device=device)
    ids = torch.empty((*logits.shape[:-1], k), dtype=torch.int64, device=device)
    rows, dtype = logits.numel() // A, DTYPES[logits.dtype]
    if rows:
        with _on(device):
            nbytes = _lib.load_tokens().ppo_token_top_workspace_bytes(rows, A, k, dtype)
            ws = _workspace(nbytes, device)
            _call("ppo_token_top", logits.data_ptr(), dtype, rows, A, k, values.data_ptr(),
                  ids.data_ptr(), _ptr(ws), nbytes, _stream(device))
    return values, ids
