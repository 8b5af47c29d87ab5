"""Feed-forward layers of a policy network over libppo_layers (HIP, gfx950).

Next to the reference's Linear-act-Linear-act-Linear networks
(rl/deep/agents/common.py:16-28), which the fused minibatch kernels of ops.py
run at hidden sizes up to 128, these are the pieces of larger ones, with no
counterpart in the reference:

  gated_ffn      dropout(act(x wg^T + bg) * (x wu^T + bu)) and its gradients
  dropout        a mask formed from (seed, row id, column), never stored
  quantize_rows  8-bit rows with one scale each
  int8_linear    the 8-bit product with a scale per row and per output channel,
                 for acting with a quantised policy

and the modules GatedLinear, GatedMLP, Int8Linear and int8_copy built on
them.  Argument checks, streams and errors follow ops.py: tensors are
contiguous and on one GPU, work is enqueued on torch's current stream of that
device, nothing synchronises, and there is no CPU fallback.
"""

from __future__ import annotations

import contextlib
import copy
import ctypes
import math
from typing import Optional, Union

import torch
import torch.autograd.forward_ad as fwd_ad
from torch import nn

from . import _lib
from .ops import _native, _ptr, _require, _stream

__all__ = ["gated_ffn", "dropout", "quantize_rows", "int8_linear", "GatedLinear", "GatedMLP",
           "Int8Linear", "int8_copy"]

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"relu": 0, "tanh": 1, "silu": 2, "gelu": 3}
Seed = Union[int, torch.Tensor]


def _on(device: torch.device):
    """Launches go to the tensors' device, whichever is current."""
    if device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _workspace(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    """Scratch of one call.  From torch's allocator, not a buffer kept per
    stream: a captured graph then owns the scratch that its replays write, so
    graphs replayed side by side share none."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _aligned(*operands: torch.Tensor) -> int:
    """PPO_LAYER_ALIGNED where the operands start at multiples of 16 bytes: no
    room for aligned copies of them is needed then."""
    return 0 if any(t.data_ptr() % 16 for t in operands) else _lib.PPO_LAYER_ALIGNED


def _call(name: str, *args) -> None:
    _lib.check(name, getattr(_lib.load_layers(), name)(*args))


def _wants_gradient(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a derivative would have to pass, in either direction."""
    given = [t for t in tensors if t is not None]
    return (torch.is_grad_enabled() and any(t.requires_grad for t in given)
            or any(fwd_ad.unpack_dual(t).tangent is not None for t in given))


def _check_drop(p: float, seed: Seed, rows: Optional[torch.Tensor], M: int, device) -> None:
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"the dropout probability must be in [0, 1], got {p}")
    if isinstance(seed, torch.Tensor):
        _require(seed, "seed", (torch.int64,), device)
        if seed.numel() != 1:
            raise ValueError(f"seed must hold one value, got {seed.numel()}")
    elif not isinstance(seed, int):
        raise TypeError(f"seed must be an int or an int64 tensor, got {type(seed).__name__}")
    if rows is not None:
        _require(rows, "rows", (torch.int64,), device)
        if rows.dim() != 1 or rows.numel() != M:
            raise ValueError(f"rows must be [M]=[{M}], got {tuple(rows.shape)}")


def _drop(p: float, seed: Seed, rows: Optional[torch.Tensor]) -> _lib.Dropout:
    at = seed.data_ptr() if isinstance(seed, torch.Tensor) else None
    return _lib.Dropout(float(p), 0 if at else int(seed) & (2**64 - 1), at, _ptr(rows))


# ---------------------------------------------------------------------------
# Dropout
# ---------------------------------------------------------------------------
def _dropout_into(x: torch.Tensor, drop: _lib.Dropout) -> torch.Tensor:
    y = torch.empty_like(x)
    if x.numel():
        cols = x.shape[-1]
        with _on(x.device):
            _call("ppo_layer_dropout", x.data_ptr(), y.data_ptr(), DTYPES[x.dtype],
                  x.numel() // cols, cols, ctypes.byref(drop), _stream(x.device))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, rows):
        ctx.p, ctx.seed = p, None if isinstance(seed, torch.Tensor) else seed
        ctx.save_for_backward(seed if ctx.seed is None else None, rows)
        return _dropout_into(x, _drop(p, seed, rows))

    @staticmethod
    def backward(ctx, dy):
        seed, rows = ctx.saved_tensors
        # (a saved-tensor hook hands back whatever it likes)
        _check_drop(ctx.p, ctx.seed if seed is None else seed, rows,
                    dy.numel() // dy.shape[-1] if dy.numel() else math.prod(dy.shape[:-1]),
                    dy.device)
        # linear in x: its derivative is the same mask (create_graph comes again)
        return (_Dropout.apply(dy.contiguous(), ctx.p, ctx.seed if seed is None else seed, rows),
                None, None, None)


def dropout(x: torch.Tensor, p: float, seed: Seed, rows: Optional[torch.Tensor] = None
            ) -> torch.Tensor:
    """Dropout of x [..., C] (fp32, bf16 or fp16): elements are kept with
    probability 1 - p and divided by 1 - p, others are 0.

    The mask is a function of (seed, row id, column): with the same arguments
    it is the same mask, on any device, stream or batch.  Row ids are `rows`
    (int64 [M], M the product of the leading sizes; ids may repeat), or
    0..M-1: with the samples' rollout indices as row ids, a minibatch of an
    update meets the masks its samples were acted with, whatever their order,
    so the first ratio of a PPO update is 1.  `seed` is an int (its low 64
    bits), or an int64 tensor of one value on x's device that is read when the
    kernel runs, so that a captured graph takes a new one per replay.

    Differentiable in x; the backward pass forms the mask again, from `seed`
    and `rows` as they were (neither may be changed in place in between).
    Other than torch's, it drops infinities and NaN to 0.
    """
    got = _native().layer_dropout(x, p, seed, rows)
    if got is not None:
        return got
    _require(x, "x", tuple(DTYPES))
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    M = x.numel() // x.shape[-1] if x.numel() else math.prod(x.shape[:-1])
    _check_drop(p, seed, rows, M, x.device)
    return _Dropout.apply(x, p, seed, rows)


# ---------------------------------------------------------------------------
# Gated feed-forward block
# ---------------------------------------------------------------------------
def _check_gated_operands(x, w_gate, w_up, b_gate=None, b_up=None) -> None:
    _require(x, "x", tuple(DTYPES))
    device, dtype = x.device, (x.dtype,)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must be [..., D] with D > 0, got {tuple(x.shape)}")
    D = x.shape[-1]
    _require(w_gate, "w_gate", dtype, device)
    _require(w_up, "w_up", dtype, device)
    if w_gate.dim() != 2 or w_gate.shape[1] != D or w_gate.shape[0] == 0:
        raise ValueError(f"w_gate must be [F,{D}] with F > 0, got {tuple(w_gate.shape)}")
    if w_up.shape != w_gate.shape:
        raise ValueError(f"w_up must be {tuple(w_gate.shape)}, got {tuple(w_up.shape)}")
    F = w_gate.shape[0]
    if (b_gate is None) != (b_up is None):
        raise ValueError("b_gate and b_up go together")
    for b, name in ((b_gate, "b_gate"), (b_up, "b_up")):
        if b is not None:
            _require(b, name, dtype, device)
            if b.shape != (F,):
                raise ValueError(f"{name} must be [{F}], got {tuple(b.shape)}")


def _check_activation(activation) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return ACTIVATIONS[activation]


def _check_gated(x, w_gate, w_up, b_gate, b_up, activation, dropout_p, seed, rows) -> int:
    """Refuses what the kernels do not take; the activation's number."""
    _check_gated_operands(x, w_gate, w_up, b_gate, b_up)
    act = _check_activation(activation)
    _check_drop(dropout_p, seed, rows, x.numel() // x.shape[-1], x.device)
    return act


def _check_gated_backward(dh, x, w_gate, w_up, saved, dropout_p, seed, rows) -> None:
    """Refuses what the backward kernels do not take."""
    _check_gated_operands(x, w_gate, w_up)
    M, F = x.numel() // x.shape[-1], w_gate.shape[0]
    _check_drop(dropout_p, seed, rows, M, x.device)
    _require(dh, "dh", (x.dtype,), x.device)
    if dh.shape != (*x.shape[:-1], F):
        raise ValueError(f"dh must be {(*x.shape[:-1], F)}, got {tuple(dh.shape)}")
    _require(saved, "saved", (torch.float32,), x.device)
    if saved.shape != (2, M, (F + 3) // 4 * 4):
        raise ValueError(f"saved must be {(2, M, (F + 3) // 4 * 4)}, got {tuple(saved.shape)}")


def _gated_forward(x, wg, wu, bg, bu, act, p, seed, rows, save):
    D, F = x.shape[-1], wg.shape[0]
    M, device, dtype = x.numel() // D, x.device, DTYPES[x.dtype]
    h = torch.empty((*x.shape[:-1], F), dtype=x.dtype, device=device)
    saved = None
    if save:
        saved = torch.empty((2, M, (F + 3) // 4 * 4), dtype=torch.float32, device=device)
    if M:
        drop = _drop(p, seed, rows)
        dtype |= _aligned(x, wg, wu)
        with _on(device):
            nbytes = _lib.load_layers().ppo_layer_gated_workspace_bytes(dtype, M, D, F)
            ws = _workspace(nbytes, device)
            _call("ppo_layer_gated_forward", x.data_ptr(), wg.data_ptr(), wu.data_ptr(), _ptr(bg),
                  _ptr(bu), dtype, M, D, F, act, ctypes.byref(drop), h.data_ptr(), _ptr(saved),
                  _ptr(ws), nbytes, _stream(device))
    return h, saved


def _gated_backward(dh, x, wg, wu, saved, act, p, seed, rows, need):
    """dx, dwg, dwu, dbg, dbu; None for those that `need` does not ask for."""
    D, F = x.shape[-1], wg.shape[0]
    M, device, dtype = x.numel() // D, x.device, DTYPES[x.dtype]
    new = torch.empty if M else torch.zeros
    like = dict(dtype=x.dtype, device=device)
    dx = torch.empty_like(x) if need[0] else None
    dwg = dwu = dbg = dbu = None
    if need[1] or need[2]:
        dwg, dwu = new((F, D), **like), new((F, D), **like)
    if need[3] or need[4]:
        dbg, dbu = new(F, **like), new(F, **like)
    if M:
        drop = _drop(p, seed, rows)
        dtype |= _aligned(x, wg, wu)
        with _on(device):
            nbytes = _lib.load_layers().ppo_layer_gated_backward_workspace_bytes(dtype, M, D, F)
            ws = _workspace(nbytes, device)
            _call("ppo_layer_gated_backward", dh.data_ptr(), x.data_ptr(), wg.data_ptr(),
                  wu.data_ptr(), saved.data_ptr(), dtype, M, D, F, act, ctypes.byref(drop),
                  _ptr(dx), _ptr(dwg), _ptr(dwu), _ptr(dbg), _ptr(dbu), _ptr(ws), nbytes,
                  _stream(device))
    return (dx, dwg if need[1] else None, dwu if need[2] else None, dbg if need[3] else None,
            dbu if need[4] else None)


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, bg, bu, act, p, seed, rows):
        h, saved = _gated_forward(x, wg, wu, bg, bu, act, p, seed, rows, True)
        ctx.act, ctx.p = act, p
        ctx.seed = None if isinstance(seed, torch.Tensor) else seed
        ctx.save_for_backward(x, wg, wu, saved, seed if ctx.seed is None else None, rows)
        return h

    @staticmethod
    def backward(ctx, dh):
        if torch.is_grad_enabled():
            raise RuntimeError("gated_ffn can be differentiated once: its backward pass has no "
                               "create_graph")
        x, wg, wu, saved, seed, rows = ctx.saved_tensors
        seed = ctx.seed if seed is None else seed
        dh = dh.contiguous()
        # (a saved-tensor hook hands back whatever it likes)
        _check_gated_backward(dh, x, wg, wu, saved, ctx.p, seed, rows)
        grads = _gated_backward(dh, x, wg, wu, saved, ctx.act, ctx.p, seed, rows,
                                ctx.needs_input_grad)
        return (*grads, None, None, None, None)


def gated_ffn(
    x: torch.Tensor,
    w_gate: torch.Tensor,
    w_up: torch.Tensor,
    b_gate: Optional[torch.Tensor] = None,
    b_up: Optional[torch.Tensor] = None,
    activation: str = "silu",
    dropout_p: float = 0.0,
    seed: Seed = 0,
    rows: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """dropout(act(x w_gate^T + b_gate) * (x w_up^T + b_up)) in one kernel.

    x [..., D], weights [F, D] as nn.Linear holds them, biases [F] (both or
    neither), all fp32, bf16 or fp16 alike; returns [..., F].  `activation` is
    "relu", "tanh", "silu" or "gelu" (with the error function).  The dropout
    arguments are those of dropout(), whose mask over [M, F] it applies.
    Differentiable once in x, the weights and the biases (create_graph raises):
    g and u are kept for the backward pass in 32 bits (8 M F bytes), the mask
    is formed again.  The gradients of g and u are rounded to x's type for the
    products behind them: 16-bit gradients are off by up to 1.4 times what
    their own rounding makes, and in fp16 those past 65504 become infinite
    (scale the loss accordingly).
    """
    got = _native().layer_gated_ffn(x, w_gate, w_up, b_gate, b_up,
                                    ACTIVATIONS.get(activation), dropout_p, seed, rows)
    if got is not None:
        return got
    act = _check_gated(x, w_gate, w_up, b_gate, b_up, activation, dropout_p, seed, rows)
    leaves = (x, w_gate, w_up, b_gate, b_up)
    if _wants_gradient(*leaves):  # (a tangent is refused there)
        return _GatedFFN.apply(*leaves, act, dropout_p, seed, rows)
    return _gated_forward(*leaves, act, dropout_p, seed, rows, False)[0]


# ---------------------------------------------------------------------------
# 8-bit products
# ---------------------------------------------------------------------------
def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q int8 like x, scale fp32 [...]) of x [..., K] (fp32, bf16 or fp16):
    scale = max |x| times 1/127 (in fp32) of each row and q = x / scale to the
    nearest integer, ties to even.  For a weight [N, K] these are int8_linear's weight
    and weight_scale.  A row of zeros has scale 0; one that holds an infinity
    or a NaN has scale NaN and q = 0, so products with it are NaN.  Not
    differentiable."""
    got = _native().layer_quantize_rows(x)
    if got is not None:
        return got
    _require(x, "x", tuple(DTYPES))
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must be [..., K] with K > 0, got {tuple(x.shape)}")
    K = x.shape[-1]
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if x.numel():
        with _on(x.device):
            _call("ppo_layer_quantize_rows", x.data_ptr(), DTYPES[x.dtype], x.numel() // K, K,
                  q.data_ptr(), scale.data_ptr(), _stream(x.device))
    return q, scale


def int8_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    x_scale: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """x weight^T in 8 bits: (sum_k xq wq) * x_scale * weight_scale + bias.

    weight int8 [N, K] and weight_scale fp32 [N] come from quantize_rows.  x
    is fp32, bf16 or fp16 [..., K], whose rows are quantised in the same call,
    or int8 with x_scale fp32 [...] (quantize_rows' pair, for several products
    of one x).  Sums are exact in int32 (K <= 131072), scales and bias applied
    in fp32, the result rounded once to out_dtype (default: x's type; needed
    for an int8 x).  bias [N] has the result's type.  For acting: not
    differentiable, and refused where x, a scale or the bias requires a
    gradient."""
    got = _native().layer_int8_linear(x, weight, weight_scale, bias, x_scale, out_dtype)
    if got is not None:
        return got
    _require(x, "x", (*DTYPES, torch.int8))
    device = x.device
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must be [..., K] with K > 0, got {tuple(x.shape)}")
    if _wants_gradient(x, weight_scale, bias, x_scale):
        raise RuntimeError("int8_linear has no gradient: call it under torch.no_grad()")
    K = x.shape[-1]
    _require(weight, "weight", (torch.int8,), device)
    if weight.dim() != 2 or weight.shape[1] != K or weight.shape[0] == 0:
        raise ValueError(f"weight must be [N,{K}] with N > 0, got {tuple(weight.shape)}")
    N, M = weight.shape[0], x.numel() // K
    _require(weight_scale, "weight_scale", (torch.float32,), device)
    if weight_scale.shape != (N,):
        raise ValueError(f"weight_scale must be [{N}], got {tuple(weight_scale.shape)}")
    eight = x.dtype == torch.int8
    if eight != (x_scale is not None):
        raise ValueError("x_scale goes with an int8 x")
    if eight:
        _require(x_scale, "x_scale", (torch.float32,), device)
        if x_scale.shape != x.shape[:-1]:
            raise ValueError(f"x_scale must be {tuple(x.shape[:-1])}, got {tuple(x_scale.shape)}")
        if out_dtype is None:
            raise ValueError("an int8 x needs out_dtype")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in DTYPES or (not eight and out_dtype != x.dtype):
        raise TypeError(f"out_dtype {out_dtype}: expected x's type, or one of "
                        f"{', '.join(map(str, DTYPES))} for an int8 x")
    if bias is not None:
        _require(bias, "bias", (out_dtype,), device)
        if bias.shape != (N,):
            raise ValueError(f"bias must be [{N}], got {tuple(bias.shape)}")
    out = torch.empty((*x.shape[:-1], N), dtype=out_dtype, device=device)
    if M:
        flag = _aligned(x, weight) if eight else _aligned(weight)
        with _on(device):
            nbytes = _lib.load_layers().ppo_layer_int8_linear_workspace_bytes(
                M, N, K, int(not eight) | flag)
            ws = _workspace(nbytes, device)
            _call("ppo_layer_int8_linear", None if eight else x.data_ptr(),
                  x.data_ptr() if eight else None, _ptr(x_scale), weight.data_ptr(),
                  weight_scale.data_ptr(), _ptr(bias), DTYPES[out_dtype] | flag, M, N, K,
                  out.data_ptr(), _ptr(ws), nbytes, _stream(device))
    return out


# ---------------------------------------------------------------------------
# Modules
# ---------------------------------------------------------------------------
def _int64(seed: int) -> int:
    """The low 64 bits of an int as an int64 tensor holds them."""
    return (int(seed) + 2**63) % 2**64 - 2**63


class GatedLinear(nn.Module):
    """gated_ffn with its parameters: weights and biases initialised as two
    nn.Linear's (gate first).  Dropout acts in training mode; `seed` is a
    buffer (int64 [1], reseed() fills it with the low 64 bits of an int), so
    captured graphs read its current value.  Nothing else changes it: until the
    next reseed() a row id (or position) meets the same mask in every call."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 activation: str = "silu", dropout: float = 0.0, seed: int = 0) -> None:
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"dropout must be in [0, 1], got {dropout}")
        self.in_features, self.out_features = in_features, out_features
        self.activation, self.dropout = activation, dropout
        gate, up = (nn.Linear(in_features, out_features, bias) for _ in range(2))
        self.weight_gate, self.bias_gate = gate.weight, gate.bias
        self.weight_up, self.bias_up = up.weight, up.bias
        self.register_buffer("seed", torch.tensor([_int64(seed)], dtype=torch.int64))

    def reseed(self, seed: int) -> None:
        self.seed.fill_(_int64(seed))

    def forward(self, x: torch.Tensor, rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        p = self.dropout if self.training else 0.0
        # (a copy: the buffer may be reseeded before the backward pass)
        return gated_ffn(x, self.weight_gate, self.weight_up, self.bias_gate, self.bias_up,
                         self.activation, p, self.seed + 0 if p > 0.0 else 0, rows)


class GatedMLP(nn.Module):
    """The shape of agent.MLP with gated hidden layers: two GatedLinear and an
    nn.Linear.  `rows` are dropout's row ids (the samples' rollout indices)."""

    def __init__(self, input_size: int, hidden_size: int, output_size: int,
                 activation: str = "silu", dropout: float = 0.0, seed: int = 0) -> None:
        super().__init__()
        self.hidden = nn.ModuleList([
            GatedLinear(input_size, hidden_size, True, activation, dropout, 2 * seed),
            GatedLinear(hidden_size, hidden_size, True, activation, dropout, 2 * seed + 1),
        ])
        self.out = nn.Linear(hidden_size, output_size)

    def reseed(self, seed: int) -> None:
        """New masks: every layer's seed is a function of `seed` alone."""
        for i, layer in enumerate(self.hidden):
            layer.reseed(2 * seed + i)

    def forward(self, x: torch.Tensor, rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        for layer in self.hidden:
            x = layer(x, rows)
        return self.out(x)


class Int8Linear(nn.Module):
    """The 8-bit copy of an nn.Linear, for acting: int8_linear over its
    quantised weight, its bias kept as it is."""

    def __init__(self, linear: nn.Linear) -> None:
        super().__init__()
        q, scale = quantize_rows(linear.weight.detach())
        self.register_buffer("weight", q)
        self.register_buffer("weight_scale", scale)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().clone())

    @torch.no_grad()
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return int8_linear(x, self.weight, self.weight_scale, self.bias)


class _Int8Gated(nn.Module):
    """The 8-bit copy of a GatedLinear: x is quantised once for both products,
    whose results stay in 32 bits up to the block's own; no dropout."""

    def __init__(self, layer: GatedLinear) -> None:
        super().__init__()
        self.act = {"relu": torch.relu, "tanh": torch.tanh, "silu": nn.functional.silu,
                    "gelu": nn.functional.gelu}[layer.activation]
        for name, w, b in (("gate", layer.weight_gate, layer.bias_gate),
                           ("up", layer.weight_up, layer.bias_up)):
            q, scale = quantize_rows(w.detach())
            self.register_buffer(f"weight_{name}", q)
            self.register_buffer(f"scale_{name}", scale)
            self.register_buffer(f"bias_{name}", None if b is None
                                 else b.detach().to(torch.float32, copy=True))

    @torch.no_grad()
    def forward(self, x: torch.Tensor, rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        q, s = quantize_rows(x)
        g = int8_linear(q, self.weight_gate, self.scale_gate, self.bias_gate, s, torch.float32)
        u = int8_linear(q, self.weight_up, self.scale_up, self.bias_up, s, torch.float32)
        return torch.mul(self.act(g), u, out=torch.empty_like(g, dtype=x.dtype))


def int8_copy(module: nn.Module) -> nn.Module:
    """A copy of `module` for acting, with every nn.Linear and GatedLinear in
    it (agent.MLP's and GatedMLP's among them; subclasses stay as they are)
    replaced by its 8-bit copy.  The copy does not follow later updates: take a
    new one per rollout."""
    eight = {nn.Linear: Int8Linear, GatedLinear: _Int8Gated}
    # (deepcopy takes what the memo already holds in place of a copy)
    memo = {id(m): eight[type(m)](m) for m in module.modules() if type(m) in eight}
    return copy.deepcopy(module, memo)
