"""The feed-forward layers of a policy network, as measurable cases.

Every case is one pass through a public layer operator of ppo_amd: the gated
feed-forward block with its gradients (gated_ffn in training), the same block
when acting (no gradients), dropout with a mask that is regenerated from
counters in the backward pass (dropout), the 8-bit quantisation of rows
(quantize_rows) and the 8-bit matrix product with a scale per row and per
output channel (int8_linear).  Where `own` is false the same results come
from elementary torch operations in 32 bits; exact() restates them in 64 bits.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ROWS_SPAN = 1 << 23  # samples of a rollout that row indices address


def listed():
    return [
        # the hidden layer of the reference's 128-wide networks over one of its
        # minibatches of 128: the smallest call, launches and latency
        dict(name="drop_128x128_fp32", path="dropout", M=128, D=128, dtype="fp32", p=0.1,
             rows=True),
        # the hidden layer of a wide trunk over a large minibatch
        dict(name="drop_16384x8192_bf16", path="dropout", M=16384, D=8192, dtype="bf16", p=0.1,
             rows=False),
        # one minibatch of 256 through a 128-wide fp32 network: the update loop's
        # own sizes, where every launch counts
        dict(name="train_256x128x256_fp32", path="train", M=256, D=128, F=256, dtype="fp32",
             act="silu", bias=True, p=0.0),
        # a minibatch through a medium trunk, dropout keyed by sample indices
        dict(name="train_4096x1024x2048_bf16", path="train", M=4096, D=1024, F=2048,
             dtype="bf16", act="gelu", bias=False, p=0.1),
        # a wide trunk: the matrix cores' case
        dict(name="train_8192x4096x8192_bf16", path="train", M=8192, D=4096, F=8192,
             dtype="bf16", act="silu", bias=False, p=0.0),
        # sizes that no vector width divides, with biases
        dict(name="train_1000x1023x1365_fp16", path="train", M=1000, D=1023, F=1365,
             dtype="fp16", act="silu", bias=True, p=0.1),
        # one environment's action: the weights are read once for one row
        dict(name="act_1x4096x8192_bf16", path="act", M=1, D=4096, F=8192, dtype="bf16",
             act="silu", bias=False, p=0.0),
        # one step of 4096 environments through an fp32 trunk
        dict(name="act_4096x512x1024_fp32", path="act", M=4096, D=512, F=1024, dtype="fp32",
             act="tanh", bias=True, p=0.0),
        # acting with 8-bit weights: one environment, and a large vector of them
        dict(name="int8_1x4096x4096_bf16", path="int8", M=1, D=4096, F=4096, dtype="bf16",
             bias=False),
        dict(name="int8_8192x4096x8192_bf16", path="int8", M=8192, D=4096, F=8192,
             dtype="bf16", bias=True),
        # observations of 512 features from 4096 environments, and a wide weight
        dict(name="quant_4096x512_fp32", path="quantize", M=4096, D=512, dtype="fp32"),
        dict(name="quant_16384x8192_bf16", path="quantize", M=16384, D=8192, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of the range; half of them are multiples of 64, as layer widths
    and minibatches mostly are."""
    n = _log_int(rng, lo, hi)
    return max(64, n // 64 * 64) if n >= 64 and rng.random() < 0.5 else n


def draw(rng):
    path = rng.choice(["dropout", "train", "train", "act", "int8", "int8", "quantize"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    flag = lambda: rng.random() < 0.5  # noqa: E731
    p = rng.choice([0.05, 0.1, 0.3, 0.5])
    if path in ("dropout", "quantize"):
        M = _size(rng, 1, 16384)
        D = _size(rng, 8, min(16384, (1 << 26) // M))
        return dict(path=path, M=M, D=D, dtype=dtype,
                    **(dict(p=p, rows=flag()) if path == "dropout" else {}))
    limit = 1 << (34 if dtype == "fp32" and path != "int8" else 36)
    M = _size(rng, 1, 8192)
    D = _size(rng, 16, 4096)
    F = _size(rng, 16, max(16, min(8192, limit // (M * D))))
    if path == "int8":
        return dict(path=path, M=M, D=D, F=F, dtype=dtype, bias=flag())
    # (at relu's kink the sums' last bits decide a gradient; 16-bit types show that less)
    act = rng.choice(["tanh", "silu", "gelu"] + ([] if dtype == "fp32" else ["relu"]))
    return dict(path=path, M=M, D=D, F=F, dtype=dtype, act=act, bias=flag(),
                p=p if path == "train" and flag() else 0.0)


def work(case):
    M, D, size = case["M"], case["D"], DTYPES[case["dtype"]].itemsize
    if case["path"] == "dropout":  # forward and backward each read and write the tensor
        return {"bytes": 4 * M * D * size + (8 * M if case["rows"] else 0), "flops": 0}
    if case["path"] == "quantize":
        return {"bytes": M * D * (size + 1) + 4 * M, "flops": 0}
    F = case["F"]
    if case["path"] == "int8":
        return {"bytes": M * D * size + F * D + 4 * F + M * F * size
                + (F * size if case["bias"] else 0), "flops": 2 * M * D * F}
    weights = 2 * F * D + (2 * F if case["bias"] else 0)
    if case["path"] == "act":
        return {"bytes": (M * D + weights + M * F) * size, "flops": 4 * M * D * F}
    # training: x, weights and dh in; h, dx and the weights' gradients out
    return {"bytes": (2 * M * D + 2 * weights + 2 * M * F) * size
            + (8 * M if case["p"] > 0 else 0), "flops": 12 * M * D * F}


# --- inputs, from the seed alone ------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * seed + 29)
    return g


def _rn(g, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _key(seed):
    """The 64-bit dropout seed of a training step."""
    return (seed * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 63)


def _sample_rows(g, M):
    """Indices of a minibatch's samples in the rollout it was drawn from."""
    return torch.randint(0, ROWS_SPAN, (M,), generator=g, device="cuda")


def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    M, D, path = case["M"], case["D"], case["path"]
    s = dict(case=case, key=_key(seed), rows=None)
    if path == "quantize":
        s["x"] = _rn(g, dt, M, D)
        return s
    # activations after a normalisation: unit scale
    s["x"] = _rn(g, dt, M, D)
    if path == "dropout":
        s["x"].requires_grad_()
        s["dy"] = _rn(g, dt, M, D, scale=0.1)
        s["rows"] = _sample_rows(g, M) if case["rows"] else None
        return s
    F = case["F"]
    if path == "int8":
        w = _rn(g, torch.float32, F, D, scale=D ** -0.5)
        # what a policy's 8-bit copy holds: int8 rows and a scale per output channel
        s["ws"] = (w.abs().amax(1) / 127.0).contiguous()
        s["wq"] = torch.round(w / s["ws"][:, None]).to(torch.int8)
        s["b"] = _rn(g, dt, F, scale=0.1) if case["bias"] else None
        return s
    s["wg"] = _rn(g, dt, F, D, scale=D ** -0.5)
    s["wu"] = _rn(g, dt, F, D, scale=D ** -0.5)
    s["bg"] = _rn(g, dt, F, scale=0.1) if case["bias"] else None
    s["bu"] = _rn(g, dt, F, scale=0.1) if case["bias"] else None
    if path == "train":
        s["dh"] = _rn(g, dt, M, F, scale=0.1)
        s["rows"] = _sample_rows(g, M) if case["p"] > 0 else None
        for k in ("x", "wg", "wu", "bg", "bu"):
            if s[k] is not None:
                s[k].requires_grad_()
    return s


def _leaves(s):
    return [s[k] for k in ("x", "wg", "wu", "bg", "bu") if s[k] is not None]


# --- the framework's operators ------------------------------------------------------------

def _package():
    if "ppo_amd" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(
            os.path.abspath(__file__))), "zero-to-hero_amd"))
    import ppo_amd

    return ppo_amd


def _run_own(s):
    amd, case = _package(), s["case"]
    if case["path"] == "dropout":
        y = amd.dropout(s["x"], case["p"], s["key"], rows=s["rows"])
        (dx,) = torch.autograd.grad(y, [s["x"]], s["dy"])
        return {"y": y.detach(), "dx": dx}
    if case["path"] == "quantize":
        q, scale = amd.quantize_rows(s["x"])
        return {"q": q, "scale": scale}
    if case["path"] == "int8":
        return amd.int8_linear(s["x"], s["wq"], s["ws"], bias=s["b"])
    if case["path"] == "act":
        with torch.no_grad():
            return amd.gated_ffn(s["x"], s["wg"], s["wu"], s["bg"], s["bu"],
                                 activation=case["act"])
    h = amd.gated_ffn(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=case["act"],
                      dropout_p=case["p"], seed=s["key"], rows=s["rows"])
    return [h.detach(), *torch.autograd.grad(h, _leaves(s), s["dh"])]


# --- the same results from elementary operations in 32 bits -----------------------------------

LOW = 0xFFFFFFFF
PHILOX_M = (0xD2511F53, 0xCD9E8D57)
PHILOX_W = (0x9E3779B9, 0xBB67AE85)
PHILOX_ROUNDS = 7


def _keep(key, rows, M, D, p):
    """The mask [M,D]: word c % 4 of Philox4x32-7 at the counter (c // 4, row id,
    0) below the share of the 2^32 values that is kept."""
    dev = "cuda"
    rows = torch.arange(M, device=dev) if rows is None else rows
    groups = (D + 3) // 4
    c0 = torch.arange(groups, device=dev)[None, :].expand(M, groups)
    c1 = (rows & LOW)[:, None].expand(M, groups)
    c2 = ((rows >> 32) & LOW)[:, None].expand(M, groups)
    c3 = torch.zeros_like(c0)
    k0, k1 = key & LOW, (key >> 32) & LOW
    for _ in range(PHILOX_ROUNDS):
        # (64-bit integer products keep their low 64 bits)
        p0, p1 = c0 * PHILOX_M[0], c2 * PHILOX_M[1]
        c0, c1, c2, c3 = (((p1 >> 32) & LOW) ^ c1 ^ k0, p1 & LOW,
                          ((p0 >> 32) & LOW) ^ c3 ^ k1, p0 & LOW)
        k0, k1 = (k0 + PHILOX_W[0]) & LOW, (k1 + PHILOX_W[1]) & LOW
    words = torch.stack([c0, c1, c2, c3], 2).reshape(M, groups * 4)[:, :D]
    return words < round((1.0 - p) * 2.0 ** 32)


def _activation(g, act):
    """(act(g), act'(g)) in g's type."""
    if act == "relu":
        on = g > 0
        return torch.where(on, g, torch.zeros_like(g)), on.to(g.dtype)
    if act == "tanh":
        t = torch.tanh(g)
        return t, 1 - t * t
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))


def _quantize(x):
    x = x.float()
    scale = x.abs().amax(1) / 127.0
    q = torch.round(x / scale[:, None])
    return torch.where(scale[:, None] > 0, q, torch.zeros_like(q)), scale


def _run_plain(s):
    case = s["case"]
    path, dt = case["path"], DTYPES[case["dtype"]]
    x = s["x"].detach()
    M, D = x.shape
    if path == "quantize":
        q, scale = _quantize(x)
        return {"q": q.to(torch.int8), "scale": scale}
    if path == "dropout":
        keep, up = _keep(s["key"], s["rows"], M, D, case["p"]), 1.0 / (1.0 - case["p"])
        zero = torch.zeros((), device="cuda")
        return {"y": torch.where(keep, x.float() * up, zero).to(dt),
                "dx": torch.where(keep, s["dy"].float() * up, zero).to(dt)}
    if path == "int8":
        q, scale = _quantize(x)
        # (32 bits do not hold the sums of 8-bit products: 64)
        y = (q.double() @ s["wq"].double().t()).float() * scale[:, None] * s["ws"]
        return (y if s["b"] is None else y + s["b"].float()).to(dt)
    x32, wg, wu = x.float(), s["wg"].detach().float(), s["wu"].detach().float()
    g, u = x32 @ wg.t(), x32 @ wu.t()
    if case["bias"]:
        g, u = g + s["bg"].detach().float(), u + s["bu"].detach().float()
    a, da = _activation(g, case["act"])
    h, keep, up = a * u, None, 1.0 / (1.0 - case["p"])
    if case["p"] > 0:
        keep = _keep(s["key"], s["rows"], M, case["F"], case["p"])
        h = torch.where(keep, h * up, torch.zeros_like(h))
    if path == "act":
        return h.to(dt)
    dh = s["dh"].float()
    if keep is not None:
        dh = torch.where(keep, dh * up, torch.zeros_like(dh))
    du, dg = dh * a, dh * u * da
    grads = [dg @ wg + du @ wu, dg.t() @ x32, du.t() @ x32]
    if case["bias"]:
        grads += [dg.sum(0), du.sum(0)]
    return [h.to(dt)] + [t.to(dt) for t in grads]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --- 64 bits ----------------------------------------------------------------------------------

def _mul_high_low(a, m):
    """(high, low) 32 bits of the products a * m, by 16-bit halves of m."""
    lo, hi = a * (m & 0xFFFF), a * (m >> 16)
    carry = lo + ((hi & 0xFFFF) << 16)
    return (hi >> 16) + (carry >> 32), carry & LOW


def _mask64(key, rows, M, D, p):
    rows = torch.arange(M, device="cuda") if rows is None else rows
    shape = (M, (D + 3) // 4)
    zeros = torch.zeros(shape, dtype=torch.int64, device="cuda")
    x = [zeros + torch.arange(shape[1], device="cuda"), zeros + (rows % (1 << 32))[:, None],
         zeros + (rows // (1 << 32))[:, None], zeros]
    for r in range(PHILOX_ROUNDS):
        k0 = (key + r * PHILOX_W[0]) % (1 << 32)
        k1 = ((key >> 32) + r * PHILOX_W[1]) % (1 << 32)
        h0, l0 = _mul_high_low(x[0], PHILOX_M[0])
        h1, l1 = _mul_high_low(x[2], PHILOX_M[1])
        x = [h1 ^ x[1] ^ k0, l1, h0 ^ x[3] ^ k1, l0]
    return (torch.stack(x, -1).flatten(1)[:, :D] < round((1 - p) * 2 ** 32)).double()


def exact(case, seed):
    s = prepare(case, seed)
    path, M, D = case["path"], case["M"], case["D"]
    x = s["x"].detach().double()
    if path == "dropout":
        f = _mask64(s["key"], s["rows"], M, D, case["p"]) / (1 - case["p"])
        return {"y": x * f, "dx": s["dy"].double() * f}
    if path in ("quantize", "int8"):
        scale = (x.abs().max(1).values / 127).float().double()  # (the scale is a 32-bit value)
        if path == "quantize":
            return {"q": None, "scale": scale}
        q = (x / scale[:, None]).round()
        y = torch.matmul(q, s["wq"].double().T) * scale[:, None] * s["ws"].double()[None]
        return y if s["b"] is None else y + s["b"].double()
    act = {"relu": torch.relu, "tanh": torch.tanh, "silu": torch.nn.functional.silu,
           "gelu": torch.nn.functional.gelu}[case["act"]]
    leaves = [t.detach().double().requires_grad_(path == "train") for t in _leaves(s)]
    b = leaves[3:] or [None, None]
    h = (act(torch.nn.functional.linear(leaves[0], leaves[1], b[0]))
         * torch.nn.functional.linear(leaves[0], leaves[2], b[1]))
    if case["p"] > 0:
        h = h * (_mask64(s["key"], s["rows"], M, case["F"], case["p"]) / (1 - case["p"]))
    if path == "act":
        return h
    return [h.detach(), *torch.autograd.grad(h, leaves, s["dh"].double())]
