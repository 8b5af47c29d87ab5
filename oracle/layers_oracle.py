"""64-bit restatement of the feed-forward layer operators (test infrastructure
only): Philox4x32 and the dropout mask, 8-bit rows, the 8-bit product, and the
gated feed-forward block with its gradients written out."""

import math

import numpy as np
import torch

M0, M1 = np.uint64(0xD2511F53), np.uint64(0xCD9E8D57)
W0, W1 = 0x9E3779B9, 0xBB67AE85
LOW = np.uint64(0xFFFFFFFF)


def philox4x32(counter, key, rounds=7):
    """Salmon et al., SC 2011: counter four arrays of 32-bit values in uint64,
    key two ints; returns four such arrays."""
    x = [np.asarray(c, dtype=np.uint64) for c in counter]
    k0, k1 = key
    for _ in range(rounds):
        p0, p1 = x[0] * M0, x[2] * M1
        x = [(p1 >> np.uint64(32)) ^ x[1] ^ np.uint64(k0), p1 & LOW,
             (p0 >> np.uint64(32)) ^ x[3] ^ np.uint64(k1), p0 & LOW]
        k0, k1 = (k0 + W0) & 0xFFFFFFFF, (k1 + W1) & 0xFFFFFFFF
    return x


def keep_mask(p, seed, rows, cols):
    """bool [len(rows), cols]: which elements dropout keeps."""
    rows = np.asarray(rows, dtype=np.int64).astype(np.uint64)
    groups = (cols + 3) // 4
    c0 = np.broadcast_to(np.arange(groups, dtype=np.uint64), (len(rows), groups))
    r = np.broadcast_to(rows[:, None], c0.shape)
    words = philox4x32((c0, r & LOW, r >> np.uint64(32), np.zeros_like(c0)),
                       (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    words = np.stack(words, -1).reshape(len(rows), groups * 4)[:, :cols]
    return words < np.uint64(round((1.0 - p) * 2.0 ** 32))


def dropout(x, p, seed, rows=None):
    """fp64 [M,C] tensor x -> fp64."""
    M, C = x.shape
    keep = torch.from_numpy(keep_mask(p, seed, np.arange(M) if rows is None else rows, C))
    return torch.where(keep, x / (1.0 - p) if p < 1.0 else x, torch.zeros_like(x))


def quantize_rows(x):
    """fp32-valued x [M,K] -> (q int8, scale fp32), in 32-bit IEEE arithmetic."""
    x = np.asarray(x, dtype=np.float32)
    top = np.abs(x).max(1)
    scale = np.where(np.isfinite(top), top * (np.float32(1) / np.float32(127)),
                     np.float32(np.nan)).astype(np.float32)
    live = scale > 0
    with np.errstate(all="ignore"):
        q = np.clip(np.rint(x / scale[:, None]), -127, 127)
    return np.where(live[:, None], q, 0).astype(np.int8), scale


def int8_linear(xq, xs, wq, ws, bias=None):
    """fp64 result of the 8-bit product (numpy arrays)."""
    y = (xq.astype(np.int64) @ wq.astype(np.int64).T).astype(np.float64)
    y = y * xs.astype(np.float64)[:, None] * ws.astype(np.float64)[None]
    return y if bias is None else y + bias[None]


def activation(g, act):
    """(act(g), act'(g)) of an fp64 tensor."""
    if act == "relu":
        return g.clamp(min=0), (g > 0).double()
    if act == "tanh":
        t = torch.tanh(g)
        return t, 1 - t * t
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * torch.erfc(-g * math.sqrt(0.5))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def gated_ffn(x, wg, wu, bg, bu, act, keep=None, p=0.0):
    """fp64 forward; `keep` the dropout mask or None.  Returns (h, g, u)."""
    g, u = x @ wg.T, x @ wu.T
    if bg is not None:
        g, u = g + bg, u + bu
    h = activation(g, act)[0] * u
    if keep is not None:
        h = torch.where(keep, h / (1 - p) if p < 1 else h, torch.zeros_like(h))
    return h, g, u


def gated_ffn_grads(x, wg, wu, g, u, act, dh, keep=None, p=0.0):
    """fp64 dx, dwg, dwu, dbg, dbu."""
    if keep is not None:
        dh = torch.where(keep, dh / (1 - p) if p < 1 else dh, torch.zeros_like(dh))
    a, da = activation(g, act)
    dg, du = dh * u * da, dh * a
    return dg @ wg + du @ wu, dg.T @ x, du.T @ x, dg.sum(0), du.sum(0)
