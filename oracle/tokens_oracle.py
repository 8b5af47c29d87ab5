"""64-bit restatement of the token-policy operators (test infrastructure only):
every function takes fp64 tensors with rows flattened to [R, A] and writes the
gradients out."""

import torch


def log_softmax(x, tau=1.0):
    z = x / tau
    z = z - z.max(-1, keepdim=True).values
    return z - z.exp().sum(-1, keepdim=True).log()


def entropy(ls):
    p = ls.exp()
    return -torch.where(p > 0, p * ls, torch.zeros_like(p)).sum(-1)


def log_probs(x, actions, tau=1.0):
    """(log p[a], H, log p) of [R, A] and [R]."""
    ls = log_softmax(x, tau)
    return ls.gather(1, actions[:, None])[:, 0], entropy(ls), ls


def log_probs_grad(ls, actions, g, ge, tau=1.0):
    """dlogits for the gradients g of log p[a] and ge of H."""
    p, H = ls.exp(), entropy(ls)
    plp = torch.where(p > 0, p * ls, torch.zeros_like(p))
    d = -p * g[:, None] - ge[:, None] * (plp + p * H[:, None])
    d.scatter_add_(1, actions[:, None], g[:, None])
    return d / tau


def weights(mask, reduction="token", denominator=None):
    """[S, T] weights of a mask [S, T]."""
    m = mask.double()
    if reduction == "token":
        n = float(m.sum()) if denominator is None else denominator
        return m / n if n else m
    n = m.sum(1, keepdim=True)
    some = float((n > 0).sum()) if denominator is None else denominator
    return m / n.clamp(min=1) / (some if some else 1.0)


def policy_terms(lp, H, old, adv, ref, low, high, kl_coef, entropy_coef):
    """Per row: (surrogate, kl, approx_kl, clipped, dloss/dlp, dloss/dH)."""
    ratio = torch.exp(lp - old)
    clip = ratio.clamp(1 - low, 1 + high)
    u, v = ratio * adv, clip * adv
    g = torch.where(u > v, torch.zeros_like(u), -u)
    kl = torch.zeros_like(lp)
    if ref is not None:
        d = ref - lp
        kl = torch.expm1(d) - d
        if kl_coef:
            g = g - kl_coef * torch.expm1(d)
    clipped = ((ratio < 1 - low) | (ratio > 1 + high)).double()
    return -torch.minimum(u, v), kl, old - lp, clipped, g, torch.full_like(lp, -entropy_coef)


def preference(relative, mask, beta, margin, smoothing, average):
    """(loss, rewards [S], dloss/dlp [S, T]) of relative [S, T]."""
    m = mask.double()
    n = m.sum(1)
    w = 1 / n.clamp(min=1) if average else torch.ones_like(n)
    rewards = beta * w * torch.where(mask, relative, torch.zeros_like(relative)).sum(1)
    P = len(rewards) // 2
    x = rewards[:P] - rewards[P:] - margin
    ls = torch.nn.functional.logsigmoid
    loss = (-(1 - smoothing) * ls(x) - smoothing * ls(-x)).mean()
    dx = (smoothing * torch.sigmoid(x) - (1 - smoothing) * torch.sigmoid(-x)) / P
    return loss, rewards, torch.cat([dx, -dx])[:, None] * beta * w[:, None] * m


def distill_rows(ls, teacher, ids, tau):
    """(row losses, dloss/dz [R, A], q) without the factor tau^2 w / tau; entries with
    ids < 0 are none, and so is a teacher's -inf."""
    live = (ids >= 0) & (teacher != -float("inf"))
    t = torch.where(live, teacher / tau, torch.full_like(teacher, -float("inf")))
    some = live.any(1, keepdim=True)
    lq = t - torch.where(some, torch.logsumexp(t, 1, keepdim=True), torch.zeros(len(t), 1).double())
    q = torch.where(live, lq.exp(), torch.zeros_like(lq))
    at = ids.clamp(min=0)
    terms = q * (lq - ls.gather(1, at))
    rows = torch.where(q > 0, terms, torch.zeros_like(q)).sum(1)
    d = ls.exp() * some.double()
    return rows, d.scatter_add(1, at, -q), q


def top(x, k):
    """(values, ids) of the k largest, ties by column, NaN first."""
    v, i = x.sort(dim=-1, descending=True, stable=True)
    return v[..., :k], i[..., :k]
