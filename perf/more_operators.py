"""Token policies, as measurable cases: policies that pick one of up to a
vocabulary of actions at every step of a sequence, trained from their logits.

Every case is one pass through a public operator of ppo_amd: the taken actions'
log-probabilities and the entropies, when acting and in training
(token_log_probs), the clipped policy loss with a KL term
(token_policy_loss), the loss of preferred over rejected sequences
(preference_loss), the distillation of a teacher's top logits
(distillation_loss), each with its gradient, and the top logits themselves
(top_logits).  Where `own` is false the same results come from elementary torch
operations in 32 bits; exact() restates them in 64 bits.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # acting over the actions of a small environment: a minibatch of 256, where
        # only launches and latency count
        dict(name="logp_256x18_fp32", path="logp", S=256, T=1, A=18, dtype="fp32", tau=1.0,
             mask=False, train=False),
        # one new token of one sequence: its log-probability and entropy
        dict(name="logp_1x131072_bf16", path="logp", S=1, T=1, A=131072, dtype="bf16", tau=1.0,
             mask=False, train=False),
        # log-probabilities and entropies with their gradients, a row no vector divides
        dict(name="logp_train_2x1000x50257_fp16", path="logp", S=2, T=1000, A=50257,
             dtype="fp16", tau=0.8, mask=True, train=True),
        # a minibatch of short episodes over a few hundred actions
        dict(name="policy_16x33x500_fp32", path="policy", S=16, T=33, A=500, dtype="fp32",
             tau=1.0, mask=True, reduction="sequence", entropy=0.01, kl=0.05, per_token=True),
        # sequences of an ordinary vocabulary, one advantage each
        dict(name="policy_8x512x32768_bf16", path="policy", S=8, T=512, A=32768, dtype="bf16",
             tau=1.0, mask=True, reduction="token", entropy=0.0, kl=0.05, per_token=False),
        # a large batch over a large vocabulary, with the entropy's gradient
        dict(name="policy_8x1024x131072_bf16", path="policy", S=8, T=1024, A=131072,
             dtype="bf16", tau=1.0, mask=False, reduction="token", entropy=0.001, kl=0.0,
             per_token=True),
        # a few pairs of short sequences
        dict(name="pref_8x31x1000_fp32", path="pref", S=8, T=31, A=1000, dtype="fp32", tau=1.0,
             mask=True, average=False),
        # a training step's pairs over an ordinary vocabulary
        dict(name="pref_16x256x50304_bf16", path="pref", S=16, T=256, A=50304, dtype="bf16",
             tau=1.0, mask=True, average=False),
        # a few tokens over a very large vocabulary
        dict(name="distill_1x24x262144_bf16", path="distill", S=1, T=24, A=262144, dtype="bf16",
             tau=1.0, mask=False, K=20),
        # a student's batch, the teacher's 64 top logits
        dict(name="distill_4x1024x65536_bf16", path="distill", S=4, T=1024, A=65536,
             dtype="bf16", tau=2.0, mask=True, K=64),
        # the top logits of one new token
        dict(name="top_1x131072_bf16", path="top", S=1, T=1, A=131072, dtype="bf16", K=50),
        # a teacher's pass over a batch
        dict(name="top_4x1024x32001_fp32", path="top", S=4, T=1024, A=32001, dtype="fp32", K=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["logp", "logp", "policy", "policy", "pref", "distill", "distill", "top"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    A = _log_int(rng, 16, 262144)
    if A >= 256 and rng.random() < 0.5:  # vocabularies are mostly padded to such sizes
        A = A // 128 * 128
    rows = _log_int(rng, 2, max(2, min(16384, (1 << (27 if path == "top" else 29)) // A)))
    T = _log_int(rng, 1, rows)
    S = max(1, rows // T)
    if path == "pref":
        T, S = (T, S) if S > 1 else (max(1, T // 2), 2)
        S -= S % 2
    flag = lambda: rng.random() < 0.5  # noqa: E731
    case = dict(path=path, S=S, T=T, A=A, dtype=dtype)
    if path in ("distill", "top"):
        case["K"] = _log_int(rng, 1, min(128, A))
    if path == "top":
        return case
    case.update(tau=rng.choice([1.0, 1.0, 0.7, 1.5]), mask=flag())
    if path == "logp":
        case.update(train=flag())
    if path == "policy":
        case.update(reduction=rng.choice(["token", "sequence"]), per_token=flag(),
                    entropy=rng.choice([0.0, 0.01]), kl=rng.choice([0.0, 0.05]))
    if path == "pref":
        case.update(average=flag())
    return case


def _lengths(S, T):
    """Tokens that count in each of S sequences of T: from none (where there are
    many sequences) to all."""
    return [0 if i == 0 and S >= 8 else max(1, round(T * (0.3 + 0.7 * (i + 1) / S)))
            for i in range(S)]


def work(case):
    S, T, A, path, size = case["S"], case["T"], case["A"], case["path"], \
        DTYPES[case["dtype"]].itemsize
    R = S * T
    if path == "top":
        return {"bytes": R * A * size + R * case["K"] * (size + 8), "flops": R * A}
    n = sum(_lengths(S, T)) if case["mask"] else R
    rows = (n * A + (0 if path == "logp" and not case["train"] else R * A)) * size
    mask = R if case["mask"] else 0
    if path == "logp":  # actions in, log-probabilities and entropies out; their gradients in
        side = 8 * n + 8 * R + (8 * n if case["train"] else 0)
    elif path == "policy":
        side = n * (8 + 4 + (4 if case["per_token"] else 0) + (4 if case["kl"] else 0))
    elif path == "pref":
        side = n * (8 + 4)
    else:
        side = n * case["K"] * (size + 8)
    return {"bytes": rows + side + mask, "flops": 4 * rows // size}


# --- inputs, from the seed alone ------------------------------------------------------

BLOCK = 1 << 27  # elements that prepare() and exact() hold in wide types at a time


def _blocks(R, A):
    step = max(1, BLOCK // A)
    return [(r, min(R, r + step)) for r in range(0, R, step)]


def _logits(g, R, A, dtype):
    """Rows from nearly uniform to nearly decided ones."""
    x = torch.empty(R, A, dtype=dtype, device="cuda")
    for r, e in _blocks(R, A):
        width = 1.0 + 4.0 * torch.rand(e - r, 1, generator=g, device="cuda")
        x[r:e] = torch.randn(e - r, A, generator=g, device="cuda") * width
    return x


def _sampled(g, x, tau):
    """(actions drawn from softmax(x / tau), their log-probabilities fp32)."""
    R, A = x.shape
    actions = torch.empty(R, dtype=torch.int64, device="cuda")
    logp = torch.empty(R, dtype=torch.float32, device="cuda")
    for r, e in _blocks(R, A):
        z = x[r:e].float() / tau
        noise = torch.empty_like(z).exponential_(generator=g).clamp_(min=1e-30).log_()
        actions[r:e] = (z - noise).argmax(1)
        logp[r:e] = z.gather(1, actions[r:e, None])[:, 0] - torch.logsumexp(z, 1)
    return actions, logp


def _mask(g, S, T):
    """bool [S,T]: a run of tokens of each sequence, the lengths in random order."""
    n = torch.tensor(_lengths(S, T), device="cuda")
    n = n[torch.randperm(S, generator=g, device="cuda")]
    first = (torch.rand(S, generator=g, device="cuda") * (T - n + 1)).long().clamp_(max=T)
    t = torch.arange(T, device="cuda")[None]
    return (t >= first[:, None]) & (t < (first + n)[:, None])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * seed + 31)
    S, T, A, path, dt = case["S"], case["T"], case["A"], case["path"], DTYPES[case["dtype"]]
    x = _logits(g, S * T, A, dt)
    s = dict(case=case, logits=x.view(S, T, A))
    if path == "top":
        return s
    rn = lambda *n: torch.randn(*n, generator=g, device="cuda")  # noqa: E731
    s["mask"] = _mask(g, S, T) if case["mask"] else None
    if path == "distill":
        K = case["K"]
        # distinct ids in no order, logits falling
        start = torch.randint(0, A, (S * T, 1), generator=g, device="cuda")
        step = torch.randint(1, A // K + 1, (S * T, 1), generator=g, device="cuda")
        ids = (start + step * torch.arange(K, device="cuda")) % A
        s["ids"] = ids.view(S, T, K)
        s["teacher"] = (rn(S, T, K) * 3.0 + 8.0).sort(-1, descending=True).values.to(dt)
    else:
        actions, logp = _sampled(g, x, case["tau"])
        s["actions"] = actions.view(S, T)
    if path == "logp" and case["train"]:
        s["dlogp"], s["dent"] = rn(S, T), rn(S, T) * 0.1
    if path == "policy":
        # the ratio moves by some percent from the rollout's policy, and lies off the
        # clip's two borders, where its gradient jumps
        move = (rn(S * T) * 0.15).clamp_(-1.0, 1.0)
        for border in (math.log1p(-CLIP[0]), math.log1p(CLIP[1])):
            move = torch.where((move - border).abs() < 1e-3, move + 4e-3, move)
        s["old"] = (logp - move).view(S, T)
        s["adv"] = rn(S, T) if case["per_token"] else rn(S)
        s["ref"] = (logp + 0.3 * rn(S * T)).view(S, T) if case["kl"] else None
    if path == "pref":
        # a policy that has moved off its reference, some sequences up, some down
        s["ref"] = logp.view(S, T) + 0.3 * rn(S, T) + 0.05 * rn(S, 1)
    if path != "logp" or case["train"]:
        s["logits"].requires_grad_()
    return s


CLIP = (0.2, 0.28)
BETA, SMOOTHING = 0.1, 0.05


# --- the framework's operators ------------------------------------------------------------

def _package():
    if "ppo_amd" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(
            os.path.abspath(__file__))), "zero-to-hero_amd"))
    import ppo_amd

    return ppo_amd


def _run_own(s):
    amd, case = _package(), s["case"]
    path, x = case["path"], s["logits"]
    if path == "top":
        values, ids = amd.top_logits(x, case["K"])
        return {"values": values, "ids": ids}
    kw = dict(mask=s["mask"], temperature=case["tau"])
    if path == "logp":
        logp, entropy = amd.token_log_probs(x, s["actions"], entropy=True, **kw)
        if not case["train"]:
            return {"logp": logp, "entropy": entropy}
        (dx,) = torch.autograd.grad([logp, entropy], [x], [s["dlogp"], s["dent"]])
        return {"logp": logp.detach(), "entropy": entropy.detach(), "dlogits": dx}
    if path == "policy":
        loss, stats = amd.token_policy_loss(
            x, s["actions"], s["old"], s["adv"], s["ref"], clip_low=CLIP[0], clip_high=CLIP[1],
            kl_coef=case["kl"], entropy_coef=case["entropy"], reduction=case["reduction"], **kw)
        (dx,) = torch.autograd.grad(loss, [x])
        return {"loss": loss.detach(), "policy": stats["policy"], "kl": stats["kl"],
                "entropy": stats["entropy"], "clipfrac": stats["clipfrac"], "dlogits": dx}
    if path == "pref":
        loss, stats = amd.preference_loss(x, s["actions"], s["ref"], beta=BETA,
                                          label_smoothing=SMOOTHING, average=case["average"],
                                          **kw)
        (dx,) = torch.autograd.grad(loss, [x])
        return {"loss": loss.detach(), "chosen": stats["chosen"], "rejected": stats["rejected"],
                "dlogits": dx}
    loss = amd.distillation_loss(x, s["teacher"], s["ids"], **kw)
    (dx,) = torch.autograd.grad(loss, [x])
    return {"loss": loss.detach(), "dlogits": dx}


# --- the same results from elementary operations in 32 bits -----------------------------------

def _log_softmax(x, tau, wide=False):
    """log softmax(x / tau) in 32 bits; `wide`: the sum and the result in 64, for
    sums of small differences of log-probabilities."""
    z = x.detach().float() / tau
    z = z - z.amax(-1, keepdim=True)
    if wide:
        return z.double() - torch.exp(z).sum(-1, keepdim=True, dtype=torch.float64).log()
    return z - torch.exp(z).sum(-1, keepdim=True).log()


def _weights(s):
    """fp32 [S,T]: each token's weight in the mean."""
    case, mask = s["case"], s["mask"]
    live = torch.ones(case["S"], case["T"], device="cuda") if mask is None else mask.float()
    if case.get("reduction", "token") == "token":
        return live / live.sum().clamp(min=1.0)
    n = live.sum(1, keepdim=True)
    return live / n.clamp(min=1.0) / (n > 0).sum().clamp(min=1)


def _run_plain(s):
    case, x = s["case"], s["logits"]
    path, dt = case["path"], DTYPES[case["dtype"]]
    if path == "top":
        values, ids = x.float().sort(dim=-1, descending=True, stable=True)
        K = case["K"]
        return {"values": values[..., :K].to(dt), "ids": ids[..., :K].clone()}
    tau, zero = case["tau"], torch.zeros((), device="cuda")
    ls = _log_softmax(x, tau, wide=path == "pref")
    p = torch.exp(ls.float())
    live = torch.ones((), dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    if path == "distill":
        w = _weights(s)
        ids = s["ids"]
        t = s["teacher"].float() / tau
        t = t - t.amax(-1, keepdim=True)
        lq = t - torch.exp(t).sum(-1, keepdim=True).log()
        q = torch.exp(lq)
        rows = (q * (lq - ls.gather(-1, ids))).sum(-1)
        d = p.scatter_add(-1, ids, -q) * (w * tau)[..., None]
        return {"loss": tau * tau * (w * rows).sum(), "dlogits": d.to(dt)}
    a = s["actions"][..., None]
    logp = torch.where(live, ls.gather(-1, a)[..., 0], zero)
    if path == "pref":
        n = live.float().expand(case["S"], case["T"]).sum(1)
        scale = 1.0 / n.clamp(min=1.0) if case["average"] else torch.ones_like(n)
        rel = (torch.where(live, logp - s["ref"], zero).sum(1) * scale * BETA).float()
        half = case["S"] // 2
        m = rel[:half] - rel[half:]
        # -log sigmoid(m) = max(-m, 0) + log(1 + e^-|m|)
        soft = torch.log1p(torch.exp(-m.abs()))
        loss = ((1 - SMOOTHING) * ((-m).clamp(min=0.0) + soft)
                + SMOOTHING * (m.clamp(min=0.0) + soft)).mean()
        dm = (1.0 / (1.0 + torch.exp(-m)) - (1 - SMOOTHING)) / half
        g = torch.cat([dm, -dm]) * scale * BETA
        g = torch.where(live, g[:, None].expand(case["S"], case["T"]), zero)
        d = (-p).scatter_add(-1, a, torch.ones_like(a, dtype=torch.float32)) * (g / tau)[..., None]
        return {"loss": loss, "chosen": rel[:half], "rejected": rel[half:], "dlogits": d.to(dt)}
    H = -(p * ls).sum(-1)
    entropy = torch.where(live, H, zero)
    if path == "logp":
        out = {"logp": logp, "entropy": entropy}
        if not case["train"]:
            return out
        g, ge = torch.where(live, s["dlogp"], zero), torch.where(live, s["dent"], zero)
    else:
        w = _weights(s)
        adv = s["adv"] if case["per_token"] else s["adv"][:, None].expand(case["S"], case["T"])
        ratio = torch.exp(torch.where(live, logp - s["old"], zero))
        clipped = ratio.clamp(1 - CLIP[0], 1 + CLIP[1])
        outside = (ratio * adv) > (clipped * adv)
        surrogate = -torch.minimum(ratio * adv, clipped * adv)
        g = w * torch.where(outside, zero, -ratio * adv)
        kl = zero
        if case["kl"]:
            r = torch.where(live, s["ref"] - logp, zero)
            kl = (w * (torch.expm1(r) - r)).sum()
            g = g - case["kl"] * w * torch.expm1(r)
        ge = -case["entropy"] * w
        policy, mean_entropy = (w * surrogate).sum(), (w * entropy).sum()
        out = {"loss": policy + case["kl"] * kl - case["entropy"] * mean_entropy,
               "policy": policy, "kl": kl, "entropy": mean_entropy,
               "clipfrac": (w * ((ratio < 1 - CLIP[0]) | (ratio > 1 + CLIP[1])).float()).sum()}
    # d logp / dz_j = [j = a] - p_j,  d H / dz_j = -p_j (log p_j + H)
    d = p * (-g[..., None] - ge[..., None] * (ls + H[..., None]))
    out["dlogits"] = (d.scatter_add(-1, a, g[..., None]) / tau).to(dt)
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --- 64 bits ----------------------------------------------------------------------------------

def _exact_top(x, K):
    """Each logit and its place in one 64-bit whole number, by which no two are alike."""
    bits = (x + 0.0).float().view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = order * (1 << 20) - torch.arange(x.shape[-1], device="cuda")
    ids = torch.topk(key, K, -1).indices
    return {"values": x.double().gather(-1, ids), "ids": ids}


def exact(case, seed):
    s = prepare(case, seed)
    S, T, A, path = case["S"], case["T"], case["A"], case["path"]
    x = s["logits"].detach().view(S * T, A)
    if path == "top":
        parts = [_exact_top(x[r:e], case["K"]) for r, e in _blocks(S * T, A)]
        return {k: torch.cat([p[k] for p in parts]).view(S, T, -1) for k in ("values", "ids")}
    tau, R = case["tau"], S * T
    mask = torch.ones(S, T, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    live = mask.view(R).double()
    if case.get("reduction") == "sequence":
        n = mask.sum(1).double()
        w = (mask / n.clamp(min=1)[:, None] / int((n > 0).sum())).view(R)
    else:
        w = live / live.sum().clamp(min=1)
    flat = {k: v.detach().double().reshape(R) for k, v in s.items()
            if k in ("old", "ref", "dlogp", "dent") and v is not None}
    if path == "policy":
        adv = s["adv"].double()
        flat["adv"] = adv.reshape(R) if case["per_token"] else adv.repeat_interleave(T)
    grads, logps, ents, sums = [], [], [], {}
    coef = None
    if path == "pref":  # the pairs' margins come first: they are every row's coefficient
        rel = torch.cat([torch.log_softmax(x[r:e].double() / tau, 1).gather(
            1, s["actions"].view(R, 1)[r:e])[:, 0] for r, e in _blocks(R, A)]) - flat["ref"]
        lens = mask.sum(1).double().clamp(min=1) if case["average"] else torch.ones(
            S, dtype=torch.float64, device="cuda")
        rel = ((torch.where(mask, rel.view(S, T), 0.0).sum(1)) / lens * BETA).requires_grad_()
        m = rel[:S // 2] - rel[S // 2:]
        loss = -((1 - SMOOTHING) * torch.nn.functional.logsigmoid(m)
                 + SMOOTHING * torch.nn.functional.logsigmoid(-m)).mean()
        (drel,) = torch.autograd.grad(loss, [rel])
        coef = ((drel * BETA / lens)[:, None] * mask).view(R)
    for r, e in _blocks(R, A):
        z = x[r:e].double().requires_grad_(path != "logp" or case["train"])
        dist = torch.log_softmax(z / tau, 1)
        if path == "distill":
            lq = torch.log_softmax(s["teacher"].view(R, -1)[r:e].double() / tau, 1)
            rows = (lq.exp() * (lq - dist.gather(1, s["ids"].view(R, -1)[r:e]))).sum(1)
            total = tau * tau * (w[r:e] * rows).sum()
            sums["loss"] = sums.get("loss", 0.0) + total.detach()
        else:
            lp = dist.gather(1, s["actions"].view(R, 1)[r:e])[:, 0]
            lv = live[r:e]
            if path == "pref":
                total = (coef[r:e] * lp).sum()
            else:
                H = -(dist.exp() * dist).sum(1)
                if path == "logp":
                    logps.append((lp * lv).detach())
                    ents.append((H * lv).detach())
                    if not case["train"]:
                        continue
                    total = ((flat["dlogp"][r:e] * lp + flat["dent"][r:e] * H) * lv).sum()
                else:
                    ratio = torch.exp(lp - flat["old"][r:e])
                    ad, wr = flat["adv"][r:e], w[r:e]
                    low, high = 1 - CLIP[0], 1 + CLIP[1]
                    parts = {"policy": -torch.minimum(ratio * ad, ratio.clamp(low, high) * ad),
                             "entropy": H, "clipfrac": ((ratio < low) | (ratio > high)).double(),
                             "kl": torch.zeros_like(H)}
                    if case["kl"]:
                        diff = flat["ref"][r:e] - lp
                        parts["kl"] = torch.exp(diff) - diff - 1
                    parts = {k: (wr * torch.where(wr > 0, v, 0.0)).sum()
                             for k, v in parts.items()}
                    total = parts["loss"] = (parts["policy"] + case["kl"] * parts["kl"]
                                             - case["entropy"] * parts["entropy"])
                    for k, v in parts.items():
                        sums[k] = sums.get(k, 0.0) + v.detach()
        grads.append(torch.autograd.grad(total, [z])[0])
    out = {k: v for k, v in sums.items()}
    if path == "logp":
        out.update(logp=torch.cat(logps).view(S, T), entropy=torch.cat(ents).view(S, T))
    if path == "pref":
        out.update(loss=loss.detach(), chosen=rel[:S // 2].detach(), rejected=rel[S // 2:].detach())
    if grads:
        out["dlogits"] = torch.cat(grads).view(S, T, A)
    return out
