"""The token-policy operators as torch.ops.ppo_amd.* on the GPU: opcheck (schema,
fake tensor, autograd registration), the functions' results, and a compiled loss
with its backward pass.  (A file of its own, as test_gpu_torch_ops.py:
torch.compile switches off the argument validation of torch.distributions for the
process.)"""

import pytest
import torch

import ppo_amd

pytestmark = pytest.mark.gpu


def _case(dev, S=4, T=5, A=300, K=6):
    g = torch.Generator().manual_seed(S + T + A)
    x = (torch.randn(S, T, A, generator=g) * 2).to(dev).requires_grad_()
    a = torch.randint(0, A, (S, T), generator=g).to(dev)
    adv = torch.randn(S, T, generator=g).to(dev)
    mask = (torch.rand(S, T, generator=g) < 0.7).to(dev)
    teacher = torch.randn(S, T, K, generator=g).to(dev)
    ids = torch.randint(0, A, (S, T, K), generator=g).to(dev)
    old = ppo_amd.token_log_probs(x.detach(), a) + 0.1 * adv
    return x, a, old, adv, mask, teacher, ids


def test_registered_operators(dev):
    op = torch.ops.ppo_amd
    x, a, old, adv, mask, teacher, ids = _case(dev)
    utils = ("test_schema", "test_autograd_registration", "test_faketensor")
    policy = (x, a, old, adv, old, mask, 0.2, 0.3, 0.05, 0.01, 1.0, "sequence", None)
    preference = (x, a, old, mask, 0.1, 0.05, 0.0, False, 1.0)
    distill = (x, teacher, ids, mask, 2.0, "token", None)
    torch.library.opcheck(op.token_log_probs, (x, a, mask, 0.8), test_utils=utils)
    torch.library.opcheck(op.token_policy_loss, policy, test_utils=utils)
    torch.library.opcheck(op.preference_loss, preference, test_utils=utils)
    torch.library.opcheck(op.distillation_loss, distill, test_utils=utils)
    torch.library.opcheck(op.top_logits, (x.detach(), 7), test_utils=utils)

    lp, H, _ = op.token_log_probs(x, a, mask, 0.8)
    flp, fH = ppo_amd.token_log_probs(x, a, mask, 0.8, entropy=True)
    pairs = [((lp * adv + H).sum(), (flp * adv + fH).sum()),
             (op.token_policy_loss(*policy)[0][0],
              ppo_amd.token_policy_loss(x, a, old, adv, old, mask, 0.2, 0.3, 0.05, 0.01, 1.0,
                                        "sequence")[0]),
             (op.preference_loss(*preference)[0],
              ppo_amd.preference_loss(x, a, old, mask, 0.1, 0.05)[0])]
    for got, want in pairs:
        assert torch.equal(got, want)
        assert torch.equal(*(torch.autograd.grad(y * 3.0, [x])[0] for y in (got, want)))
    got, want = op.distillation_loss(*distill)[0], ppo_amd.distillation_loss(x, teacher, ids, mask,
                                                                           2.0)
    # (the function forms its gradient with the loss for a factor of 1: 3 forms it anew)
    assert torch.equal(got, want)
    assert torch.equal(*(torch.autograd.grad(y * 3.0, [x])[0] for y in (got, want)))
    assert all(torch.equal(p, q) for p, q in zip(op.top_logits(x.detach(), 7),
                                                 ppo_amd.top_logits(x.detach(), 7)))


def test_registered_backward_refuses(dev):
    op = torch.ops.ppo_amd
    x, a, old, adv, mask, teacher, ids = _case(dev)
    x = x.detach()
    _, _, saved = op.token_log_probs(x, a, mask, 1.0)
    one = torch.ones((), device=dev)

    def call(x=x, a=a, mask=mask, saved=saved, dlp=old, dH=None, scale=None):
        return op.token_log_probs_backward(x, a, mask, 1.0, saved, dlp, dH, scale)

    assert call(scale=one).shape == x.shape
    for kw in (dict(saved=saved[:3].contiguous()), dict(dlp=old[:2].contiguous()),
               dict(dH=old.t().contiguous()), dict(scale=old), dict(a=a[:3].contiguous()),
               dict(x=x.transpose(0, 1))):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(saved=saved.half()), dict(dlp=old.double()), dict(scale=one.double()),
               dict(a=a.float())):
        with pytest.raises(TypeError):
            call(**kw)
    f = op.distillation_loss_backward
    _, saved = op.distillation_loss(x, teacher, ids, mask, 1.0, "token", None)
    assert f(x, teacher, ids, mask, 1.0, saved, one).shape == x.shape
    with pytest.raises(ValueError):
        f(x, teacher, ids, mask, 1.0, saved[:2].contiguous(), one)
    with pytest.raises(ValueError):
        f(x, teacher[..., :3].contiguous(), ids, mask, 1.0, saved, one)


def test_registered_operators_compile(dev):
    """A compiled step of the losses with its backward is traced whole and equals eager."""
    op = torch.ops.ppo_amd
    x, a, old, adv, mask, teacher, ids = _case(dev)

    def step(x):
        y = x * 1.5
        lp = op.token_log_probs(y, a, mask, 1.0)[0]
        policy = op.token_policy_loss(y, a, old, adv, None, mask, 0.2, 0.2, 0.0, 0.01, 1.0, "token",
                                      None)[0][0]
        pref = op.preference_loss(y, a, old, mask, 0.1, 0.0, 0.0, True, 1.0)[0]
        values, where = op.top_logits(teacher, 3)
        distill = op.distillation_loss(y, values, where, mask, 1.0, "sequence", 7.0)[0]
        return policy + pref + distill + lp.sum()

    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    runs = []
    for f in (step, compiled):
        y = f(x)
        runs.append([y.detach(), *torch.autograd.grad(y, [x])])
    assert all(torch.equal(p, q) for p, q in zip(*runs))


def test_registered_constants_that_ask_for_a_gradient(dev):
    op = torch.ops.ppo_amd
    x, a, old, adv, mask, teacher, ids = _case(dev)
    calls = [("old_log_probs", old, lambda v: op.token_policy_loss(
                  x, a, v, adv, old, mask, 0.2, 0.3, 0.05, 0.01, 1.0, "token", None)),
             ("advantages", adv, lambda v: op.token_policy_loss(
                 x, a, old, v, old, mask, 0.2, 0.3, 0.05, 0.01, 1.0, "token", None)),
             ("ref_log_probs", old, lambda v: op.token_policy_loss(
                 x, a, old, adv, v, mask, 0.2, 0.3, 0.05, 0.01, 1.0, "token", None)),
             ("ref_log_probs", old, lambda v: op.preference_loss(
                 x, a, v, mask, 0.1, 0.05, 0.0, False, 1.0)),
             ("teacher_logits", teacher, lambda v: op.distillation_loss(
                 x, v, ids, mask, 2.0, "token", None))]
    for name, v, call in calls:
        wants = v.clone().requires_grad_()
        for f in (call, torch.compile(call, fullgraph=True, backend="aot_eager")):
            with pytest.raises(RuntimeError, match=f"no gradient in {name}"):
                f(wants)
        with torch.no_grad():
            quiet = call(wants)[0]
        assert torch.equal(quiet, call(v)[0])
