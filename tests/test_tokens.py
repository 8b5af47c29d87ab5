"""The token-policy operators without a GPU: the C ABI of include/ppo_tokens.h, its
argument checks (which return before any device work), the Python refusals, and
the oracle they are tested against."""

import ctypes
import os
import re

import pytest
import torch

import ppo_amd
from oracle import tokens_oracle as ref
from ppo_amd import _lib, tokens

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "ppo_tokens.h")
P = ctypes.c_void_p(4096)  # non-null, aligned, never dereferenced
ODD = ctypes.c_void_p(4097)


def declared_functions():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return sorted(set(re.findall(r"\b(ppo_token_[a-z0-9_]+)\s*\(", text)))


def test_exports_match_the_header():
    lib = _lib.load_tokens()
    names = declared_functions()
    assert names and set(names) == set(_lib.TOKEN_SIGNATURES)
    for name in names:
        assert hasattr(lib, name)
    syms = os.popen(f"nm -D --defined-only {_lib.TOKENS_PATH}").read()
    assert set(re.findall(r"\bT (\S+)$", syms, flags=re.M)) == set(names)


def rows(logits=P, actions=P, mask=None, S=4, T=5, A=30, dtype=0, tau=1.0):
    return ctypes.byref(_lib.TokenRows(logits, actions, mask, S, T, A, dtype, 1, tau))


def loss(low=0.2, high=0.2, kl=0.0, ent=0.0, den=0.0, scale=1.0, red=0, per=0):
    return ctypes.byref(_lib.TokenLoss(low, high, kl, ent, den, scale, red, per))


BAD_ROWS = [(dict(S=-1), 1), (dict(T=-1), 1), (dict(A=0), 1), (dict(dtype=3), 1), (dict(tau=0.0), 1),
            (dict(tau=-1.0), 1), (dict(tau=float("nan")), 1), (dict(tau=float("inf")), 1),
            (dict(logits=None), 1), (dict(logits=ctypes.c_void_p(4098)), 1),
            (dict(logits=ODD, dtype=1), 1), (dict(A=(1 << 30) + 1), 3),
            (dict(S=1 << 20, T=1 << 11), 3), (dict(S=1 << 31, T=1), 3),
            (dict(S=1 << 20, T=1 << 10, A=1 << 20), 3)]


@pytest.mark.parametrize("kw, code", BAD_ROWS)
def test_rows_are_checked_by_every_call(kw, code):
    lib = _lib.load_tokens()
    big = 1 << 40
    assert lib.ppo_token_log_probs(rows(**kw), None, P, None, None, P, big, None) == code
    assert lib.ppo_token_log_probs_backward(rows(**kw), P, P, None, None, 0.0, P, None) == code
    assert lib.ppo_token_policy_loss(rows(**kw), P, P, None, loss(), P, P, P, P, P, big,
                                     None) == code
    assert lib.ppo_token_distillation(rows(**kw), P, 0, P, 1, 3, loss(), P, P, P, P, big,
                                      None) == code
    assert lib.ppo_token_distillation_backward(rows(**kw), P, 0, P, 1, 3, P, P, 0.0, P, None) == code


def test_launches_that_do_not_fit():
    """Calls of 2^32 lanes are refused before anything is enqueued."""
    lib = _lib.load_tokens()
    f, top, big = lib.ppo_token_log_probs, lib.ppo_token_top, 1 << 44
    for S, A, dtype in ((1 << 28, 18, 0), (1 << 26, 600, 1), (1 << 24, 4096, 0), (1 << 24, 16384, 2)):
        for entropy in (None, P):
            assert f(rows(S=S, T=1, A=A, dtype=dtype), None, P, entropy, None, P, big, None) == 3
        assert top(P, dtype, S, A, 3, P, P, None, 0, None) == 3
    # (gradients that lie otherwise in 16 bytes than the logits take a workgroup a row)
    assert lib.ppo_token_policy_loss(rows(S=1 << 24, T=1, A=18), P, P, None, loss(), P, P, P,
                                     ctypes.c_void_p(4100), P, big, None) == 3
    assert lib.ppo_token_distillation(rows(S=1 << 24, T=1, A=18), P, 0, P, 1, 3, loss(), P, P,
                                      ctypes.c_void_p(4100), P, big, None) == 3


def test_top_launches_that_do_not_fit():
    """The limit counts the lanes that a row takes."""
    lib = _lib.load_tokens()
    for R, A, K in ((1 << 26, 18, 3), (1 << 24, 3000, 60), (1 << 23, 3000, 100),
                    (1 << 22, 3000, 200), (1 << 24, 20000, 3)):
        assert lib.ppo_token_top(P, 1, R, A, K, P, P, None, 0, None) == 3


def test_log_probs_arguments():
    lib = _lib.load_tokens()
    f = lib.ppo_token_log_probs
    need = lib.ppo_token_workspace_bytes(4, 5, 30, 0)
    assert need > 0 and lib.ppo_token_workspace_bytes(0, 5, 30, 0) == 0
    assert lib.ppo_token_workspace_bytes(4, 5, 0, 0) == 0
    assert lib.ppo_token_workspace_bytes(4, 5, 30, 7) == 0
    assert f(rows(), None, None, None, None, P, need, None) == 1
    assert f(rows(actions=None), None, P, None, None, P, need, None) == 1
    assert f(rows(), None, P, None, ctypes.c_void_p(4104), P, need, None) == 1
    assert f(rows(), None, P, None, None, P, need - 1, None) == 2
    assert f(rows(), None, P, None, None, None, need, None) == 2
    assert f(rows(), None, P, None, None, ODD, need, None) == 2
    assert f(rows(S=0, logits=None, actions=None), None, None, None, None, None, 0, None) == 0
    b = lib.ppo_token_log_probs_backward
    assert b(rows(), None, P, None, None, 0.0, P, None) == 1
    assert b(rows(), P, None, None, None, 0.0, P, None) == 1
    assert b(rows(), P, P, None, None, 0.0, None, None) == 1
    assert b(rows(), P, P, None, None, 1.0, P, None) == 1        # held needs a scale
    assert b(rows(dtype=1), P, P, None, None, 0.0, ODD, None) == 1
    assert b(rows(T=0, logits=None), None, None, None, None, 0.0, None, None) == 0


def test_policy_arguments():
    f = _lib.load_tokens().ppo_token_policy_loss

    def call(r=None, old=P, adv=P, ref=None, l=None, scalars=P, saved=P, coef=P, d=P, work=P,
             nbytes=1 << 40):
        return f(r or rows(), old, adv, ref, l or loss(), scalars, saved, coef, d, work, nbytes,
                 None)

    assert call(old=None) == 1 and call(adv=None) == 1 and call(scalars=None) == 1
    assert call(saved=None) == 1 and call(coef=None) == 1
    assert call(saved=None, coef=None) == 1                      # a gradient needs them
    assert call(saved=ctypes.c_void_p(4104)) == 1 and call(r=rows(dtype=2), d=ODD) == 1
    assert call(l=loss(kl=0.1)) == 1                             # no reference
    for bad in (dict(low=-0.1), dict(high=float("nan")), dict(kl=float("inf")),
                dict(ent=float("nan")), dict(den=-1.0), dict(den=float("nan")), dict(scale=0.0),
                dict(scale=float("inf")), dict(red=2), dict(red=-1)):
        assert call(l=loss(**bad)) == 1
    assert call(work=None) == 2 and call(work=ODD) == 2 and call(nbytes=100) == 2


UNHELD = [dict(den=1e46), dict(den=1e31), dict(den=1e-46), dict(den=1e-31), dict(scale=1e39),
          dict(scale=1e31), dict(scale=1e-50), dict(scale=1e-31), dict(kl=1e39), dict(ent=-1e39)]


@pytest.mark.parametrize("kw", UNHELD)
@pytest.mark.parametrize("red", [0, 1])
@pytest.mark.parametrize("mask", [None, P])
def test_numbers_that_fp32_does_not_hold(kw, red, mask):
    """Weights and coefficients that would be infinite or 0 in the kernels, or take a count's
    place back (a denominator whose inverse is 0)."""
    lib = _lib.load_tokens()
    l, big = loss(**kw, red=red), 1 << 40
    assert lib.ppo_token_policy_loss(rows(mask=mask), P, P, P, l, P, P, P, P, P, big, None) == 1
    if "den" in kw or "scale" in kw:
        assert lib.ppo_token_distillation(rows(mask=mask), P, 0, P, 1, 3, l, P, P, P, P, big,
                                          None) == 1
        with pytest.raises(ValueError, match="denominator|grad_scale"):
            tokens._check_weights("token", kw.get("den"), kw.get("scale", 1.0))
    else:
        x, a = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
        z = torch.zeros(2)
        with pytest.MonkeyPatch.context() as m, pytest.raises(ValueError, match="_coef"):
            m.setattr(tokens, "_require", lambda *args: None)
            tokens._check_policy(x, a, z, z, z, None, 0.2, 0.2, kw.get("kl", 0.0),
                                 kw.get("ent", 0.0), 1.0)


def test_preference_arguments():
    lib = _lib.load_tokens()

    def call(rel=P, S=4, T=5, beta=0.1, margin=0.0, smooth=0.0, out=P, rewards=P, coef=P, work=P,
             nbytes=1 << 20):
        return lib.ppo_token_preference(rel, None, S, T, beta, margin, smooth, 0, out, rewards, coef,
                                        work, nbytes, None)

    assert call(rel=None) == 1 and call(out=None) == 1 and call(rewards=None) == 1
    assert call(coef=None) == 1 and call(S=3) == 1 and call(S=0) == 1 and call(T=-1) == 1
    assert call(beta=float("nan")) == 1 and call(margin=float("inf")) == 1
    assert call(smooth=-0.1) == 1 and call(smooth=1.5) == 1 and call(smooth=float("nan")) == 1
    assert call(S=1 << 20, T=1 << 11) == 3
    assert call(work=None) == 2 and call(nbytes=8) == 2 and call(work=ODD) == 2
    assert lib.ppo_token_preference_workspace_bytes(0) == 0


def test_distillation_arguments():
    lib = _lib.load_tokens()

    def call(r=None, teacher=P, tt=0, ids=P, K=3, l=None, out=P, saved=P, d=P, work=P,
             nbytes=1 << 40):
        return lib.ppo_token_distillation(r or rows(actions=None), teacher, tt, ids, 1, K,
                                          l or loss(), out, saved, d, work, nbytes, None)

    assert call(teacher=None) == 1 and call(tt=3) == 1 and call(ids=None) == 1 and call(K=0) == 1
    assert call(K=257) == 3 and call(out=None) == 1 and call(saved=None) == 1
    assert call(l=loss(red=5)) == 1 and call(work=None) == 2 and call(nbytes=64) == 2
    b = lib.ppo_token_distillation_backward
    assert b(rows(), P, 0, P, 1, 257, P, P, 0.0, P, None) == 3
    assert b(rows(), P, 0, P, 1, 3, None, P, 0.0, P, None) == 1
    assert b(rows(), P, 0, P, 1, 3, P, None, 2.0, P, None) == 1
    assert b(rows(S=0), None, 0, None, 1, 3, None, None, 0.0, None, None) == 0


def test_top_arguments():
    lib = _lib.load_tokens()

    def call(x=P, dtype=0, R=4, A=30, K=3, v=P, i=P, work=None, nbytes=0):
        return lib.ppo_token_top(x, dtype, R, A, K, v, i, work, nbytes, None)

    assert call(x=None) == 1 and call(dtype=3) == 1 and call(R=-1) == 1 and call(A=0) == 1
    assert call(K=0) == 1 and call(K=31) == 1 and call(v=None) == 1 and call(i=None) == 1
    assert call(x=ODD, dtype=1) == 1 and call(v=ODD, dtype=2) == 1
    assert call(A=300, K=257) == 3 and call(A=(1 << 22) + 1) == 3
    assert call(R=0, x=None, v=None, i=None) == 0
    size = lib.ppo_token_top_workspace_bytes
    assert size(4096, 32000, 64, 0) == 0 and size(1, 131072, 64, 1) > 0
    assert call(R=1, A=131072, K=64) == 2 and size(0, 30, 3, 0) == 0
    assert call(R=1, A=131072, K=64, work=P, nbytes=size(1, 131072, 64, 0) - 1) == 2


def test_cpu_tensors_are_refused():
    x, a = torch.randn(2, 4, 6), torch.zeros(2, 4, dtype=torch.int64)
    z = torch.zeros(2, 4)
    for call in (lambda: ppo_amd.token_log_probs(x, a),
                 lambda: ppo_amd.token_policy_loss(x, a, z, z),
                 lambda: ppo_amd.preference_loss(x, a),
                 lambda: ppo_amd.distillation_loss(x, x[..., :2], a[..., None]),
                 lambda: ppo_amd.top_logits(x, 2)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


# --- the oracle against autograd ----------------------------------------------------------------

def test_oracle_log_probs():
    torch.manual_seed(0)
    x = torch.randn(5, 9, dtype=torch.float64, requires_grad=True)
    a, g, ge = torch.randint(0, 9, (5,)), torch.randn(5).double(), torch.randn(5).double()
    d = torch.distributions.Categorical(logits=x / 0.7)
    lp, H, ls = ref.log_probs(x, a, 0.7)
    assert torch.allclose(lp, d.log_prob(a)) and torch.allclose(H, d.entropy())
    (want,) = torch.autograd.grad((g * d.log_prob(a) + ge * d.entropy()).sum(), [x])
    assert torch.allclose(ref.log_probs_grad(ls.detach(), a, g, ge, 0.7), want)


def test_oracle_policy():
    torch.manual_seed(1)
    lp = torch.randn(40).double().requires_grad_()
    H = torch.rand(40).double().requires_grad_()
    old, adv, r = lp.detach() + 0.3 * torch.randn(40), torch.randn(40).double(), \
        lp.detach() + torch.randn(40)
    pol, kl, _, clipped, g, ge = ref.policy_terms(lp, H, old, adv, r, 0.1, 0.2, 0.3, 0.05)
    gl, gh = torch.autograd.grad((pol + 0.3 * kl - 0.05 * H).sum(), [lp, H])
    assert torch.allclose(g, gl) and torch.allclose(ge, gh) and 0 < clipped.sum() < 40


@pytest.mark.parametrize("average", [False, True])
def test_oracle_preference(average):
    torch.manual_seed(2)
    rel = torch.randn(6, 4).double().requires_grad_()
    mask = torch.rand(6, 4) < 0.6
    mask[2] = False
    loss_, rewards, coef = ref.preference(rel, mask, 0.7, 0.2, 0.1, average)
    (want,) = torch.autograd.grad(loss_, [rel])
    assert torch.allclose(coef, want) and rewards[2] == 0


def test_oracle_distillation():
    torch.manual_seed(3)
    x = torch.randn(5, 12, dtype=torch.float64, requires_grad=True)
    t, ids = torch.randn(5, 4).double(), torch.randint(0, 12, (5, 4))
    ids[:, 1], ids[0, 2], ids[3] = ids[:, 0], -1, -1
    ls = ref.log_softmax(x, 1.4)
    rows_, d, q = ref.distill_rows(ls, t, ids, 1.4)
    (want,) = torch.autograd.grad(rows_.sum(), [x])
    assert torch.allclose(d.detach() / 1.4, want) and rows_[3] == 0
    assert torch.allclose(q.sum(1), (ids >= 0).any(1).double())


def test_oracle_distillation_of_entries_that_weigh_nothing():
    torch.manual_seed(5)
    ls = ref.log_softmax(torch.randn(3, 8).double())
    t, ids = torch.randn(3, 2).double(), torch.randint(0, 8, (3, 2))
    t[1], t[2, 0] = -float("inf"), -float("inf")
    rows_, d, q = ref.distill_rows(ls, t, ids, 1.4)
    assert rows_[1] == 0 and not d[1].any() and not q[1].any() and q[2].tolist() == [0.0, 1.0]
    assert torch.allclose(rows_[2], -ls[2, ids[2, 1]])


def test_oracle_weights():
    mask = torch.tensor([[1, 1, 0], [0, 0, 0], [1, 0, 0]], dtype=torch.bool)
    assert torch.allclose(ref.weights(mask), mask.double() / 3)
    assert ref.weights(mask, "sequence").tolist() == [[0.25, 0.25, 0], [0, 0, 0], [0.5, 0, 0]]
    assert ref.weights(mask, "sequence", 4.0)[2, 0] == 0.25
    assert not ref.weights(mask & False).any()
