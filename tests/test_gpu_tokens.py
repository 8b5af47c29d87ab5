"""The token-policy operators on the GPU against their 64-bit restatement: sizes
around every layout's borders, odd rows and offsets, masks, values that are not
finite, streams, graphs, and the operators run together.

Tolerances count roundings (u = 2^-24 in 32 bits).  With t_j = z_max - z_j of a row:
e_j = 2^(c (l_j - m)) carries the rounding of l_j - m, of c and of their product,
each u t_j in e_j, and 2 u of the exponential itself; a sum of them carries one u for
each addition on the way, of which a lane makes at most 64, or A / 512 where it walks
a long row, and the lanes' join some ten more."""

import math
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

import ppo_amd
from oracle import tokens_oracle as ref
from ppo_amd import _lib, tokens
from ppo_amd.ops import _native

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U32 = 2.0 ** -24


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(11)


def u_of(t):
    return torch.finfo(t).eps / 2


def tiny_of(t):
    """Half the distance of the type's subnormals."""
    return 2.0 ** -25 if t == torch.float16 else 0.0


def adds_of(A):
    return 80 + A / 512


def rows_of(seed, t, R, A, width=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, A, generator=g) * width * (0.2 + torch.rand(R, 1, generator=g))).to(t)
    return x, torch.randint(0, A, (R,), generator=g), g


def at_offset(x, dev, offset):
    """A contiguous copy of x that starts `offset` elements into its storage."""
    flat = torch.empty(x.numel() + offset, dtype=x.dtype, device=dev)
    v = flat[offset:].view(x.shape)
    v.copy_(x)
    return v


def assert_within(got, want, bound, what=""):
    got, want = got.double().cpu(), want.double()
    assert torch.isfinite(got).all() or not torch.isfinite(want).all(), what
    over = (got - want).abs() - bound
    assert bool((over <= 0).all()), f"{what}: {float(over.max()):.3g} over its bound, error " \
                                    f"{float((got - want).abs().max()):.3g}"


class Bounds:
    """Errors of a row's results from the roundings counted above (x [R, A] in fp64)."""

    def __init__(self, x, actions, tau):
        self.tau, A = tau, x.shape[1]
        self.lp, self.H, self.ls = ref.log_probs(x, actions, tau)
        z = x / tau
        self.t = z.max(1, keepdim=True).values - z
        t = torch.where(torch.isfinite(self.t), self.t, torch.zeros_like(self.t))
        p = self.ls.exp()
        self.n = adds_of(A) + 8
        self.pt, ptt = (p * t).sum(1), (p * t * t).sum(1)
        self.e_s = U32 * (self.n + 3 * self.pt)  # of log s
        ta = t.gather(1, actions[:, None])[:, 0]
        self.e_lp = U32 * (self.lp.abs() + 3 * ta) + self.e_s
        self.e_H = 2 * U32 * self.n * (1 + self.pt) + 4 * U32 * (self.pt + ptt) + self.e_s \
            + U32 * self.H.abs()

    def dlogits(self, want, g, ge, dtype, dg=None):
        """Bound of a gradient whose coefficients g and ge [R] carry dg besides."""
        p = self.ls.exp()
        t = torch.where(torch.isfinite(self.t), self.t, torch.zeros_like(self.t))
        g, ge = g.abs()[:, None], ge.abs()[:, None]
        rel = 3 * U32 * (t + 1) + (2 * self.e_s + 12 * U32)[:, None]
        lns = (self.H - self.pt).abs()[:, None]
        size = g + ge * (self.H.abs()[:, None] + lns + t + 1)
        bound = p * (size * rel + ge * (self.e_H + U32 * self.H.abs())[:, None])
        if dg is not None:
            bound = bound + dg[:, None] * p
        # (at the action itself the terms are g (1 - p), not g p)
        near = (1 - p).abs() * g * rel + (0 if dg is None else dg[:, None] * (1 - p).abs())
        hot = want.abs() > 0
        bound = (bound + torch.where(hot, near.clamp(max=1e30) * self.hot, 0 * near)) / self.tau
        return bound + u_of(dtype) * (want.abs() + bound) + tiny_of(dtype)


def bounds(x, actions, tau=1.0):
    b = Bounds(x.double(), actions, tau)
    b.hot = torch.zeros_like(b.ls).scatter_(1, actions[:, None], 1.0)
    return b


# --- log-probabilities and entropies ---------------------------------------------------------

SHAPES = [(1, 1), (3, 2), (5, 7), (256, 18), (33, 64), (19, 127), (9, 500), (7, 513), (6, 1003),
          (5, 2049), (64, 3001), (3, 4100), (2, 8191), (66, 12289), (3, 16385), (67, 17001),
          (65, 33001), (64, 50257), (2, 131072), (1, 262147)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_log_probs_match_oracle(dev, shape, dtype):
    R, A = shape
    t, tau = TYPES[dtype], (1.0, 0.7, 1.5)[(R + A) % 3]
    x, a, g = rows_of(R * 31 + A, t, R, A)
    b = bounds(x, a, tau)
    xd = at_offset(x, dev, (R + A) % 4).requires_grad_()
    ad = a.to(dev) if A % 2 else a.to(dev, torch.int32)
    with torch.no_grad():
        lp0 = ppo_amd.token_log_probs(xd, ad, temperature=tau)
        both = ppo_amd.token_log_probs(xd, ad, temperature=tau, entropy=True)
    lp, H = ppo_amd.token_log_probs(xd, ad, temperature=tau, entropy=True)
    assert lp.dtype == H.dtype == torch.float32 and lp.shape == H.shape == (R,)
    assert torch.equal(lp, both[0]) and torch.equal(H, both[1])
    assert_within(lp0, b.lp, b.e_lp, "log-probabilities alone")
    assert_within(lp.detach(), b.lp, b.e_lp, "log-probabilities")
    assert_within(H.detach(), b.H, b.e_H, "entropies")
    gl, ge = torch.randn(R, generator=g), torch.randn(R, generator=g) * 0.3
    for ups in ((gl, ge), (gl, None), (None, ge)):
        outs = [o for o, u in zip((lp, H), ups) if u is not None]
        (dx,) = torch.autograd.grad(outs, [xd], [u.to(dev) for u in ups if u is not None],
                                    retain_graph=True)
        w = [torch.zeros(R).double() if u is None else u.double() for u in ups]
        want = ref.log_probs_grad(b.ls, a, *w, tau)
        assert dx.dtype == t
        assert_within(dx, want, b.dlogits(want, *w, t), f"gradient of {len(outs)}")


@pytest.mark.parametrize("dtype", list(TYPES))
def test_log_probs_keep_their_digits_where_one_action_has_all(dev, dtype):
    """p_a next to 1: log p_a and 1 - p_a relative to themselves, not to 1."""
    A = 40
    x = torch.zeros(6, A)
    x[:, 5] = torch.tensor([8.0, 12.0, 16.0, 24.0, 40.0, 60.0])
    x = x.to(TYPES[dtype])
    a = torch.full((6,), 5)
    lp, H, ls = ref.log_probs(x.double(), a)
    xd = x.to(dev).requires_grad_()
    got = ppo_amd.token_log_probs(xd, a.to(dev))
    want = -torch.log1p((A - 1) * torch.exp(-x[:, 5].double()))  # (ls itself cancels in 64 bits)
    # 3 t of the exponent's roundings, a few of the rest
    rel = U32 * (3 * x[:, 5].double() + 16)
    assert_within(got.detach(), want, want.abs() * rel, "log p")
    (dx,) = torch.autograd.grad(got.sum(), [xd])
    omp = -torch.expm1(want)
    bound = omp * (rel + u_of(TYPES[dtype])) + tiny_of(TYPES[dtype])
    assert_within(dx[:, 5], omp, bound, "1 - p")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("R, A", [(1, 1 << 27), (1030, 600001)])
def test_sums_of_very_wide_rows(dev, R, A, dtype):
    """The sums of a lane that walks thousands of elements are as good as short ones.  Every
    element weighs v = 1/2 + 2^-k (1 - 2^-6) but for one in 251, which weighs 1: added one by
    one to a sum of 2^(23 - k) or more, 32 bits would lose the 2^-k of each, 2^(1 - k) of all."""
    t = TYPES[dtype]
    if R > 1000 and t == torch.float32:
        A //= 2
    x = torch.full((R, A), 0.25, dtype=t, device=dev)
    x[:, ::251] = 1.0
    ones = (A + 250) // 251
    a = torch.full((R,), 7, device=dev)
    over = []
    for k in range(10, 17):
        z = math.log(0.5 + 2.0 ** -k * (1 - 2.0 ** -6))  # (of v; of 1 it is 0)
        with torch.no_grad():
            lp, H = ppo_amd.token_log_probs(x, a, temperature=-0.75 / z, entropy=True)
        s = ones + (A - ones) * math.exp(z)
        pt = (A - ones) * math.exp(z) / s * -z
        # a lane's eight rounds of 9 additions (16 of the entropy's sum) in 32 bits and the
        # rounding of what 64 bits have summed; the lanes', the workgroup's and the parts'
        # joins of up to ten additions and a factor of four roundings each
        n, n_H = 8 * 9 + 1 + 3 * 14, 8 * 16 + 1 + 3 * 14
        e_s = U32 * (n + 3 * pt)
        e_lp = U32 * (math.log(s) - 4 * z) + e_s
        e_H = 2 * U32 * n_H * (1 + pt) + 4 * U32 * pt * (1 - z) + e_s + U32 * (math.log(s) + pt)
        over += [float((lp.double() - z + math.log(s)).abs().max()) / e_lp,
                 float((H.double() - math.log(s) - pt).abs().max()) / e_H]
    assert max(over) <= 1, over


def test_log_probs_shapes(dev):
    x = torch.randn(2, 3, 5, 40, device=dev)
    a = torch.randint(0, 40, (2, 3, 5), device=dev)
    lp = ppo_amd.token_log_probs(x, a)
    assert lp.shape == (2, 3, 5)
    assert torch.equal(lp.view(-1), ppo_amd.token_log_probs(x.view(30, 40), a.view(-1)))
    one = ppo_amd.token_log_probs(x[0, 0, 0], a[0, 0, 0])
    assert one.shape == () and torch.equal(one, lp[0, 0, 0])
    empty = ppo_amd.token_log_probs(x[:0], a[:0], entropy=True)
    assert empty[0].shape == (0, 3, 5) and empty[1].shape == (0, 3, 5)
    xe = x[:0].clone().requires_grad_()
    (dx,) = torch.autograd.grad(ppo_amd.token_log_probs(xe, a[:0]).sum(), [xe])
    assert dx.shape == xe.shape


WIDTHS = [40, 900, 6000, 20000, 300000]


@pytest.mark.parametrize("A", WIDTHS)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_masked_rows_are_not_read(dev, dtype, A):
    """Rows that do not count hold NaN, infinities and wild actions; their results are
    0 and the others' bits are those of a call without them."""
    t = TYPES[dtype]
    R = 70 if A < 100000 else 5
    x, a, g = rows_of(A, t, R, A)
    mask = torch.rand(R, generator=g) < 0.5
    mask[0], mask[1] = True, False
    bad, wild = x.clone(), a.clone()
    bad[~mask] = float("nan")
    bad[~mask, 0] = float("inf")
    wild[~mask] = torch.tensor([-5, A, 1 << 40])[torch.arange(int((~mask).sum())) % 3]
    old = torch.zeros(R)
    old[~mask] = float("nan")
    one = torch.ones(R, device=dev)
    for m in (mask.to(dev), mask.to(dev, torch.uint8) * 7):
        runs = []
        for logits, act in ((x, a), (bad, wild)):
            xd = logits.to(dev).requires_grad_()
            lp, H = ppo_amd.token_log_probs(xd, act.to(dev), mask=m, entropy=True)
            (dx,) = torch.autograd.grad([lp, H], [xd], [one, one])
            xl = logits.to(dev).requires_grad_()
            loss, _ = ppo_amd.token_policy_loss(xl, act.to(dev), old.to(dev), old.to(dev) + 1,
                                                mask=m, entropy_coef=0.1)
            (dl,) = torch.autograd.grad(loss, [xl])
            runs.append([lp.detach(), H.detach(), dx, loss.detach(), dl])
        assert all(torch.equal(u, v) for u, v in zip(*runs))
        for out in runs[1][:3] + runs[1][4:]:
            assert not out[~mask.to(dev)].any()
            assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("A", WIDTHS)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_logits_that_are_not_finite(dev, dtype, A):
    """-inf is an action that cannot be taken; +inf, NaN and rows of nothing but -inf
    give NaN, as log_softmax does, and touch no other row."""
    t = TYPES[dtype]
    R = 72 if A < 100000 else 9
    x, a, g = rows_of(A + 1, t, R, A)
    hide = torch.rand(R, A, generator=g) < 0.6
    hide.scatter_(1, a[:, None], False)
    x[hide] = -float("inf")
    x[1, 3] = float("inf")
    x[2, A - 1] = float("nan")
    x[3] = -float("inf")
    x[4] = torch.finfo(t).min         # a mask's lowest value everywhere: uniform
    x[5] = torch.finfo(t).min
    x[5, A // 2] = 1.0                # ... everywhere but one
    a[5] = A // 2
    x[6] = -float("inf")
    x[6, 0], a[6] = 2.0, 0            # one action that can be taken, and is
    x[7, 1], a[7] = -float("inf"), 1  # one that cannot, taken
    nan = [1, 2, 3]
    ok = [r for r in range(R) if r not in nan]
    b = bounds(x[ok], a[ok])
    xd = x.to(dev).requires_grad_()
    lp, H = ppo_amd.token_log_probs(xd, a.to(dev), entropy=True)
    assert torch.isnan(lp[nan]).all() and torch.isnan(H[nan]).all()
    assert lp[7] == -float("inf")
    fine = [i for i, r in enumerate(ok) if r != 7]
    keep = [r for r in ok if r != 7]
    assert_within(lp.detach()[keep], b.lp[fine], b.e_lp[fine], "log p")
    assert_within(H.detach()[ok], b.H, b.e_H, "H")
    gl, ge = torch.randn(R, generator=g), torch.randn(R, generator=g)
    (dx,) = torch.autograd.grad([lp, H], [xd], [gl.to(dev), ge.to(dev)])
    assert torch.isnan(dx[nan]).all()
    want = ref.log_probs_grad(b.ls, a[ok], gl[ok].double(), ge[ok].double())
    assert_within(dx[ok], want, b.dlogits(want, gl[ok].double(), ge[ok].double(), t), "dlogits")
    assert not dx[ok][(x[ok] == -float("inf")).to(dev) & ~(b.hot > 0).to(dev)].any()


@pytest.mark.parametrize("A", [30, 1000, 20000, 300000])
@pytest.mark.parametrize("low", [-float("inf"), torch.finfo(torch.float32).min])
def test_entropy_gradients_of_a_scaled_loss_where_nothing_can_be_taken(dev, A, low):
    """Logits that are left out get a gradient of 0 whatever the incoming one's size; the
    others' are in proportion (a power of two: the same roundings)."""
    R, k = (70, 1) if A < 100000 else (4, 16)
    x, a, g = rows_of(A, torch.float32, R, A)
    hide = torch.rand(R, A, generator=g) < 0.5
    hide.scatter_(1, a[:, None], False)
    x[hide] = low
    hide, ad, up, z = hide.to(dev), a.to(dev), k * 2.0 ** 34, torch.zeros(R, device=dev)
    for offset in (0, 3):
        xd = at_offset(x, dev, offset).requires_grad_()
        _, H = ppo_amd.token_log_probs(xd, ad, entropy=True)
        small, big = (torch.autograd.grad(H, [xd], torch.full_like(z, v), retain_graph=True)[0]
                      for v in (1.0, up))
        assert not big[hide].any() and torch.equal(big, small * up)
        old = ppo_amd.token_log_probs(xd.detach(), ad)
        for scale in (1.0, up):
            loss, _ = ppo_amd.token_policy_loss(xd, ad, old, z, entropy_coef=1.0, grad_scale=scale)
            (d,) = torch.autograd.grad(loss, [xd], torch.tensor(up, device=dev))
            assert torch.isfinite(d).all() and not d[hide].any()


def test_actions_outside_the_row(dev):
    for A in (18, 5000, 40000):
        x = torch.randn(66, A, device=dev).requires_grad_()
        a = torch.randint(0, A, (66,), device=dev)
        lp0 = ppo_amd.token_log_probs(x, a)
        (d0,) = torch.autograd.grad(lp0.sum(), [x])
        bad = a.clone()
        bad[3], bad[7], bad[9] = -1, A, 1 << 40
        lp = ppo_amd.token_log_probs(x, bad)
        (d,) = torch.autograd.grad(lp.sum(), [x])
        rest = torch.ones(66, dtype=torch.bool, device=dev)
        rest[[3, 7, 9]] = False
        assert torch.isnan(lp[~rest]).all() and torch.isnan(d[~rest]).all()
        assert torch.equal(lp[rest], lp0[rest]) and torch.equal(d[rest], d0[rest])
        loss, _ = ppo_amd.token_policy_loss(x, bad, lp0.detach(), lp0.detach())
        assert torch.isnan(loss)


# --- the policy loss -----------------------------------------------------------------------

def policy_case(seed, t, S, T, A, tau=1.0, empty=True):
    x, a, g = rows_of(seed, t, S * T, A)
    lp, _, _ = ref.log_probs(x.double(), a, tau)
    move = (torch.randn(S * T, generator=g) * 0.2).double()
    for border in (math.log1p(-0.2), math.log1p(0.3)):  # off the borders of the clip
        move = torch.where((move - border).abs() < 1e-3, move + 4e-3, move)
    case = dict(x=x, a=a, old=(lp - move).float(), adv=torch.randn(S * T, generator=g),
                ref=(lp + 0.4 * torch.randn(S * T, generator=g)).float(),
                mask=torch.rand(S, T, generator=g) < 0.7, g=g)
    case["mask"][0, 0] = True
    if empty and S > 1:
        case["mask"][1] = False
    return case


def policy_want(c, S, T, tau, low, high, kc, ec, mask, reduction, denominator, t, with_ref):
    """(scalars in order, their bounds, dlogits, its bound) of the loss."""
    b = bounds(c["x"], c["a"], tau)
    d = lambda v: v.double()  # noqa: E731
    w = ref.weights(mask, reduction, denominator).view(-1)
    pol, kl, akl, clipped, g, ge = ref.policy_terms(
        b.lp, b.H, d(c["old"]), d(c["adv_rows"]), d(c["ref"]) if with_ref else None, low, high, kc, ec)
    g, ge = g * w, ge * w
    sums = [(w * v).sum() for v in (pol, kl, b.H, akl, clipped)]
    e = b.e_lp + 2 * U32  # of a ratio, relative: the difference's rounding is in e_lp's size
    e = e + U32 * (b.lp - d(c["old"])).abs()
    e_pol = pol.abs() * (e + 4 * U32)
    e_kl = (torch.expm1(d(c["ref"]) - b.lp).abs() * (b.e_lp + U32) + kl * 16 * U32
            if with_ref else torch.zeros_like(kl))
    e_akl = b.e_lp + U32 * akl.abs()
    errs = [(w * v).sum() for v in (e_pol, e_kl, b.e_H, e_akl, 0 * e)]
    size = [(w * v.abs()).sum() for v in (pol, kl, b.H, akl, clipped)]
    errs = [x + 4 * U32 * s for x, s in zip(errs, size)]  # (weights and the result's rounding)
    loss = sums[0] + kc * sums[1] - ec * sums[2]
    loss_err = errs[0] + kc * errs[1] + ec * errs[2] + U32 * loss.abs()
    order = [(loss, loss_err), (sums[0], errs[0]), (sums[1], errs[1]), (sums[2], errs[2]),
             (sums[3], errs[3]), (sums[4], errs[4])]
    dg = w * (c["adv_rows"].double() * torch.exp(b.lp - d(c["old"]))).abs() * (e + 4 * U32)
    if with_ref and kc:
        dg = dg + w * kc * (torch.exp(d(c["ref"]) - b.lp) * (b.e_lp + U32) + kl * 16 * U32)
    want = ref.log_probs_grad(b.ls, c["a"], g, ge, tau)
    bound = b.dlogits(want, g, ge, t, dg + 4 * U32 * g.abs())
    return order, want, bound


POLICY_SHAPES = [(1, 1, 1), (2, 3, 5), (16, 16, 18), (64, 65, 900), (3, 50, 200), (3, 5, 300),
                 (4, 9, 1000), (3, 4, 2111),
                 (2, 35, 4097), (3, 30, 9001), (2, 40, 17000), (5, 13, 33000), (2, 33, 70001),
                 (3, 2, 131071), (2, 32, 129000), (1, 2, 300001), (2, 33, 150000),
                 (2, 33, 196000)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", POLICY_SHAPES)
def test_policy_loss_matches_oracle(dev, shape, dtype):
    S, T, A = shape
    t, k = TYPES[dtype], S + T + A
    if dtype != "bf16" and S * T * A > 5000000:
        A = A // 2  # (the same layouts: fp32 rows are twice as long)
    tau = (1.0, 0.8)[k % 2]
    c = policy_case(k, t, S, T, A, tau)
    masked, per_seq, with_ref = k % 3 != 0, k % 4 == 1, k % 5 != 2
    kc, ec = (0.07 if with_ref and k % 2 else 0.0), (0.02 if k % 3 else 0.0)
    reduction, denominator = ("token", "sequence")[k % 2], (None, None, 37.0)[k % 3]
    mask = c["mask"] if masked else torch.ones(S, T, dtype=torch.bool)
    adv = c["adv"].view(S, T)[:, 0] if per_seq else c["adv"].view(S, T)
    c["adv_rows"] = (adv[:, None].expand(S, T) if per_seq else adv).reshape(-1)
    order, want, bound = policy_want(c, S, T, tau, 0.2, 0.3, kc, ec, mask, reduction, denominator,
                                     t, with_ref)
    v = lambda n: c[n].view(S, T).to(dev)  # noqa: E731
    xd = at_offset(c["x"].view(S, T, A), dev, 8 * (k % 2)).requires_grad_()
    run = lambda x: ppo_amd.token_policy_loss(  # noqa: E731
        x, v("a"), v("old"), adv.contiguous().to(dev), v("ref") if with_ref else None,
        mask.to(dev) if masked else None, 0.2, 0.3, kc, ec, tau, reduction, denominator)
    loss, stats = run(xd)
    for name, (value, err) in zip(_lib.TOKEN_SCALAR_NAMES, order):
        assert_within(stats[name], value, err, name)
    assert torch.equal(loss.detach(), stats["loss"])
    (dx,) = torch.autograd.grad(loss, [xd])
    assert dx.dtype == t and dx.shape == (S, T, A)
    assert_within(dx.view(S * T, A), want, bound, "dlogits")
    # without a gradient, and from an offset that the result does not share
    with torch.no_grad():
        quiet, stats0 = run(xd)
        assert all(torch.equal(stats0[n], stats[n]) for n in stats) and torch.equal(quiet, loss)
    xo = at_offset(c["x"].view(S, T, A), dev, 3).requires_grad_()
    loss, stats = run(xo)
    for name, (value, err) in zip(_lib.TOKEN_SCALAR_NAMES, order):
        assert_within(stats[name], value, err, name + " off alignment")
    assert_within(torch.autograd.grad(loss, [xo])[0].view(S * T, A), want, bound, "off alignment")


@pytest.mark.parametrize("A", [18, 1000, 9000, 40000, 280000])
def test_policy_loss_incoming_gradients(dev, A):
    """grad_scale 1, another, the loss differentiated twice: each gradient is the loss's
    own, rounded once."""
    S, T, t = 2, 33 if A < 100000 else 1, torch.bfloat16
    c = policy_case(A, t, S, T, A)
    c["adv_rows"] = c["adv"]
    _, want, _ = policy_want(c, S, T, 1.0, 0.2, 0.2, 0.1, 0.01, c["mask"], "token", None, t, True)
    v = lambda n: c[n].view(S, T).to(dev)  # noqa: E731
    base = policy_want(c, S, T, 1.0, 0.2, 0.2, 0.1, 0.01, c["mask"], "token", None, torch.float32,
                       True)[2]
    for scale in (1.0, 1024.0, 3.0):
        x = c["x"].view(S, T, A).to(dev).requires_grad_()
        loss, _ = ppo_amd.token_policy_loss(x, v("a"), v("old"), v("adv"), v("ref"),
                                            v("mask"), 0.2, None, 0.1, 0.01, grad_scale=scale)
        kept = []
        for up in (scale, 1.0, 0.0, scale, -2.5):
            (dx,) = torch.autograd.grad(loss * up, [x], retain_graph=True)
            bound = abs(up) * (base + u_of(t) * (want.abs() + base))
            assert_within(dx.view(S * T, A), up * want, bound + 1e-40, f"{scale} {up}")
            kept.append((dx, dx.clone()))
        assert all(torch.equal(p, q) for p, q in kept)  # (no later pass writes an earlier one's)


@pytest.mark.parametrize("A", [18, 1000, 9000, 40000, 280000])
def test_policy_loss_far_from_the_reference(dev, A):
    """The KL term's derivative in log p is -(e^d - 1) however far the reference lies, and
    finite where it rules out the action that was taken (the loss is infinite there)."""
    far = torch.tensor([-float("inf"), -1e30, -1e9, -3e4, -200.0, -30.0, -5.0, -1.01, -0.99, -1e-4,
                        0.0, 0.5, 1.0, 1.5, 20.0])
    S, T, t = (6 if A < 100000 else 1), 15, torch.float32
    c = policy_case(A, t, S, T, A)
    b = bounds(c["x"], c["a"])
    r = (b.lp + far.repeat(S)).float()
    old, adv, kc, w = c["old"].double(), c["adv"].double(), 0.3, 1.0 / (S * T)
    _, kl, _, _, g, _ = ref.policy_terms(b.lp, b.H, old, adv, r.double(), 0.2, 0.2, kc, 0.0)
    # e^d carries log p's error, d's rounding and two units of expf; of the series 16 in all
    d, ratio = r.double() - b.lp, torch.exp(b.lp - old)
    dg = w * (adv * ratio).abs() * (b.e_lp + U32 * (6 + (b.lp - old).abs()))
    dg = dg + w * kc * (torch.exp(d) * (b.e_lp + U32 * (4 + d.abs().clamp(max=100)))
                        + 4 * U32 * torch.expm1(d).abs() + 16 * U32 * kl.clamp(max=1.0))
    want = ref.log_probs_grad(b.ls, c["a"], g * w, 0 * g)
    bound = b.dlogits(want, g * w, 0 * g, t, dg + 4 * U32 * (g * w).abs())
    v = lambda u: u.view(S, T).to(dev)  # noqa: E731
    for offset in (0, 3):
        xd = at_offset(c["x"].view(S, T, A), dev, offset).requires_grad_()
        loss, stats = ppo_amd.token_policy_loss(xd, v(c["a"]), v(c["old"]), v(c["adv"]), v(r),
                                                kl_coef=kc)
        assert loss == float("inf") and stats["kl"] == float("inf")
        for up in (1.0, 2.0):
            (dx,) = torch.autograd.grad(loss, [xd], torch.tensor(up, device=dev), retain_graph=True)
            assert_within(dx.view(S * T, A), up * want, up * bound, f"{offset} {up}")


def test_policy_loss_over_nothing(dev):
    """Masks that leave nothing, and no rows at all: 0, and gradients of 0."""
    f = ppo_amd.token_policy_loss
    for S, T, A in ((3, 5, 40), (2, 2, 40000), (0, 5, 40), (3, 0, 40)):
        x = torch.full((S, T, A), float("nan"), device=dev).requires_grad_()
        z = torch.full((S, T), float("nan"), device=dev)
        mask = torch.zeros(S, T, dtype=torch.bool, device=dev)
        for reduction in ("token", "sequence"):
            loss, stats = f(x, z.long(), z, z, z, mask, kl_coef=0.1, reduction=reduction)
            assert loss == 0 and all(s == 0 for s in stats.values())
            (dx,) = torch.autograd.grad(loss, [x])
            assert dx.shape == x.shape and not dx.any()


def test_policy_loss_first_update(dev):
    """Old log-probabilities of the same policy: ratio 1, nothing clipped, and the
    gradient is that of -mean(advantage log p)."""
    x = torch.randn(4, 20, 3000, device=dev, dtype=torch.bfloat16).requires_grad_()
    a = torch.randint(0, 3000, (4, 20), device=dev)
    adv = torch.randn(4, 20, device=dev)
    old = ppo_amd.token_log_probs(x, a).detach()
    loss, stats = ppo_amd.token_policy_loss(x, a, old, adv)
    assert stats["clipfrac"] == 0 and abs(float(stats["approx_kl"])) < 4 * U32 * 16
    (dx,) = torch.autograd.grad(loss, [x])
    lp = ppo_amd.token_log_probs(x, a)
    (want,) = torch.autograd.grad(-(adv * lp).mean(), [x])
    # two roundings to bf16 a step apart at most: of values within a few u of each other
    assert bool(((dx - want).abs().float() <= 2 * u_of(torch.bfloat16) * want.abs().float()
                 * (1 + 1e-4) + 1e-12).all())


# --- preferences ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(2, 1, 1), (2, 1, 7), (4, 9, 40), (8, 31, 1000), (6, 300, 257),
                                   (2, 40, 9000), (4, 17, 40001), (2, 1, 300001), (2, 9000, 7),
                                   (2, 17001, 5), (40, 900, 3), (4, 3000, 5),
                                   (10, 65, 9), (130, 3, 6), (2000, 17, 3), (4, 9000, 2)])
def test_preference_loss_matches_oracle(dev, shape, dtype):
    S, T, A = shape
    t, k = TYPES[dtype], S + T + A
    tau, beta, margin = (1.0, 1.3)[k % 2], (0.1, 2.0)[k % 2], (0.0, 0.4)[k % 3 % 2]
    smoothing, average = (0.0, 0.1, 1.0)[k % 3], k % 2 == 1
    c = policy_case(k, t, S, T, A, tau, empty=S > 2)
    mask = c["mask"] if k % 4 else torch.ones(S, T, dtype=torch.bool)
    b = bounds(c["x"], c["a"], tau)
    lp = b.lp.view(S, T)
    with_ref = k % 5 != 0
    r = c["ref"].double().view(S, T) if with_ref else torch.zeros(S, T).double()
    want_loss, want_rewards, coef = ref.preference(lp - r, mask, beta, margin, smoothing, average)
    n = mask.double().sum(1).clamp(min=1) if average else torch.ones(S).double()
    # (log p - ref is rounded once; e_lp covers what log p itself carries)
    e_row = torch.where(mask, b.e_lp.view(S, T) + U32 * (lp - r).abs(), 0 * lp)
    e_rew = beta * e_row.sum(1) / n + 2 * U32 * want_rewards.abs()
    e_m = (e_rew[:S // 2] + e_rew[S // 2:])
    v = lambda x: x.view(S, T).to(dev)  # noqa: E731
    xd = at_offset(c["x"].view(S, T, A), dev, k % 3).requires_grad_()
    run = lambda: ppo_amd.preference_loss(  # noqa: E731
        xd, v(c["a"]), v(c["ref"]) if with_ref else None, mask.to(dev) if k % 4 else None, beta,
        smoothing, margin, average, tau)
    loss, stats = run()
    rewards = torch.cat([stats["chosen"], stats["rejected"]])
    assert_within(rewards, want_rewards, e_rew, "rewards")
    assert_within(loss.detach(), want_loss, e_m.mean() + 2 * U32 * want_loss.abs(), "loss")
    with torch.no_grad():
        again, stats0 = run()
    assert torch.equal(again, loss) and torch.equal(stats0["chosen"], stats["chosen"])
    up = 2.0 if k % 2 else 1.0
    (dx,) = torch.autograd.grad(loss * up, [xd])
    g = (up * coef).view(-1)
    want = ref.log_probs_grad(b.ls, c["a"], g, 0 * g, tau)
    # the coefficient moves with m: |d sigmoid| <= 1/4
    dg = up * (beta / n[:, None] * mask.double() * torch.cat([e_m, e_m])[:, None] / (S // 2)).view(-1)
    bound = b.dlogits(want, g, 0 * g, t, dg + 4 * U32 * g.abs())
    assert_within(dx.view(S * T, A), want, bound, "dlogits")


def test_preference_loss_of_far_pairs(dev):
    """Margins where a sigmoid leaves 32 bits, and sequences without tokens."""
    x = torch.zeros(4, 2, 4, device=dev).requires_grad_()
    a = torch.zeros(4, 2, dtype=torch.int64, device=dev)
    r = torch.tensor([[-400.0, -400.0], [300.0, 300.0], [0.0, 0.0], [0.0, 0.0]], device=dev)
    loss, stats = ppo_amd.preference_loss(x, a, r, beta=1.0)
    base = -2 * math.log(4.0)
    m = [800.0, -600.0]
    assert torch.allclose(stats["chosen"].double().cpu(), torch.tensor([base + 800, base - 600]).double())
    assert abs(float(loss.detach()) - 300.0) < 1e-4
    (dx,) = torch.autograd.grad(loss, [x])
    assert m and not dx[0].any() and not dx[2].any()          # e^-800 is 0
    want = torch.tensor([-0.375, 0.125, 0.125, 0.125], device=dev)  # -(1 - p) / 2, p / 2
    assert torch.allclose(dx[1, 0], want) and torch.allclose(dx[3, 1], -want)
    loss, stats = ppo_amd.preference_loss(x, a, r, torch.zeros(4, 2, dtype=torch.bool, device=dev),
                                          average=True)
    assert abs(float(loss) - math.log(2.0)) < 1e-6 and not stats["chosen"].any()
    assert not torch.autograd.grad(loss, [x])[0].any()
    loss, _ = ppo_amd.preference_loss(x[:, :0], a[:, :0])
    assert abs(float(loss) - math.log(2.0)) < 1e-6


@pytest.mark.parametrize("A", [40, 20000])
def test_preference_at_the_largest_temperatures(dev, A):
    """Nearly uniform rows but for the actions that cannot be taken, up to where
    log2(e) / temperature is no normal number."""
    x = torch.randn(4, 3, A, device=dev)
    x[:, :, 7] = -float("inf")
    a, z = torch.zeros(4, 3, dtype=torch.int64, device=dev), torch.zeros(4, 3, device=dev)
    want = -0.1 * 3 * math.log(A - 1)
    for k in range(48):
        tau = 1e37 * 1.07 ** k
        _, stats = ppo_amd.preference_loss(x, a, z, temperature=tau)
        for reward in (*stats["chosen"], *stats["rejected"]):
            assert abs(float(reward) - want) <= 8 * U32 * -want, tau


@pytest.mark.parametrize("tau", [0.3, 0.7, 1.0, 1.5])
@pytest.mark.parametrize("A", [40, 900, 20000, 300000])
def test_preference_of_close_policies(dev, A, tau):
    """Unlikely actions of policies close to their reference: what is left of the
    difference is not the rounding of log2(e) / tau, up to u of 80.  With the row's sum
    in 64 bits a difference is off by the exponentials (2 u each, and again where a
    part's maximum is taken to the row's), their exponents' roundings (u t each) and its own
    rounding: u (8 + 4 sum p t + |rel|) with room for the factors."""
    g = torch.Generator().manual_seed(A)
    S, T = 4, 3
    x = -20.0 * tau + torch.randn(S, T, A, generator=g)
    a = torch.randint(1, A, (S, T), generator=g)
    x[..., 0] = 0.0
    x.scatter_(-1, a[..., None], -80.0 * tau)
    b = bounds(x.view(S * T, A), a.view(-1), tau)
    ref_ = (b.lp + 0.01 * torch.randn(S * T, generator=g)).float()
    rel = (b.lp - ref_.double()).view(S, T)
    err = (U32 * (8 + 4 * b.pt + rel.abs().view(-1))).view(S, T)
    _, stats = ppo_amd.preference_loss(x.to(dev), a.to(dev), ref_.view(S, T).to(dev), beta=1.0,
                                       temperature=tau)
    got = torch.cat([stats["chosen"], stats["rejected"]])
    assert_within(got, rel.sum(1), err.sum(1) + U32 * rel.sum(1).abs(), "rewards")


# --- distillation ------------------------------------------------------------------------------

def distill_case(seed, t, tt, S, T, A, K):
    x, _, g = rows_of(seed, t, S * T, A)
    teacher = (torch.randn(S * T, K, generator=g) * 2 + 5).to(tt)
    ids = torch.randint(0, A, (S * T, K), generator=g)  # (ids come twice now and then)
    if K > 1:
        ids[:, 1] = ids[:, 0]
        ids[torch.rand(S * T, K, generator=g) < 0.1] = -1
    if S * T > 2:
        ids[2] = -3                                      # a row without entries
    return x, teacher, ids, g


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (2, 3, 5, 3), (16, 16, 18, 18), (3, 5, 300, 20),
                                   (4, 9, 1000, 64), (3, 4, 2111, 65), (2, 35, 4097, 100),
                                   (2, 40, 17000, 256), (5, 13, 33000, 7), (2, 32, 70001, 64),
                                   (3, 2, 131071, 200), (2, 32, 129000, 64), (1, 2, 300001, 33),
                                   (2, 70, 40, 200), (3, 7, 300, 256), (5, 9, 500, 130),
                                   (2, 9, 257, 129), (2, 33, 150000, 64), (2, 33, 196000, 20)])
def test_distillation_matches_oracle(dev, shape, dtype):
    S, T, A, K = shape
    t, k = TYPES[dtype], S + T + A + K
    if dtype != "bf16" and S * T * A > 5000000:
        A = A // 2
    tt = list(TYPES.values())[k % 3]
    tau, reduction = (1.0, 2.0)[k % 2], ("sequence", "token")[k % 2]
    denominator = (None, 11.0)[k % 2]
    x, teacher, ids, g = distill_case(k, t, tt, S, T, A, K)
    mask = torch.rand(S, T, generator=g) < 0.8
    mask[0, 0] = True
    b = bounds(x, ids[:, 0].clamp(min=0), tau)
    rows, d, q = ref.distill_rows(b.ls, teacher.double(), ids, tau)
    masked = k % 3 != 1
    w = ref.weights(mask if masked else torch.ones_like(mask), reduction, denominator).view(-1)
    want_loss, want = tau * tau * (w * rows).sum(), d * (w * tau)[:, None]
    # log q and log p: their exponents' roundings, that of their sums, and K additions
    tq = ((teacher.double().max(1, keepdim=True).values - teacher.double()) / tau * q).sum(1)
    tp = (q * b.t.gather(1, ids.clamp(min=0))).sum(1)
    e_rows = b.e_s + U32 * (8 * (tq + tp) + (K + 24) * (1 + tq + tp) + b.lp.abs())
    e_loss = tau * tau * (w * e_rows).sum() + 4 * U32 * want_loss.abs()
    e_q = torch.zeros_like(want).scatter_add_(
        1, ids.clamp(min=0), q * U32 * (3 * (teacher.double().max() - teacher.double()).abs() / tau
                                        + K + 16))
    p = b.ls.exp()
    e_p = p * (3 * U32 * (b.t + 1) + (b.e_s + 12 * U32)[:, None])
    bound = (w * tau)[:, None] * (e_p + e_q + 4 * U32 * (p + want.abs()))
    bound = bound + u_of(t) * (want.abs() + bound) + tiny_of(t)
    idd = ids.view(S, T, K).to(dev, torch.int32 if k % 2 else torch.int64)
    for offset in (0, 8, 3):
        xd = at_offset(x.view(S, T, A), dev, offset).requires_grad_()
        run = lambda: ppo_amd.distillation_loss(  # noqa: E731
            xd, teacher.view(S, T, K).to(dev), idd, mask.to(dev) if masked else None, tau,
            reduction, denominator)
        loss = run()
        with torch.no_grad():
            quiet = run()
        # (rows off alignment form their gradient apart, and small ones sum their entries
        # over 16 lanes there: other roundings of the same sum)
        assert torch.equal(quiet, loss) or offset == 3
        for value in (loss.detach(), quiet):
            assert_within(value, want_loss, e_loss, f"loss {offset}")
        for up in (1.0, -3.0, 1.0):  # formed with the loss, anew, and anew again
            (dx,) = torch.autograd.grad(loss * up, [xd], retain_graph=True)
            assert dx.dtype == t
            assert_within(dx.view(S * T, A), up * want, abs(up) * bound, f"dlogits {offset} {up}")


@pytest.mark.parametrize("A", [30, 1000, 20000, 300000])
def test_distillation_edges(dev, A):
    R = 70 if A < 100000 else 4
    x = torch.randn(R, A, device=dev).requires_grad_()
    teacher = torch.randn(R, 3, device=dev)
    ids = torch.randint(0, A, (R, 3), device=dev)
    clean = ppo_amd.distillation_loss(x, teacher, ids)
    (d0,) = torch.autograd.grad(clean, [x])
    # entries that weigh nothing: a teacher's -inf
    t1, i1 = torch.cat([teacher, torch.full((R, 1), -float("inf"), device=dev)], 1), \
        torch.cat([ids, (ids[:, :1] + 1) % A], 1)
    loss = ppo_amd.distillation_loss(x, t1, i1)
    (d1,) = torch.autograd.grad(loss, [x])
    assert torch.equal(loss, clean) and torch.allclose(d1, d0, rtol=8 * U32, atol=1e-12)
    # an id outside the row, and a teacher's NaN, are that row's NaN
    for wreck in ("id", "teacher"):
        t2, i2 = teacher.clone(), ids.clone()
        if wreck == "id":
            i2[1, 2] = A
        else:
            t2[1, 2] = float("nan")
        loss = ppo_amd.distillation_loss(x, t2, i2)
        (d2,) = torch.autograd.grad(loss, [x])
        rest = [r for r in range(R) if r != 1]
        assert torch.isnan(loss) and torch.isnan(d2[1]).sum() >= A - 3
        assert torch.equal(d2[rest], d0[rest])
    # no entries at all
    loss = ppo_amd.distillation_loss(x, teacher, ids * 0 - 1)
    assert loss == 0 and not torch.autograd.grad(loss, [x])[0].any()
    # the student's -inf at an entry of the teacher's: an infinite loss
    y = x.detach().clone()
    y[0, ids[0, 0]] = -float("inf")
    assert ppo_amd.distillation_loss(y, teacher, ids) == float("inf")
    # a student that equals its teacher learns nothing more of the entries
    if A <= 256:
        v, i = ppo_amd.top_logits(x.detach(), A)
        loss = ppo_amd.distillation_loss(x, v, i)
        assert abs(float(loss)) < 64 * U32
        (d,) = torch.autograd.grad(loss, [x])
        assert float(d.abs().max()) < 64 * U32 / R


@pytest.mark.parametrize("A", [30, 1000, 20000, 40000, 300000])
@pytest.mark.parametrize("offset", [0, 3])
def test_distillation_of_entries_that_weigh_nothing(dev, A, offset):
    """A row whose entries are all a teacher's -inf is one without entries: no loss, no
    gradient, neither with the forward pass nor formed anew, in every layout."""
    R = 70 if A < 100000 else 4
    x = at_offset(torch.randn(R, A), dev, offset).requires_grad_()
    teacher = torch.randn(R, 5, device=dev)
    ids = torch.randint(0, A, (R, 5), device=dev)
    ids[1, 3] = ids[1, 0]
    none = ids.clone()
    none[1] = -1
    teacher[1] = -float("inf")
    runs = []
    for i in (ids, none):
        loss = ppo_amd.distillation_loss(x, teacher, i, temperature=2.0)
        runs.append([loss.detach(), *(torch.autograd.grad(loss * up, [x], retain_graph=True)[0]
                                      for up in (1.0, -3.0))])
    assert all(torch.equal(p, q) for p, q in zip(*runs))
    for d in runs[0][1:]:
        assert not d[1].any() and d[0].any()
    assert torch.isfinite(runs[0][0])


@pytest.mark.parametrize("A", [30, 1000, 20000, 300000])
@pytest.mark.parametrize("wreck", ["nan", "inf", "-inf"])
def test_distillation_of_a_wrecked_row_without_entries(dev, A, wreck):
    """A row that gives NaN (NaN, +inf, nothing but -inf) does so in the loss as in the
    gradient, also without entries."""
    R = 70 if A < 100000 else 4
    x = torch.randn(R, A, device=dev)
    x[1, slice(None) if wreck == "-inf" else A // 2] = float(wreck)
    x.requires_grad_()
    ids = torch.randint(0, A, (R, 3), device=dev)
    ids[1] = -1
    teacher = torch.randn(R, 3, device=dev)
    loss = ppo_amd.distillation_loss(x, teacher, ids)
    rest = [r for r in range(R) if r != 1]
    for up in (1.0, 2.0):
        (d,) = torch.autograd.grad(loss * up, [x], retain_graph=True)
        assert torch.isnan(d[1]).all() and torch.isfinite(d[rest]).all()
    assert torch.isnan(loss)
    with torch.no_grad():
        assert torch.isnan(ppo_amd.distillation_loss(x, teacher, ids))
        mask = torch.arange(R, device=dev) != 1
        assert torch.isfinite(ppo_amd.distillation_loss(x, teacher, ids, mask))


# --- top logits ----------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 5, 5), (200, 18, 4), (7, 300, 256), (5, 1003, 64),
                                   (300, 2049, 17), (9, 8200, 200), (130, 9000, 1), (3, 16385, 50),
                                   (129, 33001, 64), (130, 66001, 100), (2, 131072, 256),
                                   (1, 262147, 50), (1, 2000001, 256),
                                   (600, 4097, 48), (300, 512, 256), (1000, 33, 20), (5, 8200, 33),
                                   (40, 511, 49)])
def test_top_logits_match_a_stable_sort(dev, shape, dtype):
    R, A, k = shape
    x, _, g = rows_of(R + A + k, TYPES[dtype], R, A)
    if dtype == "fp32" and A % 2:
        x = (x * 8).round() / 8  # (many ties)
    xd = at_offset(x, dev, (R + k) % 4)
    v, i = ppo_amd.top_logits(xd, k)
    wv, wi = ref.top(x.float(), k)
    assert v.dtype == x.dtype and i.dtype == torch.int64 and v.shape == i.shape == (R, k)
    assert torch.equal(i.cpu(), wi) and torch.equal(v.cpu().float(), wv)


def test_top_logits_of_many_narrow_rows(dev):
    """More rows than a launch of workgroups holds, by a wave each."""
    x = torch.randn((1 << 22) + 3, 3, device=dev, dtype=torch.float16)
    for got, want in zip(ppo_amd.top_logits(x, 2), x.sort(dim=-1, descending=True, stable=True)):
        assert torch.equal(got, want[:, :2])


@pytest.mark.parametrize("A", [40, 3000, 40000, 300000])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_top_logits_ties_and_values_that_are_not_finite(dev, dtype, A):
    t, k = TYPES[dtype], 30
    x = torch.zeros(12, A)
    x[1] = -float("inf")
    x[1, ::A // 7] = 1.0                     # fewer finite ones than k
    x[2] = float("nan")
    x[3, A // 3] = float("nan")
    x[3, 5] = float("inf")
    x[4, 1::2] = -0.0                        # 0 and -0 are equal
    x[5] = torch.finfo(t).min
    x[5, -1] = torch.finfo(t).max
    x[6] = torch.arange(A) % 7
    x[7] = -torch.arange(A).float()
    x[8] = torch.arange(A).float()
    x[9] = -x[3]                             # a NaN with a sign, -inf
    x[10, A // 2:] = 1.0
    x[11] = torch.randn(A, generator=torch.Generator().manual_seed(1)) * 1e-38
    x = x.to(t)
    v, i = ppo_amd.top_logits(x.to(dev), k)
    wv, wi = ref.top(x.float(), k)
    assert torch.equal(i.cpu(), wi)
    assert torch.equal(v.cpu(), x.gather(1, wi)) or torch.isnan(x).any()
    same = (v.cpu() == x.gather(1, wi)) | torch.isnan(x.gather(1, wi))
    assert bool(same.all())


@pytest.mark.parametrize("A", [4100, 20001, 36000, 140001])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_top_logits_of_long_rows(dev, dtype, A):
    """Rows that a workgroup takes whole, in segments of one round to many, with ties in
    more segments than are looked at again."""
    g = torch.Generator(dev).manual_seed(A)
    x = torch.randn(520, A, device=dev, generator=g).to(TYPES[dtype])
    x[0] = 0.0
    x[1] = (torch.arange(A, device=dev) % 7).to(x.dtype)
    x[2] = -float("inf")
    x[2, :: A // 7] = 1.0
    x[3, 5::3] = float("nan")
    x[4] = torch.arange(A, device=dev).to(x.dtype)
    x[5, A // 2:] = 9.0
    want, at = x.float().sort(dim=-1, descending=True, stable=True)
    for k in (1, 20, 64, 130, 256):
        v, i = ppo_amd.top_logits(x, k)
        assert torch.equal(i, at[:, :k]), k
        assert torch.equal(torch.nan_to_num(v.float(), 7e7), torch.nan_to_num(want[:, :k], 7e7)), k


def test_top_logits_that_change_meanwhile(dev):
    """Logits written by another stream during the call: which are found is undefined,
    but every column lies in its row and every value is NaN or was there."""
    g = torch.Generator(dev).manual_seed(3)
    for R, A in ((2, 131072), (700, 4000)):
        x = torch.randn(R, A, device=dev, generator=g)
        noise = torch.randn(R, A, device=dev, generator=g)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        for _ in range(4):
            with torch.cuda.stream(side):
                for _ in range(8):
                    x.neg_()
                    x.copy_(noise)
            v, i = ppo_amd.top_logits(x, 40)
            torch.cuda.synchronize()
            assert bool(((i >= 0) & (i < A)).all())
        v, i = ppo_amd.top_logits(x, 40)
        assert torch.equal(v, x.gather(1, i)) and torch.equal(v, x.sort(1, descending=True).values[:, :40])


# Every layout with more rows than its workgroups take at once: rows, how often.
MANY_ROWS = [(18, 512, 300), (200, 512, 300), (400, 512, 300), (900, 4096, 36), (3000, 512, 81),
             (6000, 512, 81), (9000, 256, 36), (30000, 256, 36), (40000, 128, 9), (50304, 128, 9),
             (65536, 128, 9), (80000, 128, 6), (100000, 128, 6), (131072, 128, 6), (160001, 128, 6), (196600, 128, 6)]


@pytest.mark.parametrize("A, rows, times", MANY_ROWS)
@pytest.mark.parametrize("name", ["policy", "distillation"])
def test_many_rows(dev, name, A, rows, times):
    """The same rows `times` times, each left out every third time: gradients as of the
    rows by themselves, bit for bit, zeros for those left out, and sums that are a
    multiple (of terms of one sign; a sum in 64 bits, rounded once)."""
    t = torch.bfloat16
    g = torch.Generator(dev).manual_seed(A)
    rn = lambda *n: torch.randn(*n, generator=g, device=dev)  # noqa: E731
    x = (rn(rows, A) * 2).to(t)
    a = torch.randint(0, A, (rows,), generator=g, device=dev)
    if name == "policy":
        lp = ppo_amd.token_log_probs(x, a)
        rest = (lp + 0.3 * rn(rows), rn(rows).abs() + 0.1, lp + 0.2 * rn(rows))
        call = lambda x, a, rest, mask: ppo_amd.token_policy_loss(  # noqa: E731
            x, a, *rest, mask, kl_coef=0.1, entropy_coef=0.01, denominator=1000.0)
    else:
        K = min(32, A)
        rest = (rn(rows, K) * 2, rn(rows, A).topk(K).indices)  # (no id twice: no loss below 0)
        call = lambda x, a, rest, mask: (ppo_amd.distillation_loss(  # noqa: E731
            x, *rest, mask, denominator=1000.0), {})

    def run(x, a, rest, mask):
        x = x.detach().requires_grad_()
        loss, stats = call(x, a, rest, mask)
        return loss.detach(), stats, torch.autograd.grad(loss, [x])[0]

    loss, stats, d = run(x, a, rest, None)
    again = lambda v: v.repeat(times, *[1] * (v.dim() - 1))  # noqa: E731
    out = (torch.arange(rows, device=dev) + torch.arange(times, device=dev)[:, None]) % 3 == 0
    mask = ~out.view(-1)
    many, many_stats, dm = run(again(x), again(a), [again(v) for v in rest], mask)
    dm = dm.view(times, rows, A)
    for k in range(times):
        assert torch.equal(dm[k][~out[k]], d[~out[k]]), k
        assert not dm[k][out[k]].any(), k
    n = times * 2 / 3
    for one, all_ in ((stats[k], many_stats[k]) for k in ("policy", "kl", "entropy", "clipfrac")
                      if stats):
        assert abs(float(all_) - n * float(one)) <= 2 * U32 * n * abs(float(one))
    if not stats:
        assert abs(float(many) - n * float(loss)) <= 2 * U32 * n * abs(float(loss))


# --- whole calls -----------------------------------------------------------------------------------

def losses(dev, t, S=4, T=9, A=2500, K=12, seed=5):
    """name -> f(logits) over fixed inputs, and the logits."""
    c = policy_case(seed, t, S, T, A)
    _, teacher, ids, _ = distill_case(seed, t, t, S, T, A, K)
    v = lambda n: c[n].view(S, T).to(dev)  # noqa: E731
    a, old, adv, r, mask = v("a"), v("old"), v("adv"), v("ref"), c["mask"].to(dev)
    teacher, ids = teacher.view(S, T, K).to(dev), ids.view(S, T, K).to(dev)
    f = {
        "log_probs": lambda x: (ppo_amd.token_log_probs(x, a, mask) * adv).sum(),
        "entropy": lambda x: (ppo_amd.token_log_probs(x, a, mask, entropy=True)[1] * adv).sum(),
        "policy": lambda x: ppo_amd.token_policy_loss(x, a, old, adv, r, mask, kl_coef=0.1,
                                                      entropy_coef=0.01)[0],
        "preference": lambda x: ppo_amd.preference_loss(x, a, r, mask)[0],
        "distillation": lambda x: ppo_amd.distillation_loss(x, teacher, ids, mask),
    }
    return f, c["x"].view(S, T, A).to(dev)


@pytest.mark.parametrize("name", ["log_probs", "entropy", "policy", "preference", "distillation"])
def test_gradients_against_differences(dev, name):
    """Central differences of the loss along random directions in 32 bits: the loss's
    own rounding (1e-6 of it over a step of 1e-2) and the third derivative's share
    (step^2, of order one) stay below 1e-3 of the slope's scale."""
    f, x = losses(dev, torch.float32, S=4, T=3, A=60)
    f = f[name]
    xg = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(f(xg), [xg])
    g = torch.Generator(device=dev).manual_seed(3)
    for _ in range(4):
        v = torch.randn(x.shape, generator=g, device=dev)
        h = 1e-2
        with torch.no_grad():
            slope = (f(x + h * v).double() - f(x - h * v).double()) / (2 * h)
        want = (dx.double() * v.double()).sum()
        scale = float(dx.double().norm()) + 1e-3
        assert abs(float(slope - want)) <= 1e-2 * scale


class Declines:
    """A host path that leaves every call to the interpreted one."""

    def __init__(self, native):
        self.native = native

    def __getattr__(self, name):
        return self.native.capture_id if name == "capture_id" else lambda *args: None


@pytest.mark.parametrize("A, K", [(60, 12), (2500, 200), (40000, 7)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_interpreted_path_gives_the_same_bits(dev, monkeypatch, dtype, A, K):
    t = TYPES[dtype]
    f, x = losses(dev, t, A=A, K=K)

    def run():
        out = []
        for loss in f.values():
            xg = x.clone().requires_grad_()
            y = loss(xg)
            with torch.no_grad():
                out.append(loss(x))
            for up in (1.0, 0.25, 1.0):  # formed with the loss, anew, and anew again
                out += [y.detach(), *torch.autograd.grad(y * up, [xg], retain_graph=True)]
            with torch.autograd.graph.saved_tensors_hooks(lambda s: s.cpu(), lambda s: s.to(dev)):
                xg = x.clone().requires_grad_()
                out += torch.autograd.grad(loss(xg) * 0.25, [xg])
        a = torch.zeros(x.shape[:-1], dtype=torch.int32, device=dev)
        z = torch.linspace(-3, 0, a.numel(), device=dev).view(a.shape)
        _, stats = ppo_amd.token_policy_loss(x, a, z, z[:, 0].contiguous(), z, reduction="sequence",
                                             kl_coef=0.1, denominator=7.0)
        out += stats.values()
        _, stats = ppo_amd.preference_loss(x, a, None, None, 0.2, 0.1, 0.3, True, 0.9)
        out += [*stats.values(), *ppo_amd.top_logits(x, min(A, 50))]
        return out

    here = run()
    parameter = torch.nn.Parameter(x)
    y = f["policy"](parameter)
    assert torch.equal(y, f["policy"](x))
    native = _native()
    monkeypatch.setattr(tokens, "_native", lambda: Declines(native))
    there = run()
    assert len(here) == len(there) > 40
    for n, (p, q) in enumerate(zip(here, there)):
        assert p.dtype == q.dtype and p.shape == q.shape and torch.equal(p, q), n
    for wrong in (lambda s: s.double(), lambda s: s[:1], lambda s: s.cpu()):
        for loss in f.values():
            with torch.autograd.graph.saved_tensors_hooks(lambda s: s, wrong):
                xg = x.clone().requires_grad_()
                y = loss(xg)
                with pytest.raises(RuntimeError):
                    torch.autograd.grad(y, [xg])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_calls_repeat_their_bits(dev, dtype):
    f, x = losses(dev, TYPES[dtype])
    for name, loss in f.items():
        runs = []
        for _ in range(3):
            xg = x.clone().requires_grad_()
            y = loss(xg)
            runs.append((y.detach(), torch.autograd.grad(y, [xg])[0]))
        assert all(torch.equal(p, q) for r in runs[1:] for p, q in zip(r, runs[0])), name


def test_another_stream(dev):
    f, x = losses(dev, torch.bfloat16)
    side = torch.cuda.Stream(dev)
    for name, loss in f.items():
        xg = x.clone().requires_grad_()
        y = loss(xg)
        want = [y.detach(), torch.autograd.grad(y, [xg])[0]]
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            xs = x.clone().requires_grad_()
            y = loss(xs)
            got = [y.detach(), torch.autograd.grad(y, [xs])[0]]
            top = ppo_amd.top_logits(x, 7)
        torch.cuda.current_stream(dev).wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want)), name
        assert all(torch.equal(p, q) for p, q in zip(top, ppo_amd.top_logits(x, 7)))


@pytest.mark.parametrize("name", ["policy", "preference", "distillation"])
def test_gradients_are_the_callers(dev, name):
    """What a backward pass gives back may be changed, and any incoming gradient will do."""
    f, x = losses(dev, torch.float32, A=300)
    f = f[name]
    xg = x.clone().requires_grad_()
    y = f(xg)
    (d,) = torch.autograd.grad(y, [xg], retain_graph=True)
    want = d.clone()
    d.zero_()
    assert torch.equal(torch.autograd.grad(y, [xg])[0], want)
    y = f(xg)
    y.backward(retain_graph=True)
    y.backward()
    assert torch.allclose(xg.grad, 2 * want, rtol=8 * U32, atol=1e-12)
    y = f(xg)
    assert torch.allclose(torch.autograd.grad(y + y, [xg])[0], 2 * want, rtol=8 * U32, atol=1e-12)
    for s in (0.0, -1.0):
        (d,) = torch.autograd.grad(f(xg) * s, [xg])
        assert torch.allclose(d, s * want, rtol=8 * U32, atol=1e-12)
    live = want.abs().sum(-1) > 0
    (d,) = torch.autograd.grad(f(xg) * float("nan"), [xg])
    assert torch.isnan(d[live]).all() and not d[~losses_mask(dev, x)].any()
    with torch.inference_mode():
        assert torch.equal(f(x * 1.0), f(x))


def losses_mask(dev, x, seed=5):
    S, T, A = x.shape
    return policy_case(seed, x.dtype, S, T, A)["mask"].to(dev)


def test_calls_at_once(dev):
    """Threads with a stream each, all operators forward and back, and graphs of two
    losses that replay side by side."""
    f, x = losses(dev, torch.bfloat16, S=6, T=20, A=9000, K=20)

    def run():
        out = []
        for loss in f.values():
            xg = x.clone().requires_grad_()
            y = loss(xg)
            out += [y.detach(), *torch.autograd.grad(y, [xg])]
        return [*out, *ppo_amd.top_logits(x, 30)]

    want = run()
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(8):
                got = run()
                torch.cuda.current_stream().synchronize()
                wrong.extend(n for n, (p, q) in enumerate(zip(got, want)) if not torch.equal(p, q))
            wrong.append(None)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [None] * 3
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], []
    for name in ("policy", "distillation"):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            xg = x.clone().requires_grad_()
            torch.autograd.grad(f[name](xg), [xg])
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                y = f[name](xg)
                outs.append((y, torch.autograd.grad(y, [xg])[0]))
        graphs.append(graph)
        streams.append(stream)
    names = list(f)
    for _ in range(4):
        for y, d in outs:
            y.detach().fill_(7.0)
            d.fill_(7.0)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for name, (y, d) in zip(("policy", "distillation"), outs):
            n = 2 * names.index(name)
            assert torch.equal(y.detach(), want[n]) and torch.equal(d, want[n + 1])


@pytest.mark.parametrize("A", [60, 2500, 30000])
@pytest.mark.parametrize("name", ["log_probs", "policy", "preference", "distillation"])
def test_graph_replays(dev, name, A):
    """A captured pass, replayed on new logits and new incoming gradients between eager
    ones; two graphs replayed in turn share no scratch."""
    S, T = (4, 9) if A < 10000 else (2, 33)
    f, x0 = losses(dev, torch.bfloat16, S, T, A)
    f = f[name]
    side = torch.cuda.Stream(dev)
    graphs = []
    for k in range(2):
        x = x0.clone().requires_grad_()
        up = torch.ones((), device=dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            for _ in range(2):
                y = f(x)
                torch.autograd.grad(y, [x], up)
        del y
        torch.cuda.current_stream(dev).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = f(x)
            (dx,) = torch.autograd.grad(y, [x], up)
            y = y.detach()
        graphs.append((graph, x, up, y, dx))
    for step, scale in enumerate((1.0, 1.0, 2.0, 1.0, -3.0, 1.0)):
        wants = []
        for k, (graph, x, up, y, dx) in enumerate(graphs):
            fresh = torch.roll(x0, step + 3 * k, 0)
            with torch.no_grad():
                x.copy_(fresh)
            up.fill_(scale)
            graph.replay()
            xe = fresh.clone().requires_grad_()
            ye = f(xe)
            wants.append((ye.detach(), torch.autograd.grad(ye, [xe], up.clone())[0]))
        torch.cuda.synchronize(dev)
        for (graph, x, up, y, dx), (ye, de) in zip(graphs, wants):
            assert torch.equal(y, ye) and torch.equal(dx, de)


@pytest.mark.parametrize("name", ["policy", "distillation"])
def test_captured_backward_of_an_eager_forward(dev, name):
    """Its replays outnumber the forward's: each forms the gradient from the logits.
    (The policy's bits are the forward pass's own.  A distilled row's entries are summed
    over as many lanes as the row has in one pass and over a wave in the other: each
    within 12 additions, 24 operations and 3 t <= 90 roundings of w (p - q), whose size
    the largest element bounds.)"""
    f, x0 = losses(dev, torch.float32)
    side = torch.cuda.Stream(dev)
    x = x0.clone().requires_grad_()
    up = torch.ones((), device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        torch.autograd.grad(f[name](x), [x], up)
        y = f[name](x)
        graph = torch.cuda.CUDAGraph()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            (dx,) = torch.autograd.grad(y, [x], up, retain_graph=True)
    torch.cuda.current_stream(dev).wait_stream(side)
    for scale in (1.0, 2.0, 1.0):
        up.fill_(scale)
        graph.replay()
        xe = x0.clone().requires_grad_()
        (want,) = torch.autograd.grad(f[name](xe), [xe], up.clone())
        if name == "policy":
            assert torch.equal(dx, want)
        assert torch.allclose(dx, want, rtol=256 * U32, atol=256 * U32 * float(want.abs().max()))
        dx.add_(1.0)  # (a caller's own write into the gradient does not last)


def test_differentiated_once(dev):
    f, x = losses(dev, torch.float32)
    for name, loss in f.items():
        xg = x.clone().requires_grad_()
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(loss(xg), [xg], create_graph=True)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="teacher"):
        ppo_amd.distillation_loss(x.detach(), x[..., :3].contiguous(),
                                  torch.zeros(4, 9, 3, dtype=torch.int64, device=dev))


def test_saved_tensor_hooks(dev):
    """Hooks that move saved tensors work; ones that hand back something else raise."""
    f, x = losses(dev, torch.bfloat16)
    for name, loss in f.items():
        xg = x.clone().requires_grad_()
        (want,) = torch.autograd.grad(loss(xg) * 2.0, [xg])
        with torch.autograd.graph.save_on_cpu():
            y = loss(xg) * 2.0
        (got,) = torch.autograd.grad(y, [xg])
        assert torch.equal(got, want), name
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[..., :1]):
            y = loss(xg)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y * 2.0, [xg])


def test_logits_changed_in_place_before_the_backward_pass(dev):
    f, x = losses(dev, torch.float32)
    for name, loss in f.items():
        xg = x.clone().requires_grad_()
        z = xg + 0.0
        y = loss(z)
        z.detach().add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad(y, [xg])


def test_rows_beyond_32_bits(dev):
    """Offsets past 2^31 elements: the last rows equal a small call's, bit for bit."""
    A, t = 131072, torch.bfloat16
    R = (1 << 31) // A + 70
    x = ((torch.arange(A, device=dev) % 8191) * 1e-3).to(t).expand(R, A).contiguous()
    tail = 66
    x[-tail:] = torch.randn(tail, A, device=dev, generator=torch.Generator(dev).manual_seed(2)) * 2
    a = torch.randint(0, A, (R,), device=dev)
    old = torch.full((R,), -12.0, device=dev)
    small = x[-tail:].clone()
    lp, H = ppo_amd.token_log_probs(x, a, entropy=True)
    lps, Hs = ppo_amd.token_log_probs(small, a[-tail:].clone(), entropy=True)
    # (few rows are cut into parts: the sums' order differs)
    assert torch.allclose(lp[-tail:], lps, rtol=0, atol=400 * U32)
    assert torch.allclose(H[-tail:], Hs, rtol=0, atol=400 * U32 * 12)
    kw = dict(entropy_coef=0.01, denominator=100.0)
    x.requires_grad_()
    (dx,) = torch.autograd.grad(ppo_amd.token_policy_loss(x, a, old, old, **kw)[0], [x])
    small.requires_grad_()
    (ds,) = torch.autograd.grad(ppo_amd.token_policy_loss(
        small, a[-tail:].clone(), old[-tail:].clone(), old[-tail:].clone(), **kw)[0], [small])
    assert torch.equal(dx[-tail:], ds)
    v, i = ppo_amd.top_logits(x.detach()[-tail:], 20)
    vl, il = ppo_amd.top_logits(x.detach(), 20)
    assert torch.equal(vl[-tail:], v) and torch.equal(il[-tail:], i)
    del dx, x


def test_a_training_run(dev):
    """The operators as a program uses them: a teacher's top logits are distilled into
    a student, which acts, is updated by the policy loss against itself as the
    reference, and by preferences; every gradient reaches the parameters and agrees
    with the plain form's."""
    torch.manual_seed(4)
    S, T, D, A, K = 4, 12, 32, 1500, 20
    feats = torch.randn(S, T, D, device=dev)
    teacher = torch.nn.Linear(D, A, device=dev)
    student = torch.nn.Linear(D, A, device=dev)
    mask = torch.rand(S, T, device=dev) < 0.8
    mask[0, 0] = mask[2, 0] = True
    with torch.no_grad():
        v, i = ppo_amd.top_logits(teacher(feats), K)
        actions = torch.distributions.Categorical(logits=student(feats)).sample()
        old = ppo_amd.token_log_probs(student(feats), actions, mask)
    with torch.no_grad():
        student.weight.add_(0.02 * torch.randn_like(student.weight))
    adv = torch.randn(S, device=dev)
    keep = mask.double()
    w = keep / keep.sum()

    def plain(x):
        ls = torch.log_softmax(x.double(), -1)
        lp = ls.gather(-1, actions[..., None])[..., 0]
        q = torch.softmax(v.double(), -1)
        distill = (w * (q * (q.log() - ls.gather(-1, i))).sum(-1)).sum()
        ratio = torch.exp((lp - old) * keep)
        ad = adv.double()[:, None]
        d = (old - lp) * keep
        policy = (w * (-torch.minimum(ratio * ad, ratio.clamp(0.8, 1.2) * ad)
                       + 0.05 * (torch.exp(d) - d - 1))).sum()
        rel = ((lp - old) * keep).sum(1)
        m = 0.5 * (rel[:2] - rel[2:])
        return distill + policy - torch.nn.functional.logsigmoid(m).mean()

    def ours(x):
        return (ppo_amd.distillation_loss(x, v, i, mask)
                + ppo_amd.token_policy_loss(x, actions, old, adv, old, mask, kl_coef=0.05)[0]
                + ppo_amd.preference_loss(x, actions, old, mask, beta=0.5)[0])

    params = list(student.parameters())
    got = torch.autograd.grad(ours(student(feats)), params)
    want = torch.autograd.grad(plain(student(feats)), params)
    for p, q in zip(got, want):
        # (three gradients of 32 bits, each within some hundred u of its size, through
        # one 32-bit product)
        assert float((p - q).norm()) <= 1e-5 * float(q.norm())


# --- refusals -------------------------------------------------------------------------------------

def test_refusals(dev):
    x = torch.randn(2, 4, 30, device=dev)
    a = torch.zeros(2, 4, dtype=torch.int64, device=dev)
    z = torch.zeros(2, 4, device=dev)
    lp, pl, pr, di, top = (ppo_amd.token_log_probs, ppo_amd.token_policy_loss,
                           ppo_amd.preference_loss, ppo_amd.distillation_loss, ppo_amd.top_logits)
    values = [
        lambda: lp(x.transpose(0, 1), a), lambda: lp(x, a[:, :3].contiguous()), lambda: lp(x, a.t()),
        lambda: lp(x, a, temperature=0.0), lambda: lp(x, a, temperature=float("inf")),
        lambda: lp(x, a, mask=z.bool()[:1].contiguous()), lambda: lp(x[..., :0].contiguous(), a),
        lambda: pl(x, a, z[:1].contiguous(), z), lambda: pl(x, a, z, z[0].contiguous()),
        lambda: pl(x, a, z, z, z[:1].contiguous()), lambda: pl(x, a, z, z, clip_low=-0.1),
        lambda: pl(x, a, z, z, kl_coef=0.1), lambda: pl(x, a, z, z, reduction="mean"),
        lambda: pl(x, a, z, z, denominator=0.0), lambda: pl(x, a, z, z, grad_scale=0.0),
        lambda: pl(x, a, z, z, entropy_coef=float("nan")),
        lambda: pr(x[0], a[0], z[0]), lambda: pr(x[:1], a[:1], z[:1]),
        lambda: pr(x, a, z, label_smoothing=1.1), lambda: pr(x, a, z, beta=float("inf")),
        lambda: di(x, x[..., :3].contiguous(), a), lambda: di(x, x[:1, :, :3].contiguous(), a),
        lambda: di(x, x[..., :0].contiguous(), a[..., None][..., :0].contiguous()),
        lambda: top(x, 0), lambda: top(x, 31), lambda: top(torch.randn(2, 300, device=dev), 257),
    ]
    for n, bad in enumerate(values):
        with pytest.raises(ValueError):
            bad()
            pytest.fail(str(n))
    types = [
        lambda: lp(x.double(), a), lambda: lp(x, a.float()), lambda: lp(x, a, mask=z),
        lambda: pl(x, a, z.double(), z), lambda: pl(x, a, z, z.half()),
        lambda: di(x, x[..., :3].double().contiguous(), a[..., None].expand(2, 4, 3).contiguous()),
        lambda: di(x, x[..., :3].contiguous(), x[..., :3].contiguous()),
        lambda: top(x, 2.0), lambda: top(x, True), lambda: lp(None, a),
    ]
    for n, bad in enumerate(types):
        with pytest.raises(TypeError):
            bad()
            pytest.fail(str(n))
    for bad in (lambda: lp(x.cpu(), a), lambda: lp(x, a.cpu()), lambda: pl(x, a, z, z.cpu())):
        with pytest.raises(RuntimeError, match="no CPU fallback|expected"):
            bad()
    with pytest.raises(_lib.PPOLibraryError):
        di(x.expand(2, 4, 30), torch.randn(2, 4, 257, device=dev),
           torch.zeros(2, 4, 257, dtype=torch.int64, device=dev))
    with pytest.raises(_lib.PPOLibraryError):
        top(torch.zeros(1, (1 << 22) + 1, dtype=torch.float16, device=dev), 2)
    assert tokens.top_logits(x[:0], 3)[0].shape == (0, 4, 3)


def test_constants_that_ask_for_a_gradient(dev):
    """Operands in which a loss has no gradient are refused where they ask for one, in
    either direction, and taken where nothing is differentiated."""
    x = torch.randn(2, 4, 30, device=dev, requires_grad=True)
    a = torch.zeros(2, 4, dtype=torch.int64, device=dev)
    z = torch.zeros(2, 4, device=dev)
    one = z[:, 0].contiguous()
    pl, pr = ppo_amd.token_policy_loss, ppo_amd.preference_loss
    for name, call, v in (("old_log_probs", lambda v: pl(x, a, v, z), z),
                          ("advantages", lambda v: pl(x, a, z, v), z),
                          ("advantages", lambda v: pl(x, a, z, v), one),
                          ("ref_log_probs", lambda v: pl(x, a, z, z, v, kl_coef=0.1), z),
                          ("ref_log_probs", lambda v: pr(x, a, v), z)):
        wants = v.clone().requires_grad_()
        with pytest.raises(RuntimeError, match=f"no gradient in {name}"):
            call(wants)
        with torch.no_grad():
            quiet = call(wants)[0]
        assert torch.equal(quiet, call(wants.detach())[0].detach())
        with fwd_ad.dual_level(), pytest.raises(RuntimeError, match=f"no gradient in {name}"):
            call(fwd_ad.make_dual(v, v))


def test_numbers_that_fp32_does_not_hold(dev):
    x = torch.randn(2, 4, 30, device=dev)
    a = torch.zeros(2, 4, dtype=torch.int64, device=dev)
    z, m = torch.zeros(2, 4, device=dev), torch.ones(2, 4, dtype=torch.bool, device=dev)
    top = ppo_amd.top_logits(x, 3)
    for kw in (dict(denominator=1e46), dict(denominator=1e-46), dict(grad_scale=1e39),
               dict(grad_scale=1e-50)):
        for mask in (None, m):
            with pytest.raises(ValueError, match="must be in"):
                ppo_amd.token_policy_loss(x, a, z, z, mask=mask, **kw)
            with pytest.raises(ValueError, match="must be in"):
                ppo_amd.distillation_loss(x, *top, mask, **kw)
    for kw in (dict(kl_coef=1e39), dict(entropy_coef=-1e39)):
        with pytest.raises(ValueError, match="_coef must be finite"):
            ppo_amd.token_policy_loss(x, a, z, z, z, **kw)
    one = float(ppo_amd.token_policy_loss(x, a, z, z + 1, mask=m, denominator=1.0)[0])
    for den in (1e-30, 1e-20, 1e20, 1e30):
        got = float(ppo_amd.token_policy_loss(x, a, z, z + 1, mask=m, denominator=den)[0])
        assert abs(got * den - one) <= 4 * U32 * abs(one)
