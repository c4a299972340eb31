"""The preference and the policy objective against their formulas in 64 bits.

u = 2^-24. The preference loss is computed in 64 bits and rounded once: loss and rewards are off by
u relative (plus the 64-bit sums' own 2^-50 of their terms); a gradient is a coefficient rounded
to fp32 (u), times g (u), rounded to its type. A policy term is r A with r = e^l in fp32: 4 u for
the function, u |l| for its argument, 2 u for the products; e^d - d - 1 and e^d - 1 are good to
16 u of themselves; the 64-bit sum of the terms is rounded once."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def draw(dev, n, s, dtype, seed, holes=True):
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    logp = (-randn(n, s).abs()).to(dtype)
    mask = torch.rand(n, s, device=dev, generator=g) < 0.7
    if holes and n > 1:
        mask[0] = False                                  # a row without a token
        mask[1] = False
        mask[1, -1] = True                               # and one with a single one
    return logp, mask, randn


# ---------------------------------------------------------------------------------------------
# preference


def preference64(x, mask, ref, beta, kind, eps, margin, normal, denom):
    """(loss, rewards) of 64-bit log-probabilities, differentiable."""
    m = torch.ones_like(x, dtype=torch.bool) if mask is None else mask
    d = x - ref.double() if ref is not None and ref.dim() == 2 else x
    s = torch.where(m, d, torch.zeros_like(d)).sum(1)
    if normal:
        s = s / m.sum(1).clamp(min=1)
    if ref is not None and ref.dim() == 1:
        s = s - ref.double()
    p = x.shape[0] // 2
    u = beta * (s[:p] - s[p:]) - margin
    if kind == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        loss = -(1 - eps) * ls(u) - eps * ls(-u)
    elif kind == "hinge":
        loss = torch.relu(1 - u)
    else:
        loss = (u / beta - 1 / (2 * beta)) ** 2
    return loss.sum() / (p if denom is None else denom), beta * s


def check_preference(logp, mask, ref, beta=0.1, kind="sigmoid", eps=0.0, margin=0.0,
                     normal=False, denom=None, up=1.0):
    from hackathon_b200.preference import preference_loss
    leaf = logp.detach().requires_grad_()
    loss, step = preference_loss(leaf, mask, ref, beta, kind, eps, margin, normal, denom)
    (grad,) = torch.autograd.grad(loss, leaf, torch.full_like(loss, up))
    live = mask if mask is not None else torch.ones_like(logp, dtype=torch.bool)
    keep = live != 0
    x = torch.where(keep, logp.detach().double(), 0.0).requires_grad_()
    r = ref if ref is None or ref.dim() == 1 else torch.where(keep, ref.double(), 0.0)
    want, rewards = preference64(x, keep, r, beta, kind, eps, margin, normal,
                                 None if denom is None else float(denom))
    (wg,) = torch.autograd.grad(want, x, torch.full_like(want, up))
    size = beta * (x.detach().abs().sum(1) + (r.double().abs().reshape(len(x), -1).sum(1)
                                              if r is not None else 0.0))
    tiny = 2.0 ** -45
    assert loss.dtype == torch.float32 and grad.dtype == logp.dtype and grad.is_contiguous()
    # the loss's slope in each reward is at most 1 (or 2 |D - 1 / 2 beta| / beta)
    steep = float(1 + 2 * size.max() / beta ** 2 + 1 / beta ** 2)
    value = float(want.detach())
    assert abs(float(loss.detach()) - value) <= 2 * U * abs(value) \
        + tiny * steep * float(size.max())
    got = torch.cat([step.chosen_rewards, step.rejected_rewards]).double()
    assert bool(((got - rewards.detach()).abs() <= 2 * U * rewards.detach().abs()
                 + tiny * size).all())
    tol = wg.abs() * (3 * U + HALF[logp.dtype]) + torch.finfo(logp.dtype).smallest_normal \
        + tiny * steep * abs(up)
    assert bool(((grad.double() - wg).abs() <= tol).all())
    assert not grad[~keep].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,s", [(2, 1), (2, 2), (6, 5), (4, 2047), (8, 2048), (2, 2049),
                                 (66, 33), (2, 70001), (2050, 3), (64, 5000)])
def test_preference_shapes_and_types(cuda, n, s, dtype):
    logp, mask, randn = draw(cuda, n, s, dtype, n + s)
    check_preference(logp, mask, (logp.float() + 0.1 * randn(n, s)).to(dtype))
    check_preference(logp, None, None, normal=True)


@pytest.mark.parametrize("kind,eps,margin", [("sigmoid", 0.0, 0.0), ("sigmoid", 0.2, 0.5),
                                             ("hinge", 0.0, 0.0), ("hinge", 0.0, -0.4),
                                             ("ipo", 0.0, 0.0)])
@pytest.mark.parametrize("normal", [False, True])
@pytest.mark.parametrize("ref", ["none", "token", "row"])
def test_preference_kinds(cuda, kind, eps, margin, normal, ref):
    logp, mask, randn = draw(cuda, 10, 300, torch.float32, 5)
    r = {"none": None, "token": logp + 0.3 * randn(10, 300), "row": -20 * randn(10).abs()}[ref]
    for beta in (0.01, 0.1, 2.0):
        check_preference(logp, mask, r, beta, kind, eps, margin, normal)
    check_preference(logp, mask, r, 0.1, kind, eps, margin, normal, denom=7.5, up=-3.0)
    check_preference(logp, mask, r, 0.1, kind, eps, margin, normal,
                     denom=torch.tensor(3, device=cuda))


def test_preference_masked_places_may_hold_anything(cuda):
    from hackathon_b200.preference import preference_loss
    logp, mask, randn = draw(cuda, 8, 100, torch.float32, 6)
    ref = logp + randn(8, 100)
    want = preference_loss(logp, mask, ref)[0]
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min):
        x = logp.masked_fill(~mask, bad).requires_grad_()
        loss, _ = preference_loss(x, mask, ref.masked_fill(~mask, -bad))
        (g,) = torch.autograd.grad(loss, x)
        assert torch.equal(loss, want) and torch.isfinite(g).all() and not g[~mask].any()
    for other in (mask.to(torch.uint8) * 3, mask.long(), mask.float(), mask.t().contiguous().t()):
        assert torch.equal(preference_loss(logp, other, ref)[0], want)


def test_preference_extremes(cuda):
    """Pairs far apart, both rows empty, and log-probabilities of -inf that count."""
    from hackathon_b200.preference import preference_loss
    x = torch.tensor([[-1e6], [0.0], [0.0], [-1e6]], device=cuda, requires_grad=True)
    loss, _ = preference_loss(x, beta=1.0)
    (g,) = torch.autograd.grad(loss, x)
    assert abs(float(loss.detach()) - 5e5) <= 2 * U * 5e5
    assert g.flatten().tolist() == [-0.5, 0.0, 0.5, 0.0]
    mask = torch.zeros(4, 1, dtype=torch.bool, device=cuda)
    loss, step = preference_loss(x, mask, beta=1.0, length_normalized=True)
    assert abs(float(loss) - math.log(2.0)) <= 2 * U
    assert not step.margins.any()
    (g,) = torch.autograd.grad(loss, x)
    assert not g.any()
    y = torch.tensor([[-math.inf], [-2.0]], device=cuda)
    assert float(preference_loss(y)[0]) == math.inf
    assert float(preference_loss(y.flip(0))[0]) == 0.0
    for kind in ("sigmoid", "hinge", "ipo"):
        z = torch.tensor([[math.nan], [-2.0]], device=cuda, requires_grad=True)
        loss, _ = preference_loss(z, loss_type=kind)
        assert math.isnan(float(loss))
        assert torch.isnan(torch.autograd.grad(loss, z)[0]).all()


def test_long_sums_keep_small_differences(cuda):
    """Two sums of -3e5 that differ by 1e-2: lost in fp32 sums, kept here."""
    from hackathon_b200.preference import preference_loss
    x = torch.full((2, 100_000), -3.0, device=cuda)
    x[0, 77] = -2.99
    want = float(x[0, 77].double()) + 3.0
    _, step = preference_loss(x, beta=1.0)
    got = float(step.chosen_rewards.double() - step.rejected_rewards.double())
    assert abs(got - want) <= 3e5 * 2 * U               # each reward is rounded to fp32
    loss, _ = preference_loss(x, beta=1.0)
    assert abs(float(loss) - math.log1p(math.exp(-want))) <= 2 * U
    # reference sums in fp64 keep as much: a pair that differs from its reference by 1e-2 each
    ref = x.double().sum(1) + torch.tensor([1e-2, -1e-2], dtype=torch.float64, device=cuda)
    loss, step = preference_loss(x, None, ref, beta=1.0)
    rewards = [float(step.chosen_rewards), float(step.rejected_rewards)]
    assert abs(rewards[0] + 1e-2) <= 2 * U and abs(rewards[1] - 1e-2) <= 2 * U
    assert abs(float(loss) - math.log1p(math.exp(2e-2))) <= 2 * U
    check_preference(x, None, ref, beta=1.0)


def test_preference_against_differences(cuda):
    logp, mask, randn = draw(cuda, 6, 20, torch.float32, 11)
    ref = logp + randn(6, 20)
    d = randn(6, 20).double()
    from hackathon_b200.preference import preference_loss
    for kind in ("sigmoid", "ipo"):
        leaf = logp.detach().requires_grad_()
        (g,) = torch.autograd.grad(preference_loss(leaf, mask, ref, 0.5, kind)[0], leaf)
        h = 1e-4

        def f(x):
            return preference64(x, mask, ref, 0.5, kind, 0.0, 0.0, False, None)[0]

        want = float((f(logp.double() + h * d) - f(logp.double() - h * d)) / (2 * h))
        got = float((g.double() * d).sum())
        # 64-bit differences: rounding 2^-52 |f| / h, truncation h^2 times the third derivative
        assert abs(got - want) <= 4 * U * float((g.double() * d).abs().sum()) + 1e-6


# ---------------------------------------------------------------------------------------------
# policy


def check_policy(logp, old, adv, mask, ref, low=0.2, high=None, delta=None, kl=0.0,
                 reduction="token", denom=None, up=1.0):
    from hackathon_b200.policy import policy_loss
    leaf = logp.detach().requires_grad_()
    loss, step = policy_loss(leaf, old, adv, mask, ref, low, high, delta, kl, reduction, denom)
    (grad,) = torch.autograd.grad(loss, leaf, torch.full_like(loss, up))
    keep = mask != 0 if mask is not None else torch.ones_like(logp, dtype=torch.bool)
    x = logp.detach().double()
    a = (adv if adv.dim() == 2 else adv[:, None]).double().expand_as(x)
    l = x - old.double() if old is not None else torch.zeros_like(x)
    r = l.exp()
    hi = low if high is None else high
    first = r.clamp(max=delta) if delta else r
    term = -torch.minimum(first * a, r.clamp(1 - low, 1 + hi) * a)
    inside = (l >= math.log1p(-low) if low < 1 else torch.ones_like(keep)) & (l <= math.log1p(hi))
    live = inside | ((r < 1) & ~inside & (a > 0)) | ((r > 1) & ~inside & (a < 0))
    if delta:
        live = live & (l <= math.log(delta))
    g = torch.where(live, -a * r, 0.0)
    t_term = U * (l.abs() + 8) * torch.maximum(first, torch.full_like(r, 1 + hi)) * a.abs()
    t_g = torch.where(live, U * (l.abs() + 8) * g.abs(), 0.0)
    n = keep.sum(1).double()
    tokens = n.sum().clamp(min=1)
    if ref is not None:
        d = ref.double() - x
        k3 = torch.expm1(d) - d
        em1 = torch.expm1(d)
        term, g = term + kl * k3, g - kl * em1
        # below |d| = 1/2 relative to itself, above it to its two parts
        t_k3 = U * 16 * torch.where(d.abs() < 0.5, k3, em1.abs() + d.abs() * (1 + em1.abs()))
        t_term = t_term + abs(kl) * (t_k3 + 2 * U * k3.abs())
        t_g = t_g + abs(kl) * (U * (16 + d.abs()) * em1.abs() + U * d.abs())
        want_kl = torch.where(keep, k3, 0.0).sum() / tokens
        t_kl = torch.where(keep, t_k3, 0.0).sum() / tokens + 2 * U * want_kl
        assert abs(float(step.kl) - float(want_kl)) <= float(t_kl)
    else:
        assert float(step.kl) == 0.0
    if reduction == "token":
        w = torch.full_like(n, 1.0 / float(tokens if denom is None else denom))
    else:
        w = 1.0 / (n.clamp(min=1) * float(len(n) if denom is None else denom))
    w = w[:, None]
    want = (torch.where(keep, term, 0.0) * w).sum()
    tol = (torch.where(keep, t_term, 0.0) * w).sum() + 2 * U * want.abs() \
        + (torch.where(keep, term.abs(), 0.0) * w).sum() * U
    assert abs(float(loss) - float(want)) <= float(tol), (float(loss), float(want), float(tol))
    wg = torch.where(keep, g, 0.0) * w * up
    t_grad = torch.where(keep, t_g, 0.0) * w * abs(up) + wg.abs() * 4 * U
    t_grad = t_grad + HALF[logp.dtype] * (wg.abs() + t_grad) \
        + torch.finfo(logp.dtype).smallest_normal
    assert grad.dtype == logp.dtype and grad.is_contiguous()
    assert bool(((grad.double() - wg).abs() <= t_grad).all())
    assert not grad[~keep].any()
    assert float(step.tokens) == float(n.sum())
    below, above = ~inside & (r < 1), ~inside & (r > 1)
    for got, cnt in ((step.clipped_low, keep & below & (a < 0)),
                     (step.clipped_high, keep & above & (a > 0))):
        assert abs(float(got) - float(cnt.sum() / tokens)) <= U


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,s", [(1, 1), (1, 2), (3, 5), (4, 2047), (5, 2048), (1, 2049), (33, 65),
                                 (2, 70001), (1100, 3), (16, 8000)])
def test_policy_shapes_and_types(cuda, n, s, dtype):
    logp, mask, randn = draw(cuda, n, s, dtype, n + s)
    old = (logp.float() + 0.2 * randn(n, s)).to(dtype)
    ref = (logp.float() + 0.3 * randn(n, s)).to(dtype)
    check_policy(logp, old, randn(n), mask, ref, kl=0.05)
    check_policy(logp, old, randn(n, s), mask, None, reduction="sequence")


@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("low,high,delta,kl", [(0.2, None, None, 0.0), (0.2, 0.28, None, 0.04),
                                               (0.0, 0.0, None, 0.01), (1.0, 3.0, 5.0, 0.0),
                                               (0.2, 0.2, 1.5, 1.0), (0.1, 0.3, 10.0, -0.01)])
def test_policy_kinds(cuda, reduction, low, high, delta, kl):
    logp, mask, randn = draw(cuda, 12, 257, torch.float32, 21)
    old, ref = logp + 0.6 * randn(12, 257), logp + randn(12, 257)
    ref[3] = logp[3] + 1e-4 * randn(257)                 # where e^d - d - 1 cancels
    ref[4] = logp[4]
    for adv in (randn(12), randn(12, 257), torch.zeros(12, device=cuda)):
        check_policy(logp, old, adv, mask, ref if kl else None, low, high, delta, kl, reduction)
        check_policy(logp, None, adv, None, ref if kl else None, low, high, delta, kl, reduction,
                     denom=100.0, up=2.5)
    check_policy(logp, old, randn(12), mask, ref, low, high, delta, kl, reduction,
                 denom=torch.tensor(17, device=cuda))
    check_policy(logp, old, randn(12).expand(257, 12).t(), mask, ref, low, high, delta, kl,
                 reduction)
    check_policy(logp, old, randn(24)[::2], mask, ref, low, high, delta, kl, reduction)


def test_policy_at_the_borders(cuda):
    """Ratios one fp32 step around the borders take the side their 64-bit logarithm is on."""
    from hackathon_b200.policy import policy_loss
    edge = torch.tensor([math.log(0.8), math.log(1.2)], dtype=torch.float64)
    near = torch.stack([torch.nextafter(edge.float(), torch.tensor(s * 10.0))
                        for s in (-1, 1)] + [edge.float()]).flatten()
    x = near.to(cuda)[None].repeat(2, 1)
    adv = torch.tensor([1.0, -1.0], device=cuda)
    leaf = x.clone().requires_grad_()
    loss, _ = policy_loss(leaf, torch.zeros_like(x), adv)
    (g,) = torch.autograd.grad(loss, leaf)
    l = x.double()
    inside = (l >= math.log1p(-0.2)) & (l <= math.log1p(0.2))
    live = inside | ((l < 0) & (adv[:, None] > 0)) | ((l > 0) & (adv[:, None] < 0))
    assert torch.equal(g != 0, live)


def test_policy_masked_places_may_hold_anything(cuda):
    from hackathon_b200.policy import policy_loss
    logp, mask, randn = draw(cuda, 8, 100, torch.float32, 6)
    old, ref, adv = logp + 0.2 * randn(8, 100), logp + randn(8, 100), randn(8, 100)
    for reduction in ("token", "sequence"):
        want = policy_loss(logp, old, adv, mask, ref, kl_coef=0.1, reduction=reduction)[0]
        for bad in (math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min):
            x = logp.masked_fill(~mask, bad).requires_grad_()
            loss, step = policy_loss(x, old.masked_fill(~mask, bad), adv.masked_fill(~mask, bad),
                                     mask, ref.masked_fill(~mask, -bad), kl_coef=0.1,
                                     reduction=reduction)
            (g,) = torch.autograd.grad(loss, x)
            assert torch.equal(loss, want) and torch.isfinite(g).all() and not g[~mask].any()
            assert torch.isfinite(step.state[:4]).all()
        none = torch.zeros_like(mask)
        x = logp.detach().requires_grad_()
        loss, step = policy_loss(x, old, adv, none, ref, kl_coef=0.1, reduction=reduction)
        (g,) = torch.autograd.grad(loss, x)
        assert float(loss) == 0.0 and not g.any() and float(step.tokens) == 0.0


def test_policy_infinite_ratios(cuda):
    """A ratio beyond fp32: infinite where it counts, held where the clip holds it."""
    from hackathon_b200.policy import policy_loss
    x = torch.tensor([[0.0], [0.0], [0.0], [0.0]], device=cuda, requires_grad=True)
    old = torch.tensor([[-200.0], [-200.0], [-200.0], [200.0]], device=cuda)
    adv = torch.tensor([1.0, -1.0, 0.0, 1.0], device=cuda)
    one = [policy_loss(x[k:k + 1], old[k:k + 1], adv[k:k + 1])[0] for k in range(4)]
    assert abs(float(one[0]) + 1.2) <= 2 * U * 1.2 + U
    assert float(one[1]) == math.inf and float(one[2]) == 0.0 and abs(float(one[3])) < 1e-30
    (g,) = torch.autograd.grad(one[0], x, retain_graph=True)
    assert not g.any()
    loss, _ = policy_loss(x[1:2], old[1:2], adv[1:2], delta=4.0)
    assert float(loss) == 4.0
    (g,) = torch.autograd.grad(loss, x)
    assert not g.any()
    nan = torch.tensor([[math.nan]], device=cuda)
    assert math.isnan(float(policy_loss(nan, torch.zeros_like(nan), adv[:1])[0]))


def test_policy_against_differences(cuda):
    """Directions that cross no border: the 64-bit objective's difference quotient."""
    from hackathon_b200.policy import policy_loss
    logp, mask, randn = draw(cuda, 6, 30, torch.float32, 31)
    old = logp + 0.05 * randn(6, 30).clamp(-2, 2)
    ref, adv, d = logp + 0.5 * randn(6, 30), randn(6), randn(6, 30).double().clamp(-2, 2)
    leaf = logp.detach().requires_grad_()
    loss, _ = policy_loss(leaf, old, adv, mask, ref, kl_coef=0.3, reduction="sequence")
    (g,) = torch.autograd.grad(loss, leaf)

    def f(x):
        r = (x - old.double()).exp()
        k = ref.double() - x
        t = -torch.minimum(r * adv[:, None].double(),
                           r.clamp(0.8, 1.2) * adv[:, None].double()) + 0.3 * (k.exp() - k - 1)
        return (torch.where(mask, t, 0.0).sum(1) / mask.sum(1).clamp(min=1)).mean()

    h = 1e-4
    want = float((f(logp.double() + h * d) - f(logp.double() - h * d)) / (2 * h))
    got = float((g.double() * d).sum())
    assert abs(got - want) <= 20 * U * float((g.double() * d).abs().sum()) + 1e-6


def test_policy_far_references(cuda):
    """A reference so far away that e^d overflows: an infinite KL term where it counts, none at a
    coefficient of 0; a token impossible under the reference costs infinitely much."""
    from hackathon_b200.policy import policy_loss
    x = torch.tensor([[-200.0, -1.0]], device=cuda, requires_grad=True)
    one = torch.ones(1, device=cuda)
    far = torch.zeros(1, 2, device=cuda)
    loss, step = policy_loss(x, x.detach(), one, None, far, kl_coef=0.0)
    (g,) = torch.autograd.grad(loss, x)
    assert float(loss.detach()) == -1.0 and g.tolist() == [[-0.5, -0.5]]
    assert float(step.kl) == math.inf
    assert float(policy_loss(x, x.detach(), one, None, far, kl_coef=0.1)[0]) == math.inf
    never = torch.tensor([[-200.0, -math.inf]], device=cuda)
    assert float(policy_loss(x, x.detach(), one, None, never, kl_coef=0.1)[0]) == math.inf


# ---------------------------------------------------------------------------------------------
# both


def test_compiled_functions_trace_the_operators(cuda):
    """torch.compile sees the operators whole (no graph break) and gives the eager bits."""
    from hackathon_b200.logprobs import token_logprobs
    from hackathon_b200.policy import policy_loss
    from hackathon_b200.preference import preference_loss
    logp, mask, randn = draw(cuda, 6, 70, torch.float32, 81)
    old, adv = logp + 0.2 * randn(6, 70), randn(6)
    z, t = randn(6, 300), torch.arange(6, device=cuda)

    def objective(x, logits):
        a, _ = preference_loss(x, mask, old)
        b, _ = policy_loss(x, old, adv, mask, old, kl_coef=0.1)
        lp, en = token_logprobs(logits, t, 0.9, True)
        return a + b + lp.sum() - en.sum()

    def step(fn):
        x, logits = logp.clone().requires_grad_(), z.clone().requires_grad_()
        out = fn(x, logits)
        return (out.detach(), *torch.autograd.grad(out, (x, logits)))

    torch._dynamo.reset()
    want = step(objective)
    got = step(torch.compile(objective, backend="aot_eager", fullgraph=True))
    assert all(map(torch.equal, got, want))


@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_more_than_32_bits_of_tokens(cuda, kind):
    """2.2 billion tokens: the values past 2^31 count and get their gradients."""
    from hackathon_b200.policy import policy_loss
    from hackathon_b200.preference import preference_loss
    n, s = 2, (1 << 30) + (1 << 26) + 7
    x = torch.zeros(n, s, dtype=torch.bfloat16, device=cuda)
    mask = torch.zeros(n, s, dtype=torch.bool, device=cuda)
    at = [(0, 0), (0, s - 1), (1, 0), (1, (1 << 30) + 5), (1, s - 1)]
    for k, (i, j) in enumerate(at):
        x[i, j] = -1.0 - k
        mask[i, j] = True
    x.requires_grad_()
    if kind == "preference":
        loss, step = preference_loss(x, mask, beta=1.0)
        assert [float(step.chosen_rewards), float(step.rejected_rewards)] == [-3.0, -12.0]
        slope = -1 / (1 + math.exp(9.0))
        want = [slope, slope, -slope, -slope, -slope]
    else:
        loss, step = policy_loss(x, None, torch.tensor([1.0, -2.0], device=cuda), mask)
        assert float(step.tokens) == 5.0 and abs(float(loss.detach()) - 4 / 5) <= 2 * U
        want = [-0.2, -0.2, 0.4, 0.4, 0.4]
    (g,) = torch.autograd.grad(loss, x)
    got = [float(g[i, j]) for i, j in at]
    assert all(abs(a - b) <= (2.0 ** -8 + 4 * U) * abs(b) for a, b in zip(got, want))
    assert int(torch.count_nonzero(g)) == 5


@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_same_bits_again_other_stream_and_graph(cuda, kind):
    from hackathon_b200.policy import policy_loss
    from hackathon_b200.preference import preference_loss
    logp, mask, randn = draw(cuda, 8, 5000, torch.float32, 41)
    old, adv = logp + 0.2 * randn(8, 5000), randn(8)

    def step(x):
        if kind == "preference":
            loss, s = preference_loss(x, mask, old)
            more = s.chosen_rewards
        else:
            loss, s = policy_loss(x, old, adv, mask, old, kl_coef=0.1, reduction="sequence")
            more = s.kl
        return loss.detach(), more, torch.autograd.grad(loss, x)[0]

    leaf = logp.clone().requires_grad_()
    first = step(leaf)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step(leaf)
    torch.cuda.current_stream().wait_stream(side)
    assert all(map(torch.equal, first, second))
    graphs = []
    for _ in range(2):                                   # two graphs, each with its workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(leaf)
        graphs.append((graph, out))
    other = (logp * 1.1).requires_grad_()
    want = step(other)
    with torch.no_grad():
        leaf.copy_(other)
    for graph, out in graphs * 2:
        graph.replay()
        assert all(map(torch.equal, out, want))


def test_no_grad_and_frozen_inputs(cuda):
    from hackathon_b200.policy import policy_loss
    from hackathon_b200.preference import preference_loss
    logp, mask, randn = draw(cuda, 4, 50, torch.bfloat16, 51)
    old, adv = logp.float(), randn(4)                    # mixed types are promoted
    for fn in (lambda x: preference_loss(x, mask, old)[0],
               lambda x: policy_loss(x, old, adv, mask)[0]):
        a = fn(logp)
        assert not a.requires_grad
        leaf = logp.detach().requires_grad_()
        b = fn(leaf)
        assert b.requires_grad and torch.equal(a, b.detach())
        (g,) = torch.autograd.grad(b, leaf)
        assert g.dtype == torch.bfloat16
        with torch.no_grad():
            assert not fn(leaf).requires_grad
        (g,) = torch.autograd.grad(fn(leaf), leaf, torch.zeros((), device=cuda))
        assert not g.any()


def test_strided_log_probabilities(cuda):
    from hackathon_b200.policy import policy_loss
    from hackathon_b200.preference import preference_loss
    full, _, randn = draw(cuda, 6, 41, torch.float32, 61)
    adv = randn(6)
    for x in (full[:, :-1], full[:, 1::2], full.t().contiguous().t()):
        assert torch.equal(preference_loss(x, None, x * 0.9)[0],
                           preference_loss(x.contiguous(), None, (x * 0.9).contiguous())[0])
        assert torch.equal(policy_loss(x, x * 0.9, adv)[0],
                           policy_loss(x.contiguous(), (x * 0.9).contiguous(), adv)[0])
    base = full.clone().requires_grad_()
    loss, _ = policy_loss(base[:, :-1], full[:, :-1] * 0.9, adv)
    loss.backward()
    assert not base.grad[:, -1].any() and base.grad[:, :-1].any()


def test_ops_refuse_what_their_kernels_do_not_read(cuda):
    """Direct calls of the ops with tensors of another device, dtype, shape or layout."""
    logp, mask, randn = draw(cuda, 4, 30, torch.float32, 91)
    z, t = randn(4, 90), torch.tensor([3, -100, 5, 89], device=cuda)
    ns = torch.ops.qlora_b200
    g, adv = torch.ones((), device=cuda), randn(4)
    lp, en, state = ns.token_logprobs(z, t, 0.9, True)
    for bad in (t.cpu(), t.int(), t[:3], t[None]):
        with pytest.raises(ValueError, match="token_logprobs"):
            ns.token_logprobs(z, bad, 0.9, True)
    good = [z, t, state, en, lp, en, 0.9]
    for k, bad in ((1, t.cpu()), (2, state[:4]), (2, state.double()), (3, en[:2]), (3, en.cpu()),
                   (4, lp.double()), (4, lp.cpu()), (5, en[:3])):
        with pytest.raises(ValueError, match="token_logprobs_bwd"):
            ns.token_logprobs_bwd(*good[:k], bad, *good[k + 1:])

    def pref(x=logp, m=mask, ref=None, row=None, denom=None):
        return ns.preference(x, m, ref, row, denom, 0.1, 0.0, 0.0, 0.0, 0, False)

    pstate = pref()[1]
    for bad in (dict(x=logp.t()), dict(m=mask.cpu()), dict(m=mask[:2]), dict(m=mask.float()),
                dict(m=mask.t().contiguous().t()), dict(ref=logp.half()), dict(ref=logp.cpu()),
                dict(row=adv.half()), dict(row=adv[:2]), dict(denom=g),
                dict(denom=g.double().cpu())):
        with pytest.raises(ValueError, match="preference"):
            pref(**bad)
    for bad in ((pstate[:4], mask, g), (pstate, mask[:2], g), (pstate, mask, g.double()),
                (pstate, mask, g.cpu()), (pstate.cpu(), mask, g)):
        with pytest.raises((ValueError, NotImplementedError)):
            ns.preference_bwd(*bad, 4, 30, torch.float32)

    def pol(x=logp, old=logp, a=adv, m=mask, ref=None, denom=None):
        return ns.policy(x, old, a, m, ref, denom, 0.2, 0.2, 0.0, 0.0, 0.0, True, True)

    _, lstate, unit = pol()
    for bad in (dict(x=logp.t()), dict(old=logp.half()), dict(old=logp[:2]), dict(a=adv.double()),
                dict(a=adv[:2]), dict(a=adv.cpu()), dict(m=mask.cpu()), dict(ref=logp[:, :4]),
                dict(denom=g)):
        with pytest.raises(ValueError, match="policy"):
            pol(**bad)
    for bad in ((unit.double(), lstate, g), (unit, lstate[:6], g), (unit, lstate, g.double()),
                (unit, lstate.cpu(), g), (unit.t(), lstate, g)):
        with pytest.raises(ValueError, match="policy_bwd"):
            ns.policy_bwd(*bad, True, torch.float32)


NAMES = ("token_logprobs", "token_logprobs_bwd", "preference", "preference_bwd", "policy",
         "policy_bwd")


@pytest.mark.parametrize("name", NAMES)
def test_opcheck(cuda, name):
    import hackathon_b200.objective_ops as oo
    assert set(NAMES) == set(oo.ops())
    logp, mask, randn = draw(cuda, 4, 30, torch.float32, 71)
    z, t = randn(4, 90), torch.tensor([3, -100, 5, 89], device=cuda)
    lp, en, stats = oo.token_logprobs(z, t, 0.9, True)
    g = torch.ones((), device=cuda)
    pref = (logp, mask, logp * 0.9, None, None, 0.1, 0.0, 0.0, 0.0, 0, True)
    pol = (logp, logp * 0.9, randn(4), mask, None, None, 0.2, 0.2, 0.0, 0.0, 0.0, True, True)
    args = {"token_logprobs": (z.requires_grad_(), t, 0.9, True),
            "token_logprobs_bwd": (z.detach(), t, stats, en, lp, en, 0.9),
            "preference": (logp.clone().requires_grad_(), *pref[1:]),
            "preference_bwd": (oo.preference(*pref)[1], mask, g, 4, 30, torch.bfloat16),
            "policy": (logp.clone().requires_grad_(), *pol[1:]),
            "policy_bwd": (oo.policy(*pol)[2], oo.policy(*pol)[1], g, True, torch.float32)}[name]
    # the objectives' second output ends in workspace, which no two runs fill alike in the same
    # places they leave unwritten: the schema, fake and registration checks apply
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(getattr(torch.ops.qlora_b200, name).default, args, test_utils=tests)


def test_a_rejected_sequence_that_cannot_occur(cuda):
    """A counted token of log-probability -inf in the rejected sequence: the pair is infinitely far
    apart, its loss 0 and its gradients 0, whatever the loss's slope elsewhere; the other pair
    keeps its own."""
    from hackathon_b200.preference import preference_loss
    x = torch.tensor([[-2.0, -1.0], [-1.0, -3.0], [-math.inf, -1.0], [-2.0, -1.0]], device=cuda)
    alone = torch.tensor([[-1.0, -3.0], [-2.0, -1.0]], device=cuda)
    for kind in ("sigmoid", "hinge"):
        for eps in (0.0, 0.2) if kind == "sigmoid" else (0.0,):
            leaf, one = x.clone().requires_grad_(), alone.clone().requires_grad_()
            loss, step = preference_loss(leaf, None, None, 0.5, kind, eps, denominator=1.0)
            want, _ = preference_loss(one, None, None, 0.5, kind, eps, denominator=1.0)
            (g,) = torch.autograd.grad(loss, leaf)
            (wg,) = torch.autograd.grad(want, one)
            assert torch.isfinite(g).all() and float(step.rejected_rewards[0]) == -math.inf
            assert torch.equal(g[[1, 3]], wg)
            if eps == 0.0:
                assert torch.equal(loss.detach(), want.detach()) and not g[[0, 2]].any()
            else:           # label smoothing: the flipped label costs infinitely much
                assert float(loss.detach()) == math.inf
                assert torch.equal(g[[0, 2]], torch.tensor([[0.1], [-0.1]], device=cuda)
                                   .expand(2, 2))
    # an infinitely better rejected one: an infinite loss with a finite slope
    y = torch.tensor([[-math.inf], [-2.0]], device=cuda, requires_grad=True)
    for kind in ("sigmoid", "hinge"):
        loss, _ = preference_loss(y, loss_type=kind, beta=0.5)
        (g,) = torch.autograd.grad(loss, y)
        assert float(loss.detach()) == math.inf and g.flatten().tolist() == [-0.5, 0.5]


@pytest.mark.filterwarnings("ignore:There is a performance drop")
@pytest.mark.parametrize("dim", [0, 1])
def test_batched_calls(cuda, dim):
    """Under torch.vmap every function gives each element's own results and gradients; the other
    function transforms, which need more than the ops have, are refused by name."""
    from hackathon_b200.logprobs import token_logprobs
    from hackathon_b200.policy import policy_loss
    from hackathon_b200.preference import preference_loss
    logp, mask, randn = draw(cuda, 12, 50, torch.float32, 95)
    logp, mask = logp.view(3, 4, 50), mask.view(3, 4, 50)
    old, adv = logp + 0.2 * randn(3, 4, 50), randn(3, 4)
    z, t = randn(3, 4, 700), torch.arange(12, device=cuda).view(3, 4)

    def one(x, m, o, a, logits, target):
        p, _ = preference_loss(x, m, o)
        q, step = policy_loss(x, o, a, m, o, kl_coef=0.1)
        lp, en = token_logprobs(logits, target, 0.9, True)
        return p, q, step.kl, lp, en

    args = [logp, mask, old, adv, z, t]
    want = [torch.stack(v) for v in zip(*(one(*(a[i] for a in args)) for i in range(3)))]
    moved = [a.movedim(0, dim) for a in args]
    got = torch.vmap(one, in_dims=dim)(*moved)
    assert all(map(torch.equal, got, want))

    def total(x, logits):
        p, q, _, lp, en = torch.vmap(one)(x, mask, old, adv, logits, t)
        return (p + q).sum() + (lp - en).sum()

    leaf, zl = logp.clone().requires_grad_(), z.clone().requires_grad_()
    got = torch.autograd.grad(total(leaf, zl), (leaf, zl))
    for i in range(3):
        x, y = logp[i].clone().requires_grad_(), z[i].clone().requires_grad_()
        p, q, _, lp, en = one(x, mask[i], old[i], adv[i], y, t[i])
        wx, wy = torch.autograd.grad(p + q + (lp - en).sum(), (x, y))
        assert torch.equal(got[0][i], wx) and torch.equal(got[1][i], wy)
    with pytest.raises(RuntimeError, match="setup_context"):
        torch.func.grad(lambda x: preference_loss(x)[0])(logp[0])


def test_tensor_subclasses_reach_their_own_dispatch(cuda):
    """A subclass anywhere among the arguments takes the call to its __torch_dispatch__."""
    from torch.testing._internal.two_tensor import TwoTensor

    from hackathon_b200.logprobs import token_logprobs
    from hackathon_b200.preference import preference_loss
    logp, mask, randn = draw(cuda, 4, 30, torch.float32, 96)
    z, t = randn(4, 90), torch.tensor([3, -100, 5, 89], device=cuda)
    got = token_logprobs(z, TwoTensor(t, t.flip(0)))
    assert torch.equal(got.a, token_logprobs(z, t))
    assert torch.equal(got.b, token_logprobs(z, t.flip(0)))
    got, _ = preference_loss(logp, TwoTensor(mask, mask.flip(0)))
    assert torch.equal(got.a, preference_loss(logp, mask)[0])
    assert torch.equal(got.b, preference_loss(logp, mask.flip(0))[0])


def test_profilers_see_the_ops_by_name(cuda):
    from torch.profiler import ProfilerActivity, profile

    from hackathon_b200.logprobs import token_logprobs
    from hackathon_b200.policy import policy_loss
    from hackathon_b200.preference import preference_loss
    logp, mask, randn = draw(cuda, 4, 30, torch.float32, 97)
    z, t = randn(4, 90).requires_grad_(), torch.arange(4, device=cuda)
    leaf = logp.requires_grad_()
    with profile(activities=[ProfilerActivity.CPU]) as prof:
        total = token_logprobs(z, t).sum() + preference_loss(leaf, mask)[0] \
            + policy_loss(leaf, None, randn(4), mask)[0]
        total.backward()
    seen = {e.key for e in prof.key_averages()}
    assert {f"qlora_b200::{name}" for name in NAMES} <= seen


def test_forward_mode_tangents_are_refused(cuda):
    """No forward-mode derivative: an input with a tangent is refused, not answered without it."""
    import torch.autograd.forward_ad as fwad

    from hackathon_b200.grad_norm import clip_grad_norm_, grad_norm
    from hackathon_b200.logprobs import linear_token_logprobs, token_logprobs
    from hackathon_b200.policy import policy_loss
    from hackathon_b200.preference import preference_loss
    logp, mask, randn = draw(cuda, 4, 64, torch.float32, 98)
    z, t, w, a = randn(4, 64), torch.arange(4, device=cuda), randn(80, 64), randn(4)
    p = torch.nn.Parameter(randn(5))
    calls = [(logp, lambda x: preference_loss(x, mask)), (logp, lambda x: policy_loss(x, x, a)),
             (logp, lambda x: policy_loss(logp, x, a)), (logp, lambda x: preference_loss(logp, mask, x)),
             (z, lambda x: token_logprobs(x, t)), (z, lambda x: linear_token_logprobs(x, w, t)),
             (w, lambda x: linear_token_logprobs(z, x, t)), (z, grad_norm)]
    for x, fn in calls:
        with fwad.dual_level():
            for y in (x, x.clone().requires_grad_()):
                dual = fwad.make_dual(y, torch.ones_like(x))
                with pytest.raises((NotImplementedError, ValueError)):
                    fn(dual)
            fn(x)                               # plain inputs are served there as anywhere
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(fn, (x,), (torch.ones_like(x),))
    with fwad.dual_level():
        p.grad = fwad.make_dual(randn(5), torch.ones(5, device=cuda))
        with pytest.raises(NotImplementedError):
            clip_grad_norm_(p, 1.0)


def test_preference_ops_refuse_an_odd_row(cuda):
    """The kernels read pairs: a row without a partner would be left out of everything."""
    logp, mask, _ = draw(cuda, 5, 30, torch.float32, 92)
    ns = torch.ops.qlora_b200
    with pytest.raises(ValueError, match="preference"):
        ns.preference(logp, mask, None, None, None, 0.1, 0.0, 0.0, 0.0, 0, False)
    state, g = torch.zeros(64, device=cuda), torch.ones((), device=cuda)
    with pytest.raises(ValueError, match="preference_bwd"):
        ns.preference_bwd(state, mask, g, 5, 30, torch.float32)


def test_policy_at_the_borders_rounded_differences(cuda):
    """Differences whose fp32 value is a border's own rounding: the exact one decides, for the
    gradient and for the shares. old = +- 7/16 of the border's last place moves it to either side
    of the border (each is rounded by less) without moving its fp32 value."""
    from hackathon_b200.policy import policy_loss
    low, high, delta = math.log1p(-0.2), math.log1p(0.28), math.log(1.6)
    rows = torch.tensor([low, high, delta], dtype=torch.float64).float()
    x = rows[:, None].repeat(1, 2).to(cuda)
    step = (torch.nextafter(rows, torch.full_like(rows, 9.0)) - rows)[:, None].to(cuda) * 7 / 16
    old = torch.cat([step, -step], 1)
    exact = x.double() - old.double()
    assert torch.equal(x - old, x)                              # they tie in fp32 ...
    edge = torch.tensor([low, high, delta], dtype=torch.float64, device=cuda)[:, None]
    assert torch.equal(exact < edge, torch.tensor([[True, False]] * 3, device=cuda))
    for sign in (1.0, -1.0):
        adv = torch.full((3,), sign, device=cuda)
        leaf = x.clone().requires_grad_()
        loss, step = policy_loss(leaf, old, adv, None, None, 0.2, 0.28, 1.6)
        (g,) = torch.autograd.grad(loss, leaf)
        below, above, past = exact < low, exact > high, exact > delta
        live = ~past & (~(below | above) | (below & (sign > 0)) | (above & (sign < 0)))
        assert torch.equal(g != 0, live)
        assert float(step.clipped_low) == float((below & (sign < 0)).double().mean().float())
        assert float(step.clipped_high) == float((above & (sign > 0)).double().mean().float())


def test_upstream_tangents_are_refused_in_the_backward(cuda):
    """The gradient's own op has no forward-mode derivative either."""
    import torch.autograd.forward_ad as fwad

    from hackathon_b200.preference import preference_loss
    logp, mask, _ = draw(cuda, 4, 30, torch.float32, 99)
    leaf = logp.requires_grad_()
    loss, _ = preference_loss(leaf, mask)
    one = torch.ones((), device=cuda)
    with fwad.dual_level():
        with pytest.raises(NotImplementedError, match="preference_bwd"):
            torch.autograd.grad(loss, leaf, fwad.make_dual(one, one))
