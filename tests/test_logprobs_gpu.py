"""Log-probabilities of chosen tokens (logprobs.py) against a 64-bit softmax.

Tolerances, with u = 2^-24 (half an fp32 step), x = (z - max) / T, V the row's length and L the
additions of the longest chain behind a row sum (V / 512 a thread, then the merges):
  * a term e^x: the exponent's scale and product are rounded a few times (4 u |x| together), and
    the hardware's 2^y is good to 4 u; its weight in the sum is p, and sum p |x| <= H <= ln V;
  * so ln s is off by at most u (4 ln V + 4 + L + 2), a logp by that and u (4 |logp| + 2);
  * H = ln s - sum p x has one more factor x in its terms: u (2 ln^2 V + (L + 8) ln V) more;
  * a gradient is g p / T [...]: relative to its terms u (4 |x| + L + 16), then half a step of the
    logits' type, and what is below the type's smallest normal number."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
IGNORE = -100
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def exact(logits, target, t, gl=None, ge=None):
    """(logp, entropy, gradient) in 64 bits, and the bounds on the three."""
    z = logits.detach().double()
    v = z.shape[-1]
    lnq = torch.log_softmax(z / t, -1)
    q = lnq.exp()
    keep = (target >= 0) & (target < v)
    at = torch.where(keep, target, 0)[..., None]
    logp = torch.where(keep, lnq.gather(-1, at)[..., 0], 0.0)
    ent = -torch.where(q > 0, q * lnq, 0.0).sum(-1)
    length = v / 512 + 16
    lnv = math.log(v) if v > 1 else 0.0
    t_lse = U * (4 * lnv + 6 + length)
    # a logp of -inf (a banned target) is exactly that
    t_logp = t_lse + U * (4 * logp.abs().nan_to_num(posinf=0.0) + 2)
    t_ent = t_lse + U * (2 * lnv ** 2 + (length + 8) * lnv + 2)
    if gl is None and ge is None:
        return logp, ent, None, t_logp, t_ent, None
    w = (torch.where(keep, gl, 0.0) if gl is not None else torch.zeros_like(logp))[..., None]
    h = (ge if ge is not None else torch.zeros_like(logp))[..., None].double()
    w = w.double()
    grad = -w * q - h * torch.where(q > 0, q * (lnq + ent[..., None]), 0.0)
    grad.scatter_add_(-1, at, w)
    grad = grad / t
    size = torch.where(q > 0, (lnq.abs() + ent[..., None]) * q, 0.0) * h.abs() + q * w.abs()
    x = torch.where(q > 0, (lnq - lnq.amax(-1, keepdim=True)).abs(), 0.0)
    dt = logits.dtype
    t_grad = (U * (4 * x + length + 16) * size + q * h.abs() * t_ent) / t
    t_grad = t_grad + 2 * U * (w.abs() / t) * (torch.zeros_like(q).scatter_(-1, at, 1.0))
    t_grad = t_grad + HALF[dt] * (grad.abs() + t_grad) + torch.finfo(dt).smallest_normal * U * 2 \
        + torch.finfo(dt).smallest_normal * 2.0 ** -9
    return logp, ent, grad, t_logp, t_ent, t_grad


def close(got, want, tol):
    got = got.double()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    ok = ~nan & ~inf
    over = ((got - want).abs() - tol)[ok]
    assert over.numel() == 0 or float(over.max()) <= 0, float(over.max())


def make(dev, shape, dtype, seed=0, scale=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    z = (torch.randn(*shape, device=dev, generator=g) * scale).to(dtype)
    t = torch.randint(0, shape[-1], shape[:-1], device=dev, generator=g)
    return z, t, g


def check(z, t, temperature=1.0, entropy=True, seed=1):
    """Forward (with and without a gradient) and backward of one call."""
    from hackathon_b200.logprobs import token_logprobs
    g = torch.Generator(device=z.device).manual_seed(seed)
    gl = torch.randn(t.shape, device=z.device, generator=g)
    ge = torch.randn(t.shape, device=z.device, generator=g) if entropy else None
    want = exact(z, t, temperature, gl, ge)
    leaf = z.detach().requires_grad_()
    got = token_logprobs(leaf, t, temperature, entropy)
    got = got if entropy else (got,)
    (grad,) = torch.autograd.grad(got, leaf, (gl, ge) if entropy else (gl,))
    assert grad.dtype == z.dtype and grad.is_contiguous()
    close(got[0].detach(), want[0], want[3])
    if entropy:
        close(got[1].detach(), want[1], want[4])
    close(grad, want[2], want[5])
    with torch.no_grad():
        again = token_logprobs(z, t, temperature, entropy)
    again = again if entropy else (again,)
    assert all(torch.equal(a.nan_to_num(7.0), b.detach().nan_to_num(7.0))
               for a, b in zip(again, got))
    return got, grad


SHAPES = [(1, 1), (1, 2), (3, 7), (2, 255), (5, 256), (1, 4095), (1, 4097), (2, 3, 8200),
          (300, 513), (1, 33001), (7, 33000), (2, 151936), (1, 152064), (40, 50001), (297, 4104)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(cuda, shape, dtype):
    z, t, g = make(cuda, shape, dtype)
    if t.numel() > 2:
        t.view(-1)[::3] = IGNORE
        t.view(-1)[1] = shape[-1]              # also no token
    check(z, t)
    check(z, t, entropy=False)


@pytest.mark.parametrize("temperature", [1e-3, 0.3, 0.7, 2.5, 1e4])
def test_temperature(cuda, temperature):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        z, t, _ = make(cuda, (4, 1001), dtype)
        z[1, 5:] = -math.inf
        check(z, t.clamp(max=4), temperature)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_banned_and_lowest_logits(cuda, dtype):
    low = torch.finfo(dtype).min
    for v in (37, 5000, 40001):
        z, t, _ = make(cuda, (9, v), dtype)
        t[:] = 1
        z[0, 2:] = -math.inf                   # two tokens left
        z[1, 2:] = low
        z[2, :] = low                          # every token at the lowest value: uniform
        z[3, 1] = -math.inf                    # the target itself is banned: -inf
        z[4, :] = -math.inf                    # nothing left: NaN
        z[4, 1] = 3.0                          # ... but the target: certain
        z[5, ::2] = -math.inf
        z[6, : v // 2] = low
        z[7, :] = torch.finfo(dtype).max       # the highest value everywhere: uniform
        z[8, 1:] = low                         # one token left, and it is not the target
        got, grad = check(z, t)
        assert float(got[0][4].detach()) == 0.0 and float(got[1][4].detach()) == 0.0
        assert float(got[0][3].detach()) == -math.inf


@pytest.mark.parametrize("v", [3, 999, 40000])
def test_rows_without_a_distribution_are_nan(cuda, v):
    from hackathon_b200.logprobs import token_logprobs
    z, t, _ = make(cuda, (5, v), torch.float32)
    z[1] = -math.inf
    z[2, 1] = math.inf
    z[3, 2] = math.nan
    leaf = z.requires_grad_()
    lp, en = token_logprobs(leaf, t, with_entropy=True)
    assert torch.isnan(lp[1:4]).all() and torch.isnan(en[1:4]).all()
    assert torch.isfinite(lp[[0, 4]]).all() and torch.isfinite(en[[0, 4]]).all()
    (g,) = torch.autograd.grad(lp, leaf, torch.ones_like(lp), retain_graph=True)
    assert torch.isnan(g[[1, 3]]).all() and torch.isfinite(g[[0, 4]]).all()
    assert torch.isnan(g[2]).any()
    # such a row, left out of the objective, spreads nothing
    (g,) = torch.autograd.grad(lp, leaf, torch.tensor([1.0, 0, 0, 0, 1.0], device=cuda))
    assert torch.isfinite(g).all() and not g[1:4].any()


def test_views_are_read_in_place(cuda):
    """Next-token views, sliced vocabularies, odd row starts, expanded rows (one row many times)
    and a transposed vocabulary."""
    for dtype in (torch.bfloat16, torch.float32):
        full, _, g = make(cuda, (3, 6, 4003), dtype)
        for z in (full[:, :-1], full[:, 1:, :4000], full[..., 1:], full[..., 3:4000],
                  full[1], full[:, 0, 5:], full[0, 0].expand(4, 4003),
                  full[:, :1].expand(3, 5, 4003), full.transpose(0, 1),
                  full.transpose(1, 2)):
            t = torch.randint(0, z.shape[-1], z.shape[:-1], device=cuda, generator=g)
            check(z, t)
    z, t, _ = make(cuda, (2, 2, 3, 100), torch.bfloat16)
    check(z, t)
    z, t, _ = make(cuda, (100,), torch.bfloat16)
    check(z, t)


def test_gradient_of_a_view_reaches_its_base(cuda):
    from hackathon_b200.logprobs import token_logprobs
    full, _, g = make(cuda, (2, 5, 301), torch.float32)
    full.requires_grad_()
    t = torch.randint(0, 301, (2, 4), device=cuda, generator=g)
    token_logprobs(full[:, :-1], t).sum().backward()       # an expanded upstream gradient
    want = exact(full[:, :-1], t, 1.0, torch.ones(2, 4, device=cuda))
    close(full.grad[:, :-1], want[2], want[5])
    assert not full.grad[:, -1].any()


def test_target_types_and_strides(cuda):
    from hackathon_b200.logprobs import token_logprobs
    z, t, _ = make(cuda, (4, 6, 90), torch.float32)
    want = token_logprobs(z, t)
    for other in (t.int(), t.to(torch.int16), t.to(torch.uint8),
                  t.t().contiguous().t()):
        assert torch.equal(token_logprobs(z, other), want)
    assert token_logprobs(z[:0], t[:0]).shape == (0, 6)
    assert token_logprobs(z[:, :0], t[:, :0], with_entropy=True)[1].shape == (4, 0)
    leaf = z[:0].detach().requires_grad_()
    (g,) = torch.autograd.grad(token_logprobs(leaf, t[:0]).sum(), leaf)
    assert g.shape == leaf.shape


def test_gradient_against_differences(cuda):
    """The gradient along a direction against central differences of the 64-bit function. The
    difference quotient's own error is h^2 / 6 times the third derivative (bounded by the sum of
    |direction|^3 times a few units) and 2^-52 |f| / h."""
    from hackathon_b200.logprobs import token_logprobs
    z, t, g = make(cuda, (3, 50), torch.float32)
    gl, ge = torch.randn(3, device=cuda, generator=g), torch.randn(3, device=cuda, generator=g)
    d = torch.randn(3, 50, device=cuda, generator=g).double()

    def f(x):
        q = torch.log_softmax(x / 0.8, -1)
        lp = q.gather(-1, t[:, None])[:, 0]
        return (gl.double() * lp - ge.double() * (q.exp() * q).sum(-1)).sum()

    h = 1e-4
    want = (f(z.double() + h * d) - f(z.double() - h * d)) / (2 * h)
    leaf = z.requires_grad_()
    (grad,) = torch.autograd.grad(token_logprobs(leaf, t, 0.8, True), leaf, (gl, ge))
    got = (grad.double() * d).sum()
    bound = exact(z, t, 0.8, gl, ge)[5]
    assert float((got - want).abs()) <= float((bound * d.abs()).sum()) + 1e-6


def test_only_one_output_used(cuda):
    from hackathon_b200.logprobs import token_logprobs
    z, t, g = make(cuda, (4, 700), torch.bfloat16)
    w = torch.randn(4, device=cuda, generator=g)
    for k in (0, 1):
        leaf = z.detach().requires_grad_()
        out = token_logprobs(leaf, t, with_entropy=True)[k]
        (grad,) = torch.autograd.grad(out, leaf, w)
        want = exact(z, t, 1.0, *((w, None) if k == 0 else (None, w)))
        close(grad, want[2], want[5])


def test_rows_past_32_bit_offsets(cuda):
    """Rows that start beyond 2^31 and 2^32 elements; 4.4 billion bf16 logits."""
    from hackathon_b200.logprobs import token_logprobs
    v, n = 151936, 28500
    z = torch.zeros(n, v, dtype=torch.bfloat16, device=cuda)
    pick = torch.tensor([0, 14140, 28268, n - 1], device=cuda)
    part, t, _ = make(cuda, (4, v), torch.bfloat16)
    z[pick] = part
    target = torch.full((n,), 5, device=cuda)
    target[pick] = t
    lp, en = token_logprobs(z, target, with_entropy=True)
    want = exact(part, t, 1.0)
    close(lp[pick], want[0], want[3])
    close(en[pick], want[1], want[4])
    assert abs(float(lp[1]) + math.log(v)) <= U * (8 * math.log(v) + 400)
    z = z.requires_grad_()
    w = torch.zeros(n, device=cuda)
    w[pick] = 1.0
    (grad,) = torch.autograd.grad(token_logprobs(z, target), z, w)
    want = exact(part, t, 1.0, torch.ones(4, device=cuda))
    close(grad[pick], want[2], want[5])
    assert not grad[1].any() and not grad[n - 2].any()


def test_same_bits_again_other_stream_and_graph(cuda):
    """The same bits on a second run, on another stream, and replayed from a captured graph that
    holds the forward and the backward, with new values in its inputs."""
    from hackathon_b200.logprobs import token_logprobs
    z, t, _ = make(cuda, (6, 9001), torch.bfloat16)
    w = torch.linspace(-1, 1, 6, device=cuda)

    def step(x):
        out = token_logprobs(x, t, 0.9, True)
        return (*[o.detach() for o in out], *torch.autograd.grad(out, x, (w, w)))

    leaf = z.clone().requires_grad_()
    first = step(leaf)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step(leaf)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step(leaf)
    other, _, _ = make(cuda, (6, 9001), torch.bfloat16, seed=9)
    with torch.no_grad():
        leaf.copy_(other)
    graph.replay()
    for a, b in zip(third, step(other.clone().requires_grad_())):
        assert torch.equal(a, b)
    with torch.no_grad():
        leaf.copy_(z)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, third))


def test_second_derivative_is_refused(cuda):
    from hackathon_b200.logprobs import token_logprobs
    z, t, _ = make(cuda, (2, 30), torch.float32)
    z.requires_grad_()
    (g,) = torch.autograd.grad(token_logprobs(z, t).sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_form_matches_the_materialised_one(cuda, dtype):
    """linear_token_logprobs against the 64-bit product: the bf16 head's logits stay in TMEM as
    fp32 sums of H products (an error of u (H + 2) sum |h w| in each logit, so in each logp twice
    that at most), plus token_logprobs's own bound; its gradient through bf16 dZ: 2^-8 of the
    terms each, twice (dZ and the result)."""
    from hackathon_b200.logprobs import linear_token_logprobs
    g = torch.Generator(device=cuda).manual_seed(3)
    h = torch.randn(2, 37, 256, device=cuda, generator=g).to(dtype)
    w = (torch.randn(1000, 256, device=cuda, generator=g) * 0.1).to(dtype)
    t = torch.randint(0, 1000, (2, 37), device=cuda, generator=g)
    t[0, :5] = IGNORE
    leaf = h.requires_grad_()
    lp, en = linear_token_logprobs(leaf, w, t)
    z = h.detach().double() @ w.double().t()
    per_logit = U * 258 * (h.detach().double().abs() @ w.double().abs().t()).amax(-1)
    if dtype == torch.float32:      # the logits of this path are an fp32 matmul (TF32 is off)
        per_logit = 2 * per_logit
    want = exact(z.float(), t, 1.0, torch.ones(2, 37, device=cuda))
    lp64 = torch.where(
        t >= 0, torch.log_softmax(z, -1).gather(-1, t.clamp(min=0)[..., None])[..., 0], 0.0)
    close(lp.detach(), lp64, want[3] + 2 * per_logit + U * 8 * lp64.abs())
    assert not en.requires_grad
    lp.sum().backward()
    q = torch.softmax(z, -1)
    keep = (t >= 0)[..., None]
    dz = torch.where(keep, -q, 0.0)
    dz.scatter_add_(-1, t.clamp(min=0)[..., None], keep.double())
    size = dz.abs() @ w.double().abs()
    tol = (2 * 2.0 ** -8 if dtype == torch.bfloat16 else 600 * U) * size \
        + 4 * per_logit[..., None] * size
    close(leaf.grad, dz @ w.double(), tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [777, 1000])
def test_targets_outside_the_vocabulary_score_nothing(cuda, vocab, dtype, monkeypatch):
    """Any target outside [0, vocab) is a constant 0 with no gradient, as -100 is: the same bits,
    on the recomputing and on the storing gradient pass, and 0 even from a row of NaN."""
    from hackathon_b200 import cross_entropy
    from hackathon_b200.logprobs import linear_token_logprobs
    g = torch.Generator(device=cuda).manual_seed(vocab)
    h = torch.randn(150, 256, device=cuda, generator=g).to(dtype)
    w = (torch.randn(vocab, 256, device=cuda, generator=g) * 0.1).to(dtype)
    t = torch.randint(0, vocab, (150,), device=cuda, generator=g)
    out = torch.tensor([vocab, vocab + 5, 1 << 31, 1 << 40, -1, -7, -(1 << 40)], device=cuda)
    at = torch.arange(3, 3 + 20 * len(out), 20, device=cuda)
    t[at] = out
    plain = t.clone()
    plain[at] = IGNORE

    def run(target, hidden=h):
        leaf = hidden.detach().requires_grad_()
        lp, _ = linear_token_logprobs(leaf, w, target)
        (grad,) = torch.autograd.grad(lp, leaf, torch.linspace(-2, 3, 150, device=cuda))
        return lp.detach(), grad

    for store in (False, True):
        monkeypatch.setattr(cross_entropy, "STORE_LOGITS", store)
        want, got = run(plain), run(t)
        assert all(map(torch.equal, got, want))
        assert not got[0][at].any() and not got[1][at].any() and got[1][4].any()
        broken = h.clone()
        broken[at] = math.nan
        lost = run(t, broken)
        assert torch.equal(lost[0], want[0]) and torch.equal(lost[1], want[1])


@pytest.mark.parametrize("temperature", [0.7, 0.9, 1.0, 2.5])
def test_gradient_of_a_nearly_certain_token(cuda, temperature):
    """A target of probability 1 - q with q about 2^-20 has the gradient g q / T. Its only rival's
    logit d is one whose scaled exponent is a whole number, so the row's sum 1 + 2^-k is exact and
    q is good to 4 u |d / T| + 4 u (the exponent's scale and product, 2^y); the gradient's products
    add 4 u: 2^-16 relative covers d / T of 14. One of g / T and -g p / T, each rounded by itself
    before they cancel, is off by u / q: 2^-4."""
    import numpy as np

    from hackathon_b200.logprobs import token_logprobs
    one = np.float32(1)
    c = (one / np.float32(temperature)) * np.float32(1.4426950408889634)
    for k in (18, 20):
        d = np.float32(-k / np.float64(c))
        for _ in range(40):
            if d * c == -k:
                break
            d = np.nextafter(d, np.float32(-100 if d * c > -k else 100))
        assert d * c == -k
        for v, label, rival in ((2000, 700, 3), (2001, 2000, 5), (5, 2, 4), (40001, 9, 40000)):
            z = torch.full((4, v), -math.inf, device=cuda)
            z[:, label], z[:, rival] = 0.0, float(d)
            t = torch.full((4,), label, device=cuda)
            gl = torch.tensor([1.0, 0.37, -2.9, 1e-3], device=cuda)
            leaf = z.requires_grad_()
            (g,) = torch.autograd.grad(token_logprobs(leaf, t, temperature), leaf, gl)
            x = math.exp(float(d) / temperature)
            want = gl.double() / temperature * (x / (1 + x))
            assert bool(((g[:, label].double() - want).abs() <= 2.0 ** -16 * want.abs()).all())
            assert bool(((g[:, rival].double() + want).abs() <= 2.0 ** -16 * want.abs()).all())


def test_small_terms_beside_the_top_one_count(cuda):
    """200,000 terms of 0.9 * 2^-24 beside one of 1: each is lost when added to a sum of 1 or more.
    A thread's batches hold 32 terms in two sums and there are V / 4096 of them, then come about a
    dozen merges; each such addition is off by 2^-24 at most."""
    from hackathon_b200.logprobs import token_logprobs
    v, d = 200_000, -16.75
    z = torch.full((600, v), d, dtype=torch.bfloat16, device=cuda)     # rows in one span each
    z[:, 0] = 0.0
    lp = token_logprobs(z, torch.zeros(600, dtype=torch.int64, device=cuda))
    want = -math.log1p((v - 1) * math.exp(d))
    bound = U * (v / 4096 + 16 + 12) + 4 * U * abs(want) + U * 4 * abs(d) * abs(want)
    assert float((lp.double() - want).abs().max()) <= bound
