"""The post-training operators together, as a program runs them: scoring, the objective, the
backward pass, clipping and the optimizer step of a small QLoRA model."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def tiny(**kw):
    from hackathon_b200.qlora import QwenQLoRA, preset
    shape = preset("0.5b", layers=2, vocab=2000, lora_dropout=kw.pop("dropout", 0.0))
    return QwenQLoRA(shape, device="cuda:0", seed=1, **kw), shape


def batch(shape, n, s, seed=0):
    """Token ids, labels with a prompt and padding left out, one sequence without an answer."""
    g = torch.Generator(device="cuda:0").manual_seed(seed)
    ids = torch.randint(0, shape.vocab, (n, s), device="cuda:0", generator=g)
    labels = ids.clone()
    labels[:, : s // 4] = -100
    labels[1, s // 2:] = -100
    labels[n - 1] = -100
    return ids, labels


@pytest.fixture(autouse=True)
def _attention_in_a_fixed_order():
    """Attention in its math form, whose backward adds in a fixed order: two runs of one model give
    the same bits."""
    from torch.nn.attention import SDPBackend, sdpa_kernel
    with sdpa_kernel(SDPBackend.MATH):
        yield


def grads_of(model):
    return [p.grad.clone() for p in model.adapter_parameters()]


def test_token_logprobs_are_the_losses(cuda):
    """logp is the negative per-token loss the training step sums, and scoring leaves no graph."""
    model, shape = tiny()
    ids, labels = batch(shape, 4, 48)
    with torch.no_grad():
        loss, step = model(ids, labels)
        logp, entropy, mask = model.token_logprobs(ids, labels)
    assert torch.equal(logp, -step.token_loss) and torch.equal(entropy, step.token_entropy)
    assert int(mask.sum()) == int(step.labelled) and not logp[~mask].any()
    assert not logp.requires_grad
    assert abs(float(loss) + float(logp.sum()) / int(mask.sum())) < 1e-4
    # the materialised form on the same hidden states: the bf16 logits' rounding, 2^-8 of them
    from hackathon_b200.cross_entropy import shift_labels_of
    from hackathon_b200.logprobs import token_logprobs
    with torch.no_grad():
        h = model.hidden_states(ids)
        z = h.float() @ model.lm_head.float().t()
        direct, other = token_logprobs(z, shift_labels_of(labels), with_entropy=True)
    # fp32 logits of both: H products summed, u (H + 2) of their absolute sum, in two logits
    tol = 4 * U * (shape.hidden + 2) * float(
        (h.float().abs() @ model.lm_head.float().abs().t()).max()) + 1e-4
    assert float((direct - logp).abs().max()) <= tol
    assert float((other - entropy).abs().max()) <= tol * 20


@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_objective_gradient_reaches_the_adapters(cuda, kind):
    """What reaches the log-probabilities is the gradient of the objective written in 64-bit torch
    operations, and what reaches the adapters is that gradient sent back through the model, bit
    for bit."""
    from hackathon_b200.policy import policy_loss
    from hackathon_b200.preference import preference_loss
    model, shape = tiny()
    model.train()
    ids, labels = batch(shape, 4, 64)
    g = torch.Generator(device="cuda:0").manual_seed(5)
    logp, _, mask = model.token_logprobs(ids, labels)
    base = logp.detach()
    ref = base + 0.1 * torch.randn(base.shape, device="cuda:0", generator=g)
    old = base + 0.1 * torch.randn(base.shape, device="cuda:0", generator=g)
    adv = torch.randn(4, device="cuda:0", generator=g)
    if kind == "preference":
        loss, _ = preference_loss(logp, mask, ref, beta=0.2)
    else:
        loss, _ = policy_loss(logp, old, adv, mask, ref, kl_coef=0.05)
    seen = []
    logp.register_hook(seen.append)
    loss.backward()
    got = grads_of(model)
    model.zero_grad(set_to_none=True)
    logp, _, mask = model.token_logprobs(ids, labels)
    assert torch.equal(logp.detach(), base)
    logp.backward(seen[0])
    want = grads_of(model)
    assert all(map(torch.equal, got, want)) and any(bool(w.any()) for w in want)
    x = base.double().requires_grad_()
    if kind == "preference":
        s = torch.where(mask, x - ref.double(), 0.0).sum(1)
        plain = torch.nn.functional.softplus(-0.2 * (s[:2] - s[2:])).mean()
    else:
        r = (x - old.double()).exp()
        a = adv[:, None].double()
        d = ref.double() - x
        t = -torch.minimum(r * a, r.clamp(0.8, 1.2) * a) + 0.05 * (d.exp() - d - 1)
        plain = torch.where(mask, t, 0.0).sum() / mask.sum()
    (dlogp,) = torch.autograd.grad(plain, x)
    # |d| <= 1 and r about 1: a term's parts are at most 2 |A| + 0.05 * 2, good to 20 u
    scale = (2 * float(adv.abs().max()) + 0.1) / int(mask.sum()) if kind == "policy" else 0.1
    assert float((seen[0].double() - dlogp).abs().max()) <= 20 * U * scale
    assert abs(float(loss.detach()) - float(plain.detach())) <= 20 * U * (
        scale * int(mask.sum()) if kind == "policy" else 1.0 + abs(float(plain.detach())))


@pytest.mark.parametrize("dropout", [0.0, 0.1])
@pytest.mark.parametrize("kind", ["train", "preference", "policy"])
def test_steps_clip_before_the_optimizer(cuda, kind, dropout):
    """A step with max_grad_norm moves the adapters as the same step with its gradients clipped by
    hand does; a limit above the norm changes nothing. SGD: the move is the clipped gradient."""
    from hackathon_b200.qlora import policy_step, preference_step, train_step

    def run(limit, by_hand=None):
        model, shape = tiny(dropout=dropout)
        ids, labels = batch(shape, 4, 64)
        params = model.adapter_parameters()
        before = [p.detach().clone() for p in params]
        opt = torch.optim.SGD(params, lr=1.0)
        if by_hand is not None:
            opt.register_step_pre_hook(lambda o, *_: by_hand(params))
        if kind == "train":
            train_step(model, opt, ids, labels, max_grad_norm=limit)
        else:
            with torch.no_grad():
                ref, _, mask = model.eval().token_logprobs(ids, labels)
            if kind == "preference":
                loss, step = preference_step(model, opt, ids, labels, ref, max_grad_norm=limit,
                                             beta=0.5)
                assert step.chosen_rewards.shape == (2,)
            else:
                loss, step = policy_step(model, opt, ids, labels, ref,
                                         torch.tensor([1.0, -1.0, 0.5, 2.0], device="cuda:0"),
                                         ref, max_grad_norm=limit, kl_coef=0.1)
                assert float(step.tokens) == float(mask.sum())
            assert not loss.requires_grad and math.isfinite(float(loss))
        assert all(p.grad is None for p in params)
        return [(b - p.detach()) for b, p in zip(before, params)], model

    free, model = run(None)
    norm = math.sqrt(sum(float(d.double().square().sum()) for d in free))
    assert norm > 0
    same, _ = run(1e6)
    assert all(map(torch.equal, free, same))
    limit = norm / 3

    def clip(params):
        total = sum(float(p.grad.double().square().sum()) for p in params) ** 0.5
        for p in params:
            p.grad.mul_(limit / (total + 1e-6))

    got, _ = run(limit)
    want, _ = run(None, clip)
    for a, b, p in zip(got, want, model.adapter_parameters()):
        # a difference of parameters: their own rounding, and 4 u of the gradient
        assert float((a - b).abs().max()) <= 4 * U * (float(b.abs().max())
                                                      + float(p.abs().max()))


def test_steps_with_a_flat_gradient_buffer(cuda):
    """With the data-parallel gradient sync the gradients are views into one buffer, clipped there
    and kept."""
    from hackathon_b200.dp import AdapterGradSync
    from hackathon_b200.qlora import make_optimizer, policy_step
    model, shape = tiny()
    ids, labels = batch(shape, 4, 64)
    sync = AdapterGradSync(model.adapter_parameters())
    opt = make_optimizer(model)
    norms = []
    opt.register_step_pre_hook(lambda *_: norms.append(float(sync.flat.double().norm())))
    for _ in range(2):
        policy_step(model, opt, ids, labels, None, torch.ones(4, device="cuda:0"),
                    grad_sync=sync, max_grad_norm=1e-4)
    assert all(abs(n - 1e-4) <= 2e-6 for n in norms)
    assert not sync.flat.any()


def test_materialised_logits_to_clipped_head(cuda):
    """The same chain from materialised logits: a trainable head, an entropy bonus, the policy
    loss, clipping; captured into a graph and replayed on another batch. The eager step's graph
    is gone before the capture."""
    from hackathon_b200.grad_norm import clip_grad_norm_
    from hackathon_b200.logprobs import token_logprobs
    from hackathon_b200.policy import policy_loss
    g = torch.Generator(device=cuda).manual_seed(7)
    head = torch.nn.Parameter(torch.randn(500, 64, device=cuda, generator=g) * 0.1)
    h = torch.randn(3, 11, 64, device=cuda, generator=g)
    t = torch.randint(0, 500, (3, 10), device=cuda, generator=g)
    adv = torch.randn(3, device=cuda, generator=g)
    mask = torch.ones(3, 10, dtype=torch.bool, device=cuda)
    mask[2, 4:] = False
    old = torch.full((3, 10), -6.3, device=cuda)
    head.grad = torch.zeros_like(head)

    def step():
        head.grad.zero_()
        logits = h @ head.t()
        logp, entropy = token_logprobs(logits[:, :-1], t, 0.9, True)
        loss, _ = policy_loss(logp, old, adv, mask)
        total = loss - 0.01 * torch.where(mask, entropy, 0.0).sum() / mask.sum()
        (grad,) = torch.autograd.grad(total, head)
        head.grad.add_(grad)
        return total.detach(), clip_grad_norm_(head, 0.01)

    def reference():
        w = head.detach().double().requires_grad_()
        lq = torch.log_softmax((h.double() @ w.t())[:, :-1] / 0.9, -1)
        lp = lq.gather(-1, t[..., None])[..., 0]
        r, a = (lp - old.double()).exp(), adv[:, None].double()
        term = -torch.minimum(r * a, r.clamp(0.8, 1.2) * a)
        ent = -(lq.exp() * lq).sum(-1)
        total = torch.where(mask, term - 0.01 * ent, 0.0).sum() / mask.sum()
        (grad,) = torch.autograd.grad(total, w)
        return total.detach(), grad

    def check(total, norm):
        want, grad = reference()
        n = float(grad.norm())
        # fp32 logits of 64 products, exponentials of them, 30 positions: a few hundred u
        assert abs(float(total) - float(want)) <= 300 * U * max(1.0, abs(float(want)))
        assert abs(float(norm) - n) <= 1000 * U * n
        clipped = grad * min(1.0, 0.01 / (n + 1e-6))
        assert float((head.grad.double() - clipped).norm()) <= 2000 * U * float(clipped.norm())

    check(*step())
    first = head.grad.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total, norm = step()
    graph.replay()
    assert torch.equal(head.grad, first)
    h.copy_(torch.randn(h.shape, device=cuda, generator=g))
    t.copy_(torch.randint(0, 500, t.shape, device=cuda, generator=g))
    graph.replay()
    check(total, norm)


def test_two_threads_at_once(cuda):
    """The operators hold nothing between calls: two threads on two streams get the bits of one."""
    import threading

    from hackathon_b200.grad_norm import clip_grad_norm_
    from hackathon_b200.logprobs import token_logprobs
    from hackathon_b200.policy import policy_loss
    from hackathon_b200.preference import preference_loss

    def chain(seed):
        g = torch.Generator(device=cuda).manual_seed(seed)
        z = torch.randn(4, 40, 3001, device=cuda, generator=g).requires_grad_()
        t = torch.randint(0, 3001, (4, 40), device=cuda, generator=g)
        adv = torch.randn(4, device=cuda, generator=g)
        lp, en = token_logprobs(z, t, 0.8, True)
        loss = policy_loss(lp, lp.detach() * 1.01, adv)[0] + preference_loss(lp)[0] - en.mean()
        loss.backward()
        norm = clip_grad_norm_(z, 1e-3)
        return [loss.detach(), norm, z.grad]

    want = [chain(0), chain(1)]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = chain(k)
                stream.synchronize()
                if not all(map(torch.equal, got, want[k])):
                    wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


def test_inference_mode_checkpoints_and_changed_inputs(cuda):
    """Inference mode gives the same values; a recomputing checkpoint the same gradients; logits
    changed between forward and backward are an error, not another gradient."""
    from torch.utils.checkpoint import checkpoint

    from hackathon_b200.logprobs import token_logprobs
    from hackathon_b200.policy import policy_loss
    g = torch.Generator(device=cuda).manual_seed(3)
    z = torch.randn(3, 20, 777, device=cuda, generator=g).requires_grad_()
    t = torch.randint(0, 777, (3, 20), device=cuda, generator=g)
    adv = torch.randn(3, device=cuda, generator=g)

    def loss_of(logits):
        lp = token_logprobs(logits, t)
        return policy_loss(lp, lp.detach() - 0.1, adv)[0]

    with torch.inference_mode():
        quiet = loss_of(z)
    loss = loss_of(z)
    assert torch.equal(quiet, loss.detach())
    (want,) = torch.autograd.grad(loss, z)
    (got,) = torch.autograd.grad(checkpoint(loss_of, z, use_reentrant=False), z)
    assert torch.equal(got, want)
    x = z.detach() * 1.0
    leaf = x.requires_grad_()
    loss = loss_of(leaf)
    with torch.no_grad():
        leaf.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_labels_outside_the_vocabulary_are_not_scored(cuda):
    """A label of no token takes no part in a step, as -100 takes none."""
    from hackathon_b200.policy import policy_loss
    model, shape = tiny()
    model.train()
    ids, labels = batch(shape, 4, 64)
    odd = labels.clone()
    odd[0, 40:50], odd[2, 60] = shape.vocab, shape.vocab + 9
    odd[1, 20], plain = -1, labels.clone()
    plain[0, 40:50] = plain[2, 60] = plain[1, 20] = -100

    def run(lab):
        logp, _, mask = model.token_logprobs(ids, lab)
        loss, step = policy_loss(logp, logp.detach() - 0.1, torch.ones(4, device="cuda:0"), mask)
        loss.backward()
        got = [logp.detach(), mask, loss.detach(), step.tokens, *grads_of(model)]
        model.zero_grad(set_to_none=True)
        return got

    got, want = run(odd), run(plain)
    assert all(map(torch.equal, got, want)) and int(want[1].sum()) == int(want[3])


def test_steps_keep_the_norm_they_clipped_by(cuda):
    """model.grad_norm: the gradients' norm before clipping, None after a step without clipping."""
    from hackathon_b200.qlora import train_step
    model, shape = tiny()
    ids, labels = batch(shape, 4, 64)
    params = model.adapter_parameters()
    opt = torch.optim.SGD(params, lr=0.0)
    seen = []
    opt.register_step_pre_hook(lambda *_: seen.append(
        math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))))
    assert model.grad_norm is None
    train_step(model, opt, ids, labels, max_grad_norm=1e6)
    norm = float(model.grad_norm)
    assert not model.grad_norm.requires_grad and abs(norm - seen[0]) <= 4 * U * seen[0]
    train_step(model, opt, ids, labels, max_grad_norm=norm / 4)
    assert float(model.grad_norm) == norm and abs(seen[1] - norm / 4) <= 1e-3 * norm
    assert "grad_norm" not in model.state_dict()
    train_step(model, opt, ids, labels)
    assert model.grad_norm is None
