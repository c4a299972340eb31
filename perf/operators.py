"""The post-training operators as measured work: log-probabilities of chosen tokens, the preference and
the clipped policy objective over them, and the global gradient norm with clipping.

`run` computes a case in its plain form (elementary torch operations), or, where `own` is true, through
this package's operators."""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
IGNORE = -100


def listed():
    return [
        # one sampled token of each of 8 sequences scored as it is generated: the smallest call
        {"name": "logprobs 8 x 1", "op": "logprobs", "batch": 8, "seq": 1, "vocab": 151936,
         "dtype": "bf16", "temperature": 1.0, "entropy": True, "grad": False, "shift": False,
         "banned": 0},
        # scoring rollouts or a preference batch under a frozen model: no gradient
        {"name": "logprobs 4 x 1024", "op": "logprobs", "batch": 4, "seq": 1024, "vocab": 152064,
         "dtype": "bf16", "temperature": 1.0, "entropy": False, "grad": False, "shift": False,
         "banned": 0},
        # the training pass on next-token logits (a view that drops the last position), with an
        # entropy bonus and the vocabulary's padding at -inf
        {"name": "logprobs 4 x 1023 train", "op": "logprobs", "batch": 4, "seq": 1023,
         "vocab": 151936, "dtype": "bf16", "temperature": 1.0, "entropy": True, "grad": True,
         "shift": True, "banned": 271},
        # fp32 logits of an odd vocabulary at a sampling temperature
        {"name": "logprobs 3 x 333 odd train", "op": "logprobs", "batch": 3, "seq": 333,
         "vocab": 50001, "dtype": "fp32", "temperature": 0.7, "entropy": False, "grad": True,
         "shift": False, "banned": 0},
        # a small preference batch with per-token reference log-probabilities
        {"name": "preference 4 x 512", "op": "preference", "pairs": 4, "seq": 512,
         "dtype": "fp32", "loss": "sigmoid", "smoothing": 0.0, "ref": "token",
         "normalized": False},
        # a large batch of long pairs, length-normalised, reference sums kept per sequence
        {"name": "preference 31 x 16383", "op": "preference", "pairs": 31, "seq": 16383,
         "dtype": "fp32", "loss": "ipo", "smoothing": 0.0, "ref": "sequence",
         "normalized": True},
        # one prompt's group of short rollouts, one advantage per rollout, KL to the reference
        {"name": "policy 16 x 333", "op": "policy", "rollouts": 16, "seq": 333, "dtype": "fp32",
         "token_advantages": False, "kl": 0.04, "delta": 0.0, "reduction": "token"},
        # a large batch of rollouts, per-sequence means, no reference model
        {"name": "policy 512 x 4096", "op": "policy", "rollouts": 512, "seq": 4096,
         "dtype": "fp32", "token_advantages": False, "kl": 0.0, "delta": 0.0,
         "reduction": "sequence"},
        # a few very long rollouts with an advantage for each token and the two-sided clip
        {"name": "policy 8 x 32768", "op": "policy", "rollouts": 8, "seq": 32768,
         "dtype": "fp32", "token_advantages": True, "kl": 0.02, "delta": 4.0,
         "reduction": "token"},
        # the adapters of the 0.5B configuration (rank 16), clipped
        {"name": "clip 0.5b adapters", "op": "clip", "layers": 24, "hidden": 896, "inter": 4864,
         "kv": 128, "rank": 16, "dtype": "fp32", "odd": False, "binding": True},
        # the adapters of the 7B configuration (rank 64), clipped
        {"name": "clip 7b adapters", "op": "clip", "layers": 28, "hidden": 3584, "inter": 18944,
         "kv": 512, "rank": 64, "dtype": "fp32", "odd": False, "binding": True},
        # bf16 gradients at odd addresses in one buffer, the norm within the limit: a step that
        # has to leave every gradient as it is
        {"name": "clip bf16 odd within", "op": "clip", "layers": 28, "hidden": 1536,
         "inter": 8960, "kv": 256, "rank": 15, "dtype": "bf16", "odd": True, "binding": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("logprobs", "logprobs", "preference", "policy", "clip"))
    if op == "logprobs":
        vocab = _log(rng, 1000, 152064)
        rows = _log(rng, 1, max(2, min(8192, 600_000_000 // vocab)))
        batch = rng.randint(1, max(1, min(8, rows)))
        grad = rng.random() < 0.6
        if grad:
            rows = max(1, min(rows, 300_000_000 // vocab))
            batch = min(batch, rows)
        return {"op": op, "batch": batch, "seq": max(1, rows // batch), "vocab": vocab,
                "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")),
                "temperature": rng.choice((1.0, 0.7, round(rng.uniform(0.5, 1.5), 3))),
                "entropy": rng.random() < 0.5, "grad": grad, "shift": rng.random() < 0.5,
                "banned": rng.choice((0, 0, rng.randint(1, vocab // 4)))}
    if op == "preference":
        seq = _log(rng, 1, 32768)
        loss = rng.choice(("sigmoid", "sigmoid", "hinge", "ipo"))
        return {"op": op, "pairs": _log(rng, 1, max(2, min(512, 1_000_000 // seq))), "seq": seq,
                "dtype": rng.choice(("fp32", "fp32", "bf16")), "loss": loss,
                "smoothing": rng.choice((0.0, 0.1)) if loss == "sigmoid" else 0.0,
                "ref": rng.choice(("none", "token", "sequence")),
                "normalized": rng.random() < 0.4}
    if op == "policy":
        seq = _log(rng, 1, 32768)
        return {"op": op, "rollouts": _log(rng, 1, max(2, min(1024, 2_000_000 // seq))),
                "seq": seq, "dtype": rng.choice(("fp32", "fp32", "bf16")),
                "token_advantages": rng.random() < 0.4,
                "kl": rng.choice((0.0, 0.001, 0.04)), "delta": rng.choice((0.0, 4.0)),
                "reduction": rng.choice(("token", "sequence"))}
    hidden = 8 * _log(rng, 16, 448)
    return {"op": op, "layers": rng.randint(1, 28), "hidden": hidden,
            "inter": hidden * rng.randint(2, 5), "kv": max(8, hidden // rng.choice((4, 7, 8))),
            "rank": _log(rng, 1, 64), "dtype": rng.choice(("fp32", "fp32", "bf16", "fp16")),
            "odd": rng.random() < 0.5, "binding": rng.random() < 0.6}


def _adapter_shapes(c):
    h, i, kv, r = c["hidden"], c["inter"], c["kv"], c["rank"]
    io = [(h, h), (h, kv), (h, kv), (h, h), (h, i), (h, i), (i, h)]
    return [s for _ in range(c["layers"]) for a, b in io for s in ((r, a), (b, r))]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda", torch.cuda.current_device())
    c = case
    dt = DTYPES[c["dtype"]]

    def rand(*s):
        return torch.rand(*s, device=dev, generator=g)

    def randn(*s):
        return torch.randn(*s, device=dev, generator=g)

    if c["op"] == "logprobs":
        b, s, v = c["batch"], c["seq"], c["vocab"]
        full = torch.empty(b, s + c["shift"], v, dtype=dt, device=dev)
        full.normal_(0.0, 2.5, generator=g)
        if c["banned"]:
            full[..., v - c["banned"]:] = -math.inf
        logits = full[:, :s]
        target = torch.randint(0, v - c["banned"], (b, s), device=dev, generator=g)
        # a trained model gives most of its chosen tokens a large share
        logits.scatter_add_(2, target[..., None], (rand(b, s, 1) * 16).to(dt))
        if c["grad"]:       # the prompt's positions are not scored
            target[:, : s // 4] = IGNORE
        return {"case": c, "full": full, "logits": logits.requires_grad_(c["grad"]),
                "target": target, "g_logp": randn(b, s) / (b * s),
                "g_entropy": (randn(b, s) * 0.01 - 0.01) / (b * s)}
    if c["op"] in ("preference", "policy"):
        n = 2 * c["pairs"] if c["op"] == "preference" else c["rollouts"]
        s = c["seq"]
        logp = (-3.0 * rand(n, s) ** 3 - 0.01).to(dt)
        ref = (logp.float() + 0.1 * randn(n, s)).to(dt)
        # a prompt that is not scored, then an answer of its own length, then padding
        start = (rand(n, 1) * (s * 0.25)).long()
        stop = start + 1 + (rand(n, 1) * (s - start)).long()
        at = torch.arange(s, device=dev)
        state = {"case": c, "logp": logp.requires_grad_(), "mask": (at >= start) & (at < stop)}
        if c["op"] == "preference":
            m = state["mask"]
            state["ref"] = None
            if c["ref"] == "token":
                state["ref"] = ref
            elif c["ref"] == "sequence":
                total = torch.where(m, ref.double(), 0.0).sum(1)
                state["ref"] = (total / m.sum(1).clamp(min=1) if c["normalized"] else total).float()
        else:
            state["old"] = (logp.detach().float() + 0.15 * randn(n, s)).to(dt)
            state["ref"] = ref if c["kl"] else None
            state["advantages"] = randn(n, s) if c["token_advantages"] else randn(n)
        return state
    shapes = _adapter_shapes(c)
    sizes = [a * b for a, b in shapes]
    gap = 1 if c["odd"] else 0
    flat = torch.zeros(sum(sizes) + gap * len(sizes), dtype=dt, device=dev)
    flat.normal_(0.0, 1e-3, generator=g)
    params, at = [], 0
    for (a, b), n in zip(shapes, sizes):
        flat[at: at + gap] = 0
        p = torch.nn.Parameter(torch.empty(a, b, dtype=dt, device=dev))
        p.grad = flat[at + gap: at + gap + n].view(a, b)
        params.append(p)
        at += gap + n
    # A limit below the 1e-6 of the formula's denominator clips every pass again, however often
    # the same gradients are clipped; one far above every norm never does.
    return {"case": c, "flat": flat, "params": params, "max_norm": 1e-6 if c["binding"] else 1e6}


# ---------------------------------------------------------------------------------------------
# the plain forms


def _plain_logprobs(s):
    c = s["case"]
    z = s["logits"].float()
    target = s["target"]
    scored = target != IGNORE
    y = torch.where(scored, target, 0)[..., None]
    x = (z - z.amax(-1, keepdim=True)) / c["temperature"]
    e = x.exp()
    total = e.sum(-1, keepdim=True)
    logq = x - total.log()                    # log-probabilities of the whole vocabulary
    logp = torch.where(scored, logq.gather(-1, y)[..., 0], 0.0)
    out = {"logp": logp}
    q = e / total
    if c["entropy"]:
        out["entropy"] = -torch.where(q > 0, q * logq, 0.0).sum(-1)
    if c["grad"]:
        gl = torch.where(scored, s["g_logp"], 0.0)[..., None]
        dz = -gl * q
        dz.scatter_add_(-1, y, gl)
        if c["entropy"]:
            dz -= torch.where(q > 0, s["g_entropy"][..., None] * q
                              * (logq + out["entropy"][..., None]), 0.0)
        out["grad"] = (dz / c["temperature"]).to(s["logits"].dtype)
    return out


def _plain_preference(s):
    c, m = s["case"], s["mask"]
    beta, p = 0.1, c["pairs"]
    d = s["logp"].double()
    if c["ref"] == "token":
        d = d - s["ref"].double()
    n = m.sum(1).clamp(min=1) if c["normalized"] else torch.ones_like(m[:, 0], dtype=torch.long)
    total = torch.where(m, d, 0.0).sum(1) / n
    if c["ref"] == "sequence":
        total = total - s["ref"].double()
    diff = total[:p] - total[p:]
    u = beta * diff
    eps = c["smoothing"]
    if c["loss"] == "sigmoid":
        pos, neg = torch.logaddexp(-u, torch.zeros_like(u)), torch.logaddexp(u, torch.zeros_like(u))
        loss = (1 - eps) * pos + eps * neg
        slope = beta * (eps / (1 + (-u).exp()) - (1 - eps) / (1 + u.exp()))
    elif c["loss"] == "hinge":
        loss, slope = (1 - u).clamp(min=0), torch.where(u < 1, -beta, 0.0).double()
    else:
        off = diff - 1 / (2 * beta)
        loss, slope = off * off, 2 * off
    row = torch.cat([slope, -slope]) / (p * n)
    return {"loss": loss.mean().float(), "chosen": (beta * total[:p]).float(),
            "rejected": (beta * total[p:]).float(),
            "grad": torch.where(m, row[:, None], 0.0).to(s["logp"].dtype)}


LOW, HIGH = 0.2, 0.28


def _plain_policy(s):
    c, m = s["case"], s["mask"]
    a = s["advantages"] if c["token_advantages"] else s["advantages"][:, None]
    lr = s["logp"].double() - s["old"].double()     # 64 bits: the gradient jumps at the border
    r = lr.float().exp()
    first = r.clamp(max=c["delta"]) if c["delta"] else r
    loss = -torch.minimum(first * a, r.clamp(1 - LOW, 1 + HIGH) * a)
    below, above = lr < math.log(1 - LOW), lr > math.log(1 + HIGH)
    live = ~(below | above) | (below & (a > 0)) | (above & (a < 0))
    if c["delta"]:
        live = live & (lr <= math.log(c["delta"]))
    grad = torch.where(live, -a * r, 0.0)
    count = m.sum(1)
    tokens = count.sum()
    per = tokens.clamp(min=1)
    out = {}
    if c["kl"]:
        d = s["ref"].double() - s["logp"].double()  # 64 bits: e^d - d - 1 cancels for small d
        kl = (torch.expm1(d) - d).float()
        loss = loss + c["kl"] * kl
        grad = grad - c["kl"] * torch.expm1(d).float()
        out["kl"] = (torch.where(m, kl, 0.0).double().sum() / per).float()
    rows = torch.where(m, loss, 0.0).double().sum(1)
    if c["reduction"] == "token":
        out["loss"] = (rows.sum() / per).float()
        weight = (1.0 / per).float()
    else:
        each = count.clamp(min=1)
        out["loss"] = (rows / each).mean().float()
        weight = (1.0 / (each * c["rollouts"]))[:, None].float()
    out["grad"] = torch.where(m, grad * weight, 0.0).to(s["logp"].dtype)
    out["clipped_low"] = ((m & below & (a < 0)).sum() / per).float()
    out["clipped_high"] = ((m & above & (a > 0)).sum() / per).float()
    return out


def _plain_clip(s):
    grads = [p.grad for p in s["params"]]
    squares = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads])
    norm = squares.sum().sqrt()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    [g.copy_(g.float() * coef) for g in grads]
    return {"norm": norm.float(), "grads": s["flat"]}


def run(state):
    c = state["case"]
    if own:
        return _own(state)
    with torch.no_grad():
        return {"logprobs": _plain_logprobs, "preference": _plain_preference,
                "policy": _plain_policy, "clip": _plain_clip}[c["op"]](state)


# ---------------------------------------------------------------------------------------------
# the framework's operators


def _own(s):
    c = s["case"]
    if c["op"] == "logprobs":
        from hackathon_b200.logprobs import token_logprobs
        if not c["grad"]:
            with torch.no_grad():
                got = token_logprobs(s["logits"], s["target"], c["temperature"], c["entropy"])
            return {"logp": got[0], "entropy": got[1]} if c["entropy"] else {"logp": got}
        got = token_logprobs(s["logits"], s["target"], c["temperature"], c["entropy"])
        if c["entropy"]:
            (grad,) = torch.autograd.grad(got, s["logits"], (s["g_logp"], s["g_entropy"]))
            return {"logp": got[0].detach(), "entropy": got[1].detach(), "grad": grad}
        (grad,) = torch.autograd.grad(got, s["logits"], s["g_logp"])
        return {"logp": got.detach(), "grad": grad}
    if c["op"] == "preference":
        from hackathon_b200.preference import preference_loss
        loss, step = preference_loss(s["logp"], s["mask"], s["ref"], beta=0.1,
                                     loss_type=c["loss"], label_smoothing=c["smoothing"],
                                     length_normalized=c["normalized"])
        (grad,) = torch.autograd.grad(loss, s["logp"])
        return {"loss": loss.detach(), "chosen": step.chosen_rewards,
                "rejected": step.rejected_rewards, "grad": grad}
    if c["op"] == "policy":
        from hackathon_b200.policy import policy_loss
        loss, step = policy_loss(s["logp"], s["old"], s["advantages"], s["mask"], s["ref"],
                                 clip_low=LOW, clip_high=HIGH, delta=c["delta"] or None,
                                 kl_coef=c["kl"], reduction=c["reduction"])
        (grad,) = torch.autograd.grad(loss, s["logp"])
        out = {"loss": loss.detach(), "grad": grad, "clipped_low": step.clipped_low,
               "clipped_high": step.clipped_high}
        if c["kl"]:
            out["kl"] = step.kl
        return out
    from hackathon_b200.grad_norm import clip_grad_norm_
    norm = clip_grad_norm_(s["params"], s["max_norm"])
    return {"norm": norm, "grads": s["flat"]}


# ---------------------------------------------------------------------------------------------


def work(case):
    c = case
    e = 2 if c["dtype"] != "fp32" else 4
    if c["op"] == "logprobs":
        n = c["batch"] * c["seq"]
        logits = n * c["vocab"] * e
        small = n * (8 + 4 + (4 if c["entropy"] else 0))
        if c["grad"]:
            return {"bytes": 2 * logits + small + n * (8 if c["entropy"] else 4),
                    "flops": n * c["vocab"] * (12 if c["entropy"] else 8)}
        return {"bytes": logits + small, "flops": n * c["vocab"] * (6 if c["entropy"] else 4)}
    if c["op"] == "preference":
        n = 2 * c["pairs"] * c["seq"]
        return {"bytes": n * (e * (3 if c["ref"] == "token" else 2) + 1) + c["pairs"] * 16,
                "flops": n * 3}
    if c["op"] == "policy":
        n = c["rollouts"] * c["seq"]
        per = 3 * e + 1 + (e if c["kl"] else 0) + (4 if c["token_advantages"] else 0)
        return {"bytes": n * per + c["rollouts"] * 4, "flops": n * 20}
    n = sum(a * b for a, b in _adapter_shapes(c))
    return {"bytes": n * e * (2 if c["binding"] else 1), "flops": n * (3 if c["binding"] else 2)}


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    with torch.no_grad():
        if c["op"] == "logprobs":
            return _exact_logprobs(c, s)
        if c["op"] == "preference":
            return _exact_preference(c, s)
        if c["op"] == "policy":
            return _exact_policy(c, s)
        g = s["flat"].double()
        norm = torch.linalg.vector_norm(g)
        return {"norm": norm, "grads": g * min(1.0, s["max_norm"] / (float(norm) + 1e-6))}


def _exact_logprobs(c, s):
    b, n, v = c["batch"], c["seq"], c["vocab"]
    logp = torch.empty(b * n, dtype=torch.float64, device=s["target"].device)
    entropy = torch.empty_like(logp)
    grad = torch.empty(b * n, v, dtype=torch.float64, device=logp.device) if c["grad"] else None
    rows = s["logits"].detach().reshape(b * n, v)
    target, gl, ge = s["target"].reshape(-1), s["g_logp"].reshape(-1), s["g_entropy"].reshape(-1)
    step = max(1, 200_000_000 // v)
    for at in range(0, b * n, step):
        part = slice(at, at + step)
        lq = torch.log_softmax(rows[part].double() / c["temperature"], -1)
        q = torch.softmax(rows[part].double() / c["temperature"], -1)
        t = target[part]
        ok = t >= 0
        pick = torch.arange(t.numel(), device=t.device)
        logp[part] = lq[pick, t.clamp(min=0)].masked_fill(~ok, 0.0)
        entropy[part] = torch.special.entr(q).sum(-1)
        if c["grad"]:
            w = gl[part].double() * ok
            dz = -w[:, None] * q
            dz[pick, t.clamp(min=0)] += w
            if c["entropy"]:
                dz += ge[part].double()[:, None] * (torch.special.entr(q)
                                                    - q * entropy[part][:, None])
            grad[part] = dz / c["temperature"]
    out = {"logp": logp.view(b, n)}
    if c["entropy"]:
        out["entropy"] = entropy.view(b, n)
    if c["grad"]:
        out["grad"] = grad.view(b, n, v)
    return out


def _exact_preference(c, s):
    beta, p = 0.1, c["pairs"]
    leaf = s["logp"].detach().double().requires_grad_()
    with torch.enable_grad():
        keep = s["mask"].double()
        size = keep.sum(1).clamp(min=1.0)
        given = s["ref"].double() if s["ref"] is not None else torch.zeros((), dtype=torch.float64,
                                                                          device=leaf.device)
        total = (leaf * keep).sum(1)
        if c["ref"] == "token":
            total = total - (given * keep).sum(1)
        if c["normalized"]:
            total = total / size
        if c["ref"] == "sequence":
            total = total - given
        reward = beta * total
        gap = reward[:p] - reward[p:]
        if c["loss"] == "sigmoid":
            ls = torch.nn.functional.logsigmoid
            each = -(1 - c["smoothing"]) * ls(gap) - c["smoothing"] * ls(-gap)
        elif c["loss"] == "hinge":
            each = torch.relu(1 - gap)
        else:
            each = (gap / beta - 0.5 / beta) ** 2
        loss = each.mean()
    (grad,) = torch.autograd.grad(loss, leaf)
    return {"loss": loss.detach(), "chosen": reward[:p].detach(), "rejected": reward[p:].detach(),
            "grad": grad}


def _exact_policy(c, s):
    leaf = s["logp"].detach().double().requires_grad_()
    keep = s["mask"].double()
    adv = s["advantages"].double()
    adv = adv if c["token_advantages"] else adv[:, None].expand_as(keep)
    with torch.enable_grad():
        ratio = torch.exp(leaf - s["old"].double())
        free = torch.clamp(ratio, max=c["delta"]) if c["delta"] else ratio
        held = torch.clamp(ratio, 1 - LOW, 1 + HIGH)
        each = torch.maximum(-free * adv, -held * adv)
        kl = None
        if c["kl"]:
            away = s["ref"].double() - leaf
            kl = torch.expm1(away) - away
            each = each + c["kl"] * kl
        if c["reduction"] == "token":
            loss = (each * keep).sum() / keep.sum().clamp(min=1.0)
        else:
            loss = ((each * keep).sum(1) / keep.sum(1).clamp(min=1.0)).sum() / c["rollouts"]
    (grad,) = torch.autograd.grad(loss, leaf)
    total = keep.sum().clamp(min=1.0)
    low = (keep * ((ratio < 1 - LOW) & (adv < 0))).sum() / total
    high = (keep * ((ratio > 1 + HIGH) & (adv > 0))).sum() / total
    out = {"loss": loss.detach(), "grad": grad, "clipped_low": low.detach(),
           "clipped_high": high.detach()}
    if kl is not None:
        out["kl"] = (kl.detach() * keep).sum() / total
    return out
