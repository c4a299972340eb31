"""Clipped policy loss with a KL term over sampled tokens, forward and backward."""

import torch

from . import _lib
from .objective_ops import constant, divisor, logp_matrix, mask_bytes, policy, transformed

REDUCTIONS = ("token", "sequence")


class PolicyStep:
    """What a policy loss leaves for the metrics, on the device: the number of tokens that count,
    the mean KL estimate over them (0 without a reference), and the shares of them whose gradient
    the lower and the upper border of the ratio hold."""

    def __init__(self, state):
        self.state = state          # the op's second output: the statistics come first

    @property
    def tokens(self):
        return self.state[0]

    @property
    def kl(self):
        return self.state[1]

    @property
    def clipped_low(self):
        return self.state[2]

    @property
    def clipped_high(self):
        return self.state[3]


def policy_loss(logp, old_logp, advantages, mask=None, ref_logp=None, clip_low=0.2,
                clip_high=None, delta=None, kl_coef=0.0, reduction="token", denominator=None):
    """Clipped policy loss of sampled tokens from their log-probabilities, and a PolicyStep.

    logp [N, S] (fp32, fp16 or bf16); old_logp [N, S] of the policy that sampled them (None: logp
    itself, a ratio of 1); advantages [N] or [N, S]; mask [N, S]: the tokens that count (nonzero;
    all without one), what the others hold is never used. With r = exp(logp - old_logp) and
    d = ref_logp - logp a token's loss is
        -min(min(r, delta) * A, clamp(r, 1 - clip_low, 1 + clip_high) * A)
            + kl_coef * (exp(d) - d - 1)
    (clip_high None: clip_low; delta None: no second border; the KL term with a ref_logp only).
    reduction "token": their sum / denominator, by default the number of tokens that count;
    "sequence": the sum of the rows' means (0 for a row without tokens) / denominator, by default
    N. The denominator is a number, or a tensor that is not read on the host. Differentiable in
    logp; everything else is a constant. Without a ref_logp the kl_coef has to be 0."""
    logp = logp_matrix("policy_loss", logp)
    n, s = logp.shape
    clip_low = float(clip_low)
    clip_high = clip_low if clip_high is None else float(clip_high)
    if not 0.0 <= clip_low <= 1.0 or not 0.0 <= clip_high < float("inf"):
        raise ValueError(f"policy_loss: clip range {clip_low}, {clip_high}")
    delta = None if delta is None else float(delta)
    if delta is not None and not 1.0 + clip_high < delta < float("inf"):
        raise ValueError(f"policy_loss: delta {delta} is not above 1 + clip_high")
    kl_coef = float(kl_coef)
    if not abs(kl_coef) < float("inf") or (kl_coef and ref_logp is None):
        raise ValueError("policy_loss: kl_coef is a finite number, and needs a ref_logp")
    if reduction not in REDUCTIONS:
        raise ValueError(f"policy_loss: reduction {reduction!r} is none of {REDUCTIONS}")
    dtype = logp.dtype
    for name, t in (("old_logp", old_logp), ("ref_logp", ref_logp)):
        if t is None:
            continue
        constant("policy_loss", name, t, logp)
        if t.shape != logp.shape:
            raise ValueError(f"policy_loss: {name} {tuple(t.shape)} for logp "
                             f"{tuple(logp.shape)}")
        dtype = torch.promote_types(dtype, t.dtype)
    _lib.tag(dtype)
    constant("policy_loss", "advantages", advantages, logp)
    if advantages.shape not in ((n,), (n, s)):
        raise ValueError(f"policy_loss: advantages {tuple(advantages.shape)} for logp "
                         f"{tuple(logp.shape)}")
    mask = mask_bytes("policy_loss", mask, logp)
    denom, divide_by = divisor("policy_loss", denominator, logp.device)
    # a tensor inside a function transform does not say whether the one it stands for asks for one
    with_grad = torch.is_grad_enabled() and (logp.requires_grad or transformed())
    loss, state, _ = policy(
        logp.to(dtype).contiguous(),
        None if old_logp is None else old_logp.to(dtype).contiguous(),
        advantages.to(torch.float32), mask,
        None if ref_logp is None else ref_logp.to(dtype).contiguous(), denom, clip_low, clip_high,
        delta or 0.0, kl_coef, divide_by, reduction == "sequence", with_grad)
    return loss, PolicyStep(state)
