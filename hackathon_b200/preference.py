"""Preference loss over pairs of sequences (paired log ratios), forward and backward."""

import torch

from . import _lib
from .objective_ops import constant, divisor, logp_matrix, mask_bytes, preference

LOSS_TYPES = {"sigmoid": 0, "hinge": 1, "ipo": 2}


class PreferenceStep:
    """What a preference loss leaves for the metrics, on the device: beta times each sequence's
    log ratio, preferred and rejected."""

    def __init__(self, state, rows):
        self.state, self.rows = state, rows     # the op's second output: the rewards come first

    @property
    def chosen_rewards(self):
        return self.state[:self.rows // 2]

    @property
    def rejected_rewards(self):
        return self.state[self.rows // 2:self.rows]

    @property
    def margins(self):
        return self.chosen_rewards - self.rejected_rewards

    @property
    def accuracy(self):
        return (self.chosen_rewards > self.rejected_rewards).float().mean()


def preference_loss(logp, mask=None, ref_logp=None, beta=0.1, loss_type="sigmoid",
                    label_smoothing=0.0, margin=0.0, length_normalized=False, denominator=None):
    """Loss of pairs of sequences from their tokens' log-probabilities, and a PreferenceStep.

    logp [2P, S] (fp32, fp16 or bf16): rows 0 .. P-1 the preferred sequences, P .. 2P-1 the rejected
    ones of the same pairs. mask [2P, S]: the tokens that count (nonzero; all without one); what
    the others hold is never used. ref_logp: the reference model's, per token [2P, S] or already
    summed per sequence [2P] (averaged, if length_normalized; fp64 is kept), or None. With s the
    masked sum of logp - ref_logp (its mean with length_normalized; 0 for a row without tokens),
    D = s_preferred - s_rejected and u = beta * D - margin, a pair's loss is
        sigmoid   -(1 - label_smoothing) * ln sigma(u) - label_smoothing * ln sigma(-u)
        hinge     max(0, 1 - u)
        ipo       (D - 1 / (2 * beta))^2
    and the result their sum / denominator (a number, or a tensor that is not read on the host;
    the number of pairs by default). Differentiable in logp; ref_logp is a constant."""
    logp = logp_matrix("preference_loss", logp)
    n = logp.shape[0]
    if n % 2:
        raise ValueError(f"preference_loss: {n} rows are no pairs")
    if loss_type not in LOSS_TYPES:
        raise ValueError(f"preference_loss: loss_type {loss_type!r} is none of "
                         f"{sorted(LOSS_TYPES)}")
    beta, smoothing, margin = float(beta), float(label_smoothing), float(margin)
    if not 0.0 < beta < float("inf"):
        raise ValueError(f"preference_loss: beta {beta} is not positive")
    if not 0.0 <= smoothing < 0.5 or (smoothing and loss_type != "sigmoid"):
        raise ValueError("preference_loss: label_smoothing is in [0, 0.5), for the sigmoid loss")
    if not abs(margin) < float("inf") or (margin and loss_type == "ipo"):
        raise ValueError("preference_loss: the margin is a finite number, and not for ipo")
    mask = mask_bytes("preference_loss", mask, logp)
    ref = ref_row = None
    if ref_logp is not None:
        constant("preference_loss", "ref_logp", ref_logp, logp)
        if ref_logp.shape == logp.shape:
            dtype = torch.promote_types(logp.dtype, ref_logp.dtype)
            logp, ref = logp.to(dtype), ref_logp.to(dtype).contiguous()
            _lib.tag(dtype)
        elif ref_logp.shape == (n,):
            wide = ref_logp.dtype == torch.float64      # long sums keep their 64 bits
            ref_row = ref_logp.to(torch.float64 if wide else torch.float32).contiguous()
        else:
            raise ValueError(f"preference_loss: ref_logp {tuple(ref_logp.shape)} for logp "
                             f"{tuple(logp.shape)}")
    denom, divide_by = divisor("preference_loss", denominator, logp.device)
    loss, state = preference(
        logp.contiguous(), mask, ref, ref_row, denom, beta, smoothing, margin, divide_by,
        LOSS_TYPES[loss_type], bool(length_normalized))
    return loss, PreferenceStep(state, n)
