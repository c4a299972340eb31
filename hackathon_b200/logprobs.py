"""Log-probabilities of chosen tokens: what the preference and the policy objective are made of.

    token_logprobs(logits, target)                from materialised logits, differentiable in
                                                  the log-probability and the entropy
    linear_token_logprobs(hidden, weight, target) from hidden states and a frozen head, without
                                                  the logits (the linear cross-entropy's kernels)
"""

import torch

from . import _common, _lib, objective_ops
from .cross_entropy import CHUNK_ROWS, FusedLinearCrossEntropy


def _whole_numbers(what, target):
    if target.is_floating_point() or target.is_complex() or target.dtype == torch.bool:
        raise TypeError(f"{what}: target holds token numbers, got {target.dtype}")


def token_logprobs(logits, target, temperature=1.0, with_entropy=False):
    """ln softmax(logits / temperature)[target] per position, fp32, and with_entropy the pair of it
    and the entropy of softmax(logits / temperature). logits [..., V] in fp32, fp16 or bf16,
    target [...] whole numbers; a target outside [0, V) (IGNORE_INDEX) scores 0 and has no
    gradient, its entropy counts as any other's. Both outputs are differentiable in the logits,
    whose gradient is contiguous and in their dtype. Logits of -inf have probability 0; a row of
    nothing else is NaN. Up to two leading dimensions of any strides are read in place."""
    _lib.require_cuda(logits, target, what="token_logprobs")
    _lib.tag(logits.dtype)
    if logits.dim() < 1 or logits.shape[:-1] != target.shape or logits.shape[-1] == 0:
        raise ValueError(f"token_logprobs: logits {tuple(logits.shape)} for target "
                         f"{tuple(target.shape)}")
    if target.device != logits.device:
        raise ValueError(f"token_logprobs: target on {target.device}, logits on {logits.device}")
    _whole_numbers("token_logprobs", target)
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"token_logprobs: temperature {temperature} is not in 1e-6 .. 1e6")
    if target.dtype != torch.int64:
        target = target.to(torch.int64)
    logp, entropy, _ = objective_ops.token_logprobs(logits, target, temperature,
                                                    bool(with_entropy))
    return (logp, entropy) if with_entropy else logp


def linear_token_logprobs(hidden, weight, target, chunk_rows=CHUNK_ROWS):
    """(ln softmax(hidden @ weight.T)[target], entropy) per position, fp32, without the logits:
    the linear cross-entropy's kernels, whose per-token loss is the negative log-probability. The
    log-probability is differentiable in the hidden states; the entropy is a constant and the
    head is frozen. hidden [..., H], weight [V, H], target [...]; a target outside [0, V)
    (IGNORE_INDEX) scores 0 and has no gradient."""
    _lib.require_cuda(hidden, weight, target, what="linear_token_logprobs")
    if (hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]
            or target.shape != hidden.shape[:-1]):
        raise ValueError(f"linear_token_logprobs: hidden {tuple(hidden.shape)} and weight "
                         f"{tuple(weight.shape)} for target {tuple(target.shape)}")
    _whole_numbers("linear_token_logprobs", target)
    objective_ops.refuse_tangents("linear_token_logprobs", (hidden, weight))
    matmul_dtype = _common.autocast_dtype() or torch.promote_types(hidden.dtype, weight.dtype)
    _, token_loss, entropy, _ = FusedLinearCrossEntropy.apply(hidden, weight, target, 1,
                                                              matmul_dtype, chunk_rows)
    return -token_loss, entropy
