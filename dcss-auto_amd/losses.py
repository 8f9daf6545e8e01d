"""The clipped policy loss with value, entropy and reference-KL terms, and its gradients (csrc/d1_loss.hip).

`policy_loss` is the differentiable function; `policy_loss_grads` gives the loss and its gradients in one pass for
code that runs without autograd. `ppo.ModulePPO` trains on it.
"""
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .ops import call


class PolicyLoss(NamedTuple):
    loss: torch.Tensor                   # fp32, the sum with the coefficients; differentiable
    policy: torch.Tensor                 # fp32 numbers without a gradient, from here on
    value: torch.Tensor                  # half the (clipped) squared error
    entropy: torch.Tensor
    kl: torch.Tensor                     # estimate of KL(policy || reference)
    clipped: torch.Tensor                # the share of the weight whose clip is active
    drift: torch.Tensor                  # estimate of KL(old policy || policy) that is never negative
    count: torch.Tensor                  # tokens that count, or sequences with one (level 'sequence')
    terms: torch.Tensor                  # [8]: all of them; the ones above are its elements, not copies


FP32 = 8                                 # of _call's grads: gradients in fp32


def clip_pair(clip):
    """(low, high) of a pair, or of one number for both."""
    try:
        low, high = clip
    except TypeError:
        low = high = clip
    return float(low), float(high)


def _call(grads, logp, old_logp, advantages, ref_logp, entropy, values, returns, old_values, mask, clip, kl_coef, value_coef,
          value_clip, entropy_coef, level):
    if level not in ('token', 'sequence'):
        raise ValueError(f"level is 'token' or 'sequence', not {level!r}")
    low, high = clip_pair(clip)
    return call('policy_loss', logp, logp, old_logp, advantages, ref_logp, entropy, values, returns, old_values, mask, low, high,
                kl_coef, value_coef, value_clip or 0.0, entropy_coef, level == 'sequence', grads)


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, entropy, values, old_logp, advantages, ref_logp, returns, old_values, mask, settings):
        want = sum(w << k for k, w in enumerate(ctx.needs_input_grad[:3])) | FP32
        # the gradients of the loss come with it, so nothing of the inputs is kept; in fp32, since what stands behind the loss
        # (a loss scale) has to come before a 16-bit type's rounding
        ctx.types = [logp.dtype if t is None else t.dtype for t in (logp, entropy, values)]
        terms, each, *ctx.grads = _call(want, logp, old_logp, advantages, ref_logp, entropy, values, returns, old_values, mask, *settings)
        ctx.mark_non_differentiable(terms)
        return each[0], terms

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        return (*call('scale_grads', dloss, dloss, ctx.grads, ctx.types), *[None] * 7)


def policy_loss(logp, old_logp, advantages, ref_logp=None, entropy=None, values=None, returns=None, old_values=None, mask=None,
                clip=0.2, kl_coef=0.0, value_coef=0.5, value_clip=None, entropy_coef=0.01, level='token'):
    """The clipped policy loss of tokens (actions) logp [..., length] -> PolicyLoss, differentiable in logp, entropy and
    values:

        policy + value_coef * value - entropy_coef * entropy + kl_coef * kl

    old_logp: under the policy that took the tokens. advantages: [..., length], or [...]: one a sequence. clip: the ratio
    exp(logp - old_logp) is held in [1 - clip, 1 + clip], or (low, high) for [1 - low, 1 + high]. ref_logp: under a reference
    policy, for the kl term exp(x) - x - 1 with x = ref_logp - logp. entropy: of each distribution. values and returns:
    half the squared error, with value_clip (None or 0: none) the larger of it and that of the value held within value_clip of old_values.
    mask (bool or uint8): only tokens that are true count, whatever the others hold. level: 'token' weighs all tokens
    alike, 'sequence' the sequences that have one, over their own tokens. All are fp32, bf16 or fp16, each of its own
    type, with any strides; everything is computed in fp32 and summed in fp64. Gradients are kept in fp32 (4 bytes a token
    each) until the backward pass, which multiplies them by the loss's gradient and then rounds them to their input's type, once: a
    launch each that reads and writes them (policy_loss_grads has no such pass). Without a token that counts all terms and
    gradients are 0."""
    settings = (clip, kl_coef, value_coef, value_clip, entropy_coef, level)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (logp, entropy, values)):
        loss, terms = _PolicyLoss.apply(logp, entropy, values, old_logp, advantages, ref_logp, returns, old_values, mask, settings)
        return PolicyLoss(loss, *terms.unbind()[1:], terms)
    terms, each, *_ = _call(0, logp, old_logp, advantages, ref_logp, entropy, values, returns, old_values, mask, *settings)
    return PolicyLoss(*each, terms)


def policy_loss_grads(logp, old_logp, advantages, ref_logp=None, entropy=None, values=None, returns=None, old_values=None, mask=None,
                      clip=0.2, kl_coef=0.0, value_coef=0.5, value_clip=None, entropy_coef=0.01, level='token', fp32_grads=False):
    """-> (PolicyLoss, dlogp, dentropy, dvalues): policy_loss with the gradients of its loss, each like its input, in one
    pass; None where the input is. fp32_grads: all in fp32, for a factor that has to come before the rounding (a weight of 1 / tokens
    leaves fp16 few bits from some 10^5 tokens on, none from 3 x 10^7)."""
    terms, each, *grads = _call(7 | (FP32 if fp32_grads else 0), logp, old_logp, advantages, ref_logp, entropy, values, returns, old_values,
                                mask, clip, kl_coef, value_coef, value_clip, entropy_coef, level)
    return (PolicyLoss(*each, terms), *grads)
