"""Log probabilities of given tokens (actions) with entropy, top alternatives and gradient.

`token_logprobs` is what a policy's loss and its evaluation need of a row of logits, in one pass
over it (csrc/d1_tokens.hip): the log probability of the token that was taken, the distribution's
entropy and, where asked, its most probable entries. It is differentiable in the logits through
logp and entropy; `token_logprobs_bwd` is that gradient for code that runs without autograd.
"""
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from .ops import call, is_tracing


class TokenLogprobs(NamedTuple):
    logp: torch.Tensor                   # fp32 [...]: log probability of the given token
    entropy: torch.Tensor                # fp32 [...]
    top_ids: Optional[torch.Tensor]      # int64 [..., top], falling probability, lowest index first; -1: none
    top_logp: Optional[torch.Tensor]     # fp32 [..., top]
    stats: torch.Tensor                  # fp32 [..., 2]: largest entry and sum of exponentials about it

    @property
    def lse(self):
        """log sum exp of each row's allowed logits (without a gradient)."""
        return self.stats[..., 0] + self.stats[..., 1].log()


def _forward(logits, tokens, mask, top):
    if type(top) is not int:
        raise ValueError(f'top must be an int, not {top!r}')
    return TokenLogprobs(*call('tokens_fwd', logits, logits, tokens, mask, top))


def token_logprobs_bwd(logits, tokens, result, dlogp, dentropy, mask=None):
    """The gradient of the logits (their type, contiguous) from those of logp and entropy (fp32 of
    their shapes; either may be None: zero); `result` is token_logprobs' of the same arguments."""
    return call('tokens_bwd', logits, logits, tokens, result.stats, result.entropy, dlogp, dentropy, mask)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, top):
        r = _forward(logits, tokens, mask, top)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, tokens, mask, r.entropy, r.stats)
        ctx.mark_non_differentiable(*(t for t in (r.top_ids, r.top_logp, r.stats) if t is not None))
        return tuple(r)

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp, dentropy, *_):
        logits, tokens, mask, entropy, stats = ctx.saved_tensors
        if dlogp is None and dentropy is None:
            return None, None, None, None
        r = TokenLogprobs(None, entropy, None, None, stats)
        return token_logprobs_bwd(logits, tokens, r, dlogp, dentropy, mask=mask), None, None, None


def token_logprobs(logits, tokens, mask=None, top=0):
    """Log probability of tokens [...] (int64) under softmax(logits [..., V]), with the entropy and
    the `top` (0 to 64) most probable entries of each row -> TokenLogprobs.

    logits: fp32, bf16 or fp16 (rows of any stride); everything is computed and returned in fp32.
    mask: bool or uint8, [..., V] or [V]; only entries that are true take part. A negative token is
    padding (logp 0, no gradient through it), a token of V or more gives NaN, a masked one -inf. A
    row that allows nothing gives logp -inf, entropy 0, no alternatives and a gradient of 0."""
    if is_tracing() or torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, mask, top))
    return _forward(logits, tokens, mask, top)
