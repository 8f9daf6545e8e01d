"""Log probabilities of given tokens (actions) with entropy, top alternatives and gradient.

`token_logprobs` is what a policy's loss and its evaluation need of a row of logits, in one pass
over it (csrc/d1_tokens.hip): the log probability of the token that was taken, the distribution's
entropy and, where asked, its most probable entries. It is differentiable in the logits through
logp and entropy; `token_logprobs_bwd` is that gradient for code that runs without autograd.
"""
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .rows import as_rows, call, like, type_of

MAX_TOP, MAX_VOCAB = 64, 1 << 24
UNSPLIT_VOCAB = 1024       # rows up to this are never cut into segments: no scratch memory


class TokenLogprobs(NamedTuple):
    logp: torch.Tensor                   # fp32 [...]: log probability of the given token
    entropy: torch.Tensor                # fp32 [...]
    top_ids: Optional[torch.Tensor]      # int64 [..., top], falling probability, lowest index first; -1: none
    top_logp: Optional[torch.Tensor]     # fp32 [..., top]
    stats: torch.Tensor                  # fp32 [..., 2]: largest entry and sum of exponentials about it

    @property
    def lse(self):
        """log sum exp of each row's allowed logits."""
        return self.stats[..., 0] + self.stats[..., 1].log()


def _check(logits, tokens, mask):
    """-> (logits as rows, tokens contiguous, mask as rows, its data pointer, its row stride)."""
    vocab, index = logits.shape[-1], logits.get_device()
    if vocab > MAX_VOCAB:
        raise ValueError(f'logits: at most {MAX_VOCAB} entries a row')
    tokens = like(tokens, logits.shape[:-1], index, 'tokens', torch.int64)
    rows = as_rows(logits)
    if mask is None:
        return rows, tokens, None, None, 0
    if mask.dtype not in (torch.bool, torch.uint8) or mask.get_device() != index:
        raise ValueError('mask must be bool or uint8 on the device of the logits')
    if mask.shape == logits.shape:
        mask = as_rows(mask)
        return rows, tokens, mask, mask.data_ptr(), mask.stride(0)
    if mask.shape == (vocab,):
        mask = mask.contiguous()
        return rows, tokens, mask, mask.data_ptr(), 0
    raise ValueError(f'mask must have the shape of the logits or of one row, not {tuple(mask.shape)}')


def _forward(logits, tokens, mask, top):
    code = type_of(logits, 'logits')
    if type(top) is not int or not 0 <= top <= MAX_TOP or top > logits.shape[-1]:
        raise ValueError(f'top must be 0 to {MAX_TOP} and at most the number of entries, not {top}')
    rows, tok, mask, mask_ptr, mask_stride = _check(logits, tokens, mask)
    index, (n, vocab) = logits.get_device(), rows.shape
    logp = torch.empty_like(tok, dtype=torch.float32)
    entropy = torch.empty_like(logp)
    stats = logp.new_empty((*logp.shape, 2))
    ids = top_logp = ids_ptr = top_ptr = work = None
    if top:
        ids, top_logp = tok.new_empty((*logp.shape, top)), logp.new_empty((*logp.shape, top))
        ids_ptr, top_ptr = ids.data_ptr(), top_logp.data_ptr()
    L = _lib.load_ops()
    need = L.d1_tokens_work_bytes(n, vocab, top) if vocab > UNSPLIT_VOCAB else 0
    if need:
        work = torch.empty(need, dtype=torch.uint8, device=logits.device)
    call(L.d1_tokens_fwd, index, rows.data_ptr(), code, n, vocab, rows.stride(0), tok.data_ptr(), mask_ptr, mask_stride, top,
         logp.data_ptr(), entropy.data_ptr(), stats.data_ptr(), ids_ptr, top_ptr, work.data_ptr() if need else None, need)
    return TokenLogprobs(logp, entropy, ids, top_logp, stats)


def token_logprobs_bwd(logits, tokens, result, dlogp, dentropy, mask=None):
    """The gradient of the logits (their type, contiguous) from those of logp and entropy (fp32 of
    their shapes; either may be None: zero); `result` is token_logprobs' of the same arguments."""
    code = type_of(logits, 'logits')
    rows, tok, mask, mask_ptr, mask_stride = _check(logits, tokens, mask)
    shape, index, (n, vocab) = tok.shape, logits.get_device(), rows.shape
    stats = like(result.stats, (*shape, 2), index, 'result.stats')
    entropy = like(result.entropy, shape, index, 'result.entropy')
    dlogp = None if dlogp is None else like(dlogp, shape, index, 'dlogp')
    dentropy = None if dentropy is None else like(dentropy, shape, index, 'dentropy')
    dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    call(_lib.load_ops().d1_tokens_bwd, index, rows.data_ptr(), code, n, vocab, rows.stride(0), tok.data_ptr(), mask_ptr,
         mask_stride, stats.data_ptr(), entropy.data_ptr(), None if dlogp is None else dlogp.data_ptr(),
         None if dentropy is None else dentropy.data_ptr(), dlogits.data_ptr())
    return dlogits


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
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, mask, top))
    return _forward(logits, tokens, mask, top)
