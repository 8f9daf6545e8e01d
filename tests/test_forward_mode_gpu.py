"""What has no formula for it is refused and not left out: forward-mode tangents through the token, norm,
gradient and optimizer calls, and transforms over them."""
import importlib

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def mods(pkg):
    return tuple(importlib.import_module('dcss-auto_amd.' + n) for n in ('tokens', 'norm'))


def data():
    g = torch.Generator(device='cuda').manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731
    return rand(6, 40), torch.arange(6, device='cuda'), rand(40), rand(40), rand(6, 40)


@pytest.mark.parametrize('grad', [False, True])
def test_tangents_are_refused(mods, grad):
    T, N = mods
    print(f'[forward mode] tangents {grad}', flush=True)
    x, tokens, w, b, t = data()
    r = T.token_logprobs(x, tokens)
    y, mean, rstd = N.layer_norm_fwd(x, w, b)
    one = torch.ones(6, device='cuda')
    with forward_ad.dual_level():
        dual = lambda a: forward_ad.make_dual(a.clone().requires_grad_(grad), torch.ones_like(a))  # noqa: E731
        with torch.set_grad_enabled(grad):
            for call in (lambda: T.token_logprobs(dual(x), tokens), lambda: N.layer_norm(dual(x), w, b),
                         lambda: N.layer_norm(x, dual(w), b), lambda: N.layer_norm(x, w, dual(b)),
                         lambda: N.LayerNorm(40).cuda()(dual(x)), lambda: N.layer_norm_fwd(dual(x), w, b),
                         lambda: N.layer_norm_bwd(dual(t), x, w, b, mean, rstd),
                         lambda: N.layer_norm_bwd(t, dual(x), w, b, mean, rstd),
                         lambda: T.token_logprobs_bwd(x, tokens, r, dual(one), None),
                         lambda: T.token_logprobs_bwd(x, tokens, r, None, dual(one)),
                         lambda: T.token_logprobs_bwd(dual(x), tokens, r, one, None)):
                with pytest.raises(NotImplementedError):
                    call()
        A = importlib.import_module('dcss-auto_amd.optim')
        step, z = torch.zeros(8, dtype=torch.int32, device='cuda'), lambda: torch.zeros(40, device='cuda')
        tangent = forward_ad.make_dual(w.clone(), torch.ones_like(w))
        for p, g in ((tangent, z()), (z(), tangent)):
            with pytest.raises(NotImplementedError):
                A.adamw_step([p], [g], [z()], [z()], step)
        # no tangent, no refusal
        assert torch.equal(N.layer_norm(x, w, b), y) and torch.equal(T.token_logprobs(x, tokens).logp, r.logp)


def test_transforms_are_refused(mods):
    T, N = mods
    print('[forward mode] transforms', flush=True)
    x, tokens, w, b, t = data()
    for call in (lambda z: T.token_logprobs(z, tokens).logp, lambda z: N.layer_norm(z, w, b)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(call, (x,), (t,))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.vmap(lambda z: N.layer_norm(z, w, b))(x)
