"""torch.jit.trace of the operators: a traced call computes its outputs from new inputs, and what a trace
cannot hold is refused, where it would record outputs that nothing fills."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def mods(pkg):
    return tuple(importlib.import_module('dcss-auto_amd.' + n) for n in ('tokens', 'norm'))


@pytest.mark.filterwarnings('ignore')
@pytest.mark.parametrize('grad', [False, True])
def test_trace(mods, grad):
    T, N = mods
    print(f'[trace] {grad}', flush=True)
    g = torch.Generator(device='cuda').manual_seed(1)
    x, t, w, b = (torch.randn(*s, generator=g, device='cuda') for s in ((6, 40), (6, 40), (40,), (40,)))
    tokens = torch.arange(6, device='cuda')
    r = T.token_logprobs(x, tokens)
    layer = N.LayerNorm(40).cuda()                 # with grad, parameters that want one
    with torch.set_grad_enabled(grad):
        for call in (layer, lambda z: N.layer_norm(z, w, b), lambda z: T.token_logprobs(z, tokens, top=3).top_logp,
                     lambda z: T.token_logprobs(z, tokens).logp):
            traced = torch.jit.trace(call, (x,), check_trace=False)
            for z in (x, t, 3 * x):
                assert torch.equal(traced(z), call(z))
        for call in (lambda z: N.layer_norm_fwd(z, w, b)[0],
                     lambda z: N.layer_norm_bwd(t, z, w, b, torch.zeros(6, device='cuda'), torch.ones(6, device='cuda'))[0],
                     lambda z: T.token_logprobs_bwd(z, tokens, r, torch.ones(6, device='cuda'), None)):
            with pytest.raises(RuntimeError, match='trace'):
                torch.jit.trace(call, (x,), check_trace=False)
    y = N.layer_norm(x, w, b)                      # afterwards all is as before
    assert torch.equal(N.layer_norm_fwd(x, w, b)[0], y)
