"""policy_loss with finite log probabilities far apart, down to the lowest value of their type: e^d is 0 there and every
term and gradient finite, as its definition in 64 bits has it."""
import importlib
import math

import pytest
import torch

import test_losses_gpu as base

pytestmark = pytest.mark.gpu

DEV, U = base.DEV, base.U
LOWEST = torch.finfo(torch.float32).min


@pytest.mark.parametrize('far', [-200.0, -1e4, -2.3e38, -2.5e38, LOWEST])
@pytest.mark.parametrize('tokens', [1, 7, 5000])
def test_a_token_that_the_policy_gives_up(far, tokens):
    """logp far below the old one: the ratio is 0, its drift -d - 1."""
    print(f'[loss] logp {far} {tokens}', flush=True)
    L = importlib.import_module('dcss-auto_amd.losses')
    k = base.data((tokens,), seed=3, ref=False)
    k['logp'][tokens // 2] = far
    k['old_logp'][tokens // 2] = 0.0
    for sign in (1.0, -1.0):
        k['advantages'][tokens // 2] = sign
        r = base.compare(L, k, 'token')
        assert bool(torch.isfinite(r.terms).all())
        assert math.isclose(float(r.drift), -far / tokens, rel_tol=1e-3) or far > -1e5


@pytest.mark.parametrize('far', [-200.0, -1e4, -2.5e38, LOWEST])
def test_a_token_that_the_reference_gives_up(far):
    """ref_logp far below: e^x is 0, its KL -x - 1 and the gradient kl_coef."""
    L = importlib.import_module('dcss-auto_amd.losses')
    for tokens in (1, 5000):
        k = base.data((tokens,), seed=4)
        k['ref_logp'][0] = far
        k['logp'][0] = k['old_logp'][0] = 0.0
        r = base.compare(L, k, 'token')
        assert bool(torch.isfinite(r.terms).all())


def test_bf16():
    """The lowest bf16 value, in a sequence whose other tokens are ordinary."""
    L = importlib.import_module('dcss-auto_amd.losses')
    k = base.data((6, 50), torch.bfloat16, seed=5)
    k['logp'][2, 3] = torch.finfo(torch.bfloat16).min
    k['old_logp'][2, 3] = 0.0
    k['ref_logp'][2, 3] = k['logp'][2, 3]
    base.compare(L, k, 'sequence')


def test_not_finite_stays_not_finite():
    L = importlib.import_module('dcss-auto_amd.losses')
    for value, drift in ((math.nan, math.isnan), (-math.inf, lambda x: x == math.inf), (math.inf, lambda x: x == math.inf or math.isnan(x))):
        logp = torch.zeros(9, device=DEV)
        logp[4] = value
        r, dlogp, _, _ = L.policy_loss_grads(logp, torch.zeros(9, device=DEV), torch.ones(9, device=DEV))
        assert drift(float(r.drift))
        assert not math.isnan(value) or bool(dlogp[4].isnan())
        assert bool(torch.isfinite(dlogp[[0, 1, 2, 3, 5, 6, 7, 8]]).all())
