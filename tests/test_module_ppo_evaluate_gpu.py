"""ModulePPO with policies whose evaluate gives other shapes and types than its log probabilities': what broadcasts, a number for the
entropy, 64 bits; the loss and its gradients are the elementary formula's."""
import importlib

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

DEV = 'cuda'


class Linear(nn.Module):
    """Gaussian log probabilities of a linear map, shaped and typed by `form`."""

    def __init__(self, form):
        super().__init__()
        self.form, self.w = form, nn.Parameter(torch.linspace(-0.02, 0.02, 3 * 8).view(8, 3))

    def evaluate(self, obs, actions):
        out = obs.float() @ self.w.float()
        logp, entropy, value = -0.5 * (out[:, 0] - actions.float()) ** 2, out[:, 1], out[:, 2]
        return self.form(logp, entropy, value)


FORMS = {
    'plain': lambda lp, e, v: (lp, e, v),
    'entropy is a number': lambda lp, e, v: (lp, e.mean(), v),
    'entropy of a batch of one': lambda lp, e, v: (lp, e.mean()[None], v),
    'value in a column': lambda lp, e, v: (lp, e, v[:, None]),
    'one value': lambda lp, e, v: (lp, e, v.mean()),
    'log probability in a row': lambda lp, e, v: (lp[None], e, v),
    '64 bits': lambda lp, e, v: (lp.double(), e.double(), v.double()),
    'entropy in 64 bits': lambda lp, e, v: (lp, e.double(), v),
}


def formula(evaluated, old_logp, adv, ret, clip, vcoef, ecoef):
    logp, entropy, value = evaluated
    ratio = torch.exp(logp - old_logp)
    pg = -torch.minimum(ratio * adv, ratio.clamp(1 - clip, 1 + clip) * adv).mean()
    return pg + vcoef * 0.5 * (value.float() - ret).square().mean() - ecoef * entropy.mean()


@pytest.mark.parametrize('name', list(FORMS))
@pytest.mark.parametrize('clip', [0.2, 1.0, 1.5])
def test_forms(pkg, name, clip):
    ppo = importlib.import_module('dcss-auto_amd.ppo')
    g = torch.Generator(DEV).manual_seed(1)
    model, twin = Linear(FORMS[name]).cuda(), Linear(FORMS[name]).cuda()
    n = 300
    obs = torch.randint(0, 4, (n, 8), generator=g, device=DEV, dtype=torch.uint8)
    actions = torch.randint(0, 2, (n,), generator=g, device=DEV)
    old, adv, ret = (torch.randn(n, generator=g, device=DEV) * s for s in (0.3, 1.0, 1.0))
    mine = ppo.ModulePPO(model, autocast=False, clip=clip, max_grad_norm=1e9, lr=0.0)
    loss = mine.minibatch_step(obs, actions, old, adv, ret)
    want = formula(twin.evaluate(obs, actions), old, adv, ret, clip, 0.5, 0.01)
    want.backward()
    torch.testing.assert_close(loss.double(), want.detach().double(), rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(model.w.grad, twin.w.grad, rtol=1e-4, atol=1e-5 * float(twin.w.grad.abs().max()))
    assert mine.terms.loss.requires_grad is False and bool(torch.isfinite(mine.terms.terms).all())
    assert torch.equal(mine.terms.terms[0], mine.terms.loss.float())


@pytest.mark.parametrize('name', ['64 bits', 'entropy is a number', 'log probability in a row', 'value in a column'])
def test_further_terms(pkg, name):
    """A pair of clips, a clipped value and a reference beside such forms."""
    ppo = importlib.import_module('dcss-auto_amd.ppo')
    g = torch.Generator(DEV).manual_seed(2)
    model, twin, ref = Linear(FORMS[name]).cuda(), Linear(FORMS[name]).cuda(), Linear(FORMS[name]).cuda()
    with torch.no_grad():
        ref.w.mul_(-0.5)
    n = 257
    obs = torch.randint(0, 4, (n, 8), generator=g, device=DEV, dtype=torch.uint8)
    actions = torch.randint(0, 2, (n,), generator=g, device=DEV)
    old, adv, ret, old_v = (torch.randn(n, generator=g, device=DEV) * s for s in (0.3, 1.0, 1.0, 0.3))
    mine = ppo.ModulePPO(model, autocast=False, clip=(0.1, 0.4), value_clip=0.2, kl_coef=0.3, reference=ref, max_grad_norm=1e9, lr=0.0)
    loss = mine.minibatch_step(obs, actions, old, adv, ret, old_v)
    logp, entropy, value = twin.evaluate(obs, actions)
    r = torch.exp(logp - old)
    x = ref.evaluate(obs, actions)[0].detach() - logp
    near = old_v + (value - old_v).clamp(-0.2, 0.2)
    terms = dict(policy=-torch.minimum(r * adv, r.clamp(0.9, 1.4) * adv).mean(), kl=(x.exp() - 1 - x).mean(), entropy=entropy.mean(),
                 value=0.5 * torch.maximum((value - ret) ** 2, (near - ret) ** 2).mean())
    want = terms['policy'] + 0.5 * terms['value'] - 0.01 * terms['entropy'] + 0.3 * terms['kl']
    want.backward()
    torch.testing.assert_close(loss.double(), want.detach().double(), rtol=1e-5, atol=1e-6)
    for k, t in terms.items():
        torch.testing.assert_close(getattr(mine.terms, k).double(), t.detach().double(), rtol=1e-4, atol=1e-6)
    torch.testing.assert_close(model.w.grad, twin.w.grad, rtol=1e-4, atol=1e-5 * float(twin.w.grad.abs().max()))


def test_what_does_not_broadcast_is_refused(pkg):
    ppo = importlib.import_module('dcss-auto_amd.ppo')
    model = Linear(lambda lp, e, v: (lp[:7], e, v)).cuda()
    mine = ppo.ModulePPO(model, autocast=False)
    z = torch.zeros(20, device=DEV)
    with pytest.raises((ValueError, RuntimeError)):
        mine.minibatch_step(torch.zeros(20, 8, device=DEV, dtype=torch.uint8), z.long(), z, z, z)
