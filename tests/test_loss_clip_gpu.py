"""Every form of a clip that unpacks, or is one number, is the same clip to policy_loss and to ModulePPO."""
import importlib

import numpy as np
import pytest
import torch

import test_losses_gpu as base

pytestmark = pytest.mark.gpu

PAIRS = [(0.25, 0.5), [0.25, 0.5], np.array([0.25, 0.5]), np.array([0.25, 0.5], np.float32), torch.tensor([0.25, 0.5])]
NUMBERS = [0.25, np.float32(0.25), np.float64(0.25), np.array(0.25), torch.tensor(0.25)]


@pytest.mark.parametrize('forms', [PAIRS, NUMBERS], ids=['pair', 'number'])
def test_forms(forms):
    L = importlib.import_module('dcss-auto_amd.losses')
    ppo = importlib.import_module('dcss-auto_amd.ppo')
    k = base.data((500,), seed=3, ref=False, value=True)
    z = torch.zeros(500, device=base.DEV)

    class Fixed(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.scale = torch.nn.Parameter(torch.ones((), device=base.DEV))

        def evaluate(self, obs, actions):
            return k['logp'] * self.scale, k['entropy'], k['values']
    seen = []
    for clip in forms:
        r, dlogp, _, _ = L.policy_loss_grads(k['logp'], k['old_logp'], k['advantages'], clip=clip)
        mine = ppo.ModulePPO(Fixed(), autocast=False, clip=clip, lr=0.0)
        loss = mine.minibatch_step(z, z, k['old_logp'], k['advantages'], k['returns'])
        seen.append((r.terms, dlogp, loss))
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(other, seen[0]))
    assert float(seen[0][0][5]) > 0                  # some are clipped
