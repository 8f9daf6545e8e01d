"""ModulePPO's construction (no GPU needed)."""
import importlib

import torch


def test_one_optimizer(monkeypatch):
    """Its own AdamW with the settings given, and no other optimizer beside it."""
    P, ppo, A = (importlib.import_module('dcss-auto_amd.' + n) for n in ('policy', 'ppo', 'optim'))
    model = P.NormPolicy(width=8)
    made = []
    real = torch.optim.Optimizer.__init__
    monkeypatch.setattr(torch.optim.Optimizer, '__init__', lambda self, *a, **k: (made.append(type(self)), real(self, *a, **k))[1])
    mine = ppo.ModulePPO(model, lr=0.25, eps=0.5, weight_decay=0.125, state_bits=8, max_grad_norm=2.0, seed=7)
    assert made == [A.AdamW] and type(mine.opt) is A.AdamW
    group, = mine.opt.param_groups
    assert (group['lr'], group['weight_decay'], mine.opt.eps, mine.opt.state_bits, mine.opt.max_grad_norm, mine.opt.seed) == \
        (0.25, 0.125, 0.5, 8, 2.0, 7)
    assert [id(p) for p in group['params']] == [id(p) for p in model.parameters()]
