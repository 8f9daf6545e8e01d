"""MuonAdamW as a torch optimizer: schedulers, closures, hooks, copies; its groups are those of the two (no GPU needed but for steps)."""
import copy
import importlib
import pickle

import pytest
import torch


@pytest.fixture(scope='module')
def O():
    return importlib.import_module('dcss-auto_amd.optim')


def net(device='cpu'):
    torch.manual_seed(1)
    return torch.nn.ModuleDict(dict(trunk=torch.nn.Linear(7, 9), head=torch.nn.Linear(9, 4))).to(device)


def test_groups(O):
    m = net()
    both = O.MuonAdamW(m.named_parameters(), muon=dict(lr=0.5), adamw=dict(lr=0.25))
    assert isinstance(both, torch.optim.Optimizer)
    assert [g['lr'] for g in both.param_groups] == [0.5, 0.25]
    assert both.param_groups[0] is both.muon.param_groups[0] and both.param_groups[1] is both.adamw.param_groups[0]
    both.param_groups[0]['lr'] = 0.125
    assert both.muon.param_groups[0]['lr'] == 0.125
    both.muon.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2, 2))]))
    assert len(both.param_groups) == 3
    with pytest.raises(ValueError, match='muon'):
        both.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2, 2))]))
    assert len(both.param_groups) == 3


@pytest.mark.parametrize('only', ['trunk', 'head'])
def test_one_part_alone(O, only):
    m = net()
    kept = [(n, p) for n, p in m.named_parameters() if n.startswith(only) and (p.dim() == 2 or only == 'head')]
    both = O.MuonAdamW(kept)
    assert len(both.param_groups) == 1 and (both.muon is None) == (only == 'head') and (both.adamw is None) == (only == 'trunk')
    with pytest.raises(ValueError):
        O.MuonAdamW([])


def test_schedulers(O):
    both = O.MuonAdamW(net().named_parameters(), muon=dict(lr=0.5), adamw=dict(lr=0.25))
    schedule = torch.optim.lr_scheduler.LambdaLR(both, lambda n: 1 / (1 + n))
    assert schedule.get_last_lr() == [0.5, 0.25]
    torch.optim.Optimizer.zero_grad(both)
    both.step()                                    # no gradients: nothing to do
    schedule.step()
    assert [g['lr'] for o in both.both for g in o.param_groups] == [0.25, 0.125]
    schedule.step()
    assert [round(g['lr'], 6) for g in both.muon.param_groups + both.adamw.param_groups] == [0.166667, 0.083333]


def test_hooks_and_copies(O):
    both = O.MuonAdamW(net().named_parameters(), adamw=dict(max_grad_norm=0.5))
    seen = []
    both.register_step_pre_hook(lambda *a: seen.append('before'))
    both.register_step_post_hook(lambda *a: seen.append('after'))
    both.step()
    assert seen == ['before', 'after']
    for twin in (copy.deepcopy(both), pickle.loads(pickle.dumps(O.MuonAdamW(net().named_parameters(), adamw=dict(max_grad_norm=0.5))))):
        assert twin.adamw.max_grad_norm == 0.5 and twin.muon.settings == both.muon.settings and twin.both == [twin.muon, twin.adamw]
        assert twin.param_groups[0] is twin.muon.param_groups[0] and twin.param_groups[0]['params'][0] is not both.param_groups[0]['params'][0]
        twin.step()


@pytest.mark.gpu
def test_closure_and_state(O):
    m = net('cuda')
    both = O.MuonAdamW(m.named_parameters(), adamw=dict(max_grad_norm=0.5))
    x = torch.randn(5, 7, device='cuda')

    def closure():
        both.zero_grad()
        loss = m['head'](m['trunk'](x)).square().mean()
        loss.backward()
        return loss
    first = both.step(closure)
    assert float(first) > 0 and float(both.step(closure)) != float(first)
    assert 'momentum' in both.state[m['trunk'].weight] and 'exp_avg' in both.state[m['head'].weight]
    twin = copy.deepcopy(both)
    assert torch.equal(twin.muon.ctl, both.muon.ctl) and twin.muon.ctl is not both.muon.ctl
    # a schedule over loaded groups: those of the load, not of before it
    both.load_state_dict(copy.deepcopy(both.state_dict()))
    schedule = torch.optim.lr_scheduler.LambdaLR(both, lambda n: 0.5 ** n)
    closure()
    both.step()
    schedule.step()
    assert both.muon.param_groups[0]['lr'] == 0.01 and both.adamw.param_groups[0]['lr'] == 0.0005
