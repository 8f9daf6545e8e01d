"""Options that a group of parameters cannot have of its own are refused, wherever they are set."""
import importlib

import pytest
import torch


@pytest.fixture(scope='module')
def A():
    return importlib.import_module('dcss-auto_amd.optim')


def two():
    return [torch.nn.Parameter(torch.ones(3)) for _ in range(2)]


OPTIONS = [dict(betas=(0.5, 0.5)), dict(eps=1e-3), dict(max_grad_norm=1.0), dict(state_bits=8), dict(seed=1), dict(copies={}),
           dict(amsgrad=True), dict(maximize=True)]


@pytest.mark.parametrize('option', OPTIONS, ids=lambda o: next(iter(o)))
def test_options_of_a_group_are_refused(A, option):
    a, b = two()
    with pytest.raises(ValueError, match=next(iter(option))):
        A.AdamW([dict(params=[a]), dict(params=[b], **option)])
    opt = A.AdamW([a])
    with pytest.raises(ValueError, match=next(iter(option))):
        opt.add_param_group(dict(params=[b], **option))
    assert len(opt.param_groups) == 1
    a.grad = torch.ones(3)
    opt.param_groups[0].update(option)
    with pytest.raises(ValueError, match=next(iter(option))):
        opt.step()


def test_options_that_a_group_may_have(A):
    a, b = two()
    opt = A.AdamW([dict(params=[a], lr=0.5, weight_decay=0.25, name='trunk', amsgrad=False), dict(params=[b])], lr=0.125)
    assert [g['lr'] for g in opt.param_groups] == [0.5, 0.125] and opt.param_groups[0]['name'] == 'trunk'


def test_another_optimizers_state_is_refused(A):
    a, _ = two()
    plain = torch.optim.AdamW([a])
    with pytest.raises(ValueError, match='AdamW'):
        A.AdamW([a]).load_state_dict(plain.state_dict())
