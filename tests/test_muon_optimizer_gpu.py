"""Muon and MuonAdamW as torch optimizers: groups, parameters without gradients, states saved and loaded, captured steps,
refusals."""
import copy
import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'


@pytest.fixture(scope='module')
def O():
    return importlib.import_module('dcss-auto_amd.optim')


def params(seed=0, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g, device=DEV).to(dtype)) for s in ((40, 60), (70, 20), (8, 3, 5))]


def grads(ps, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g, device=DEV).to(p.dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rms', [False, True])
def test_steps(O, dtype, rms):
    """The class makes muon_step's steps: lr and decay by group, scales by shape, a parameter without a gradient left alone."""
    a, b = params(1, dtype), params(1, dtype)
    opt = O.Muon([dict(params=a[:1], lr=0.1, weight_decay=0.2), dict(params=a[1:])], lr=0.02, momentum=0.8, rms=rms)
    m, ctl = [torch.zeros(p.shape, device=DEV) for p in b], torch.zeros(8, dtype=torch.int32, device=DEV)
    scale = [0.2 * math.sqrt(max(p.shape[0], p[0].numel())) if rms else math.sqrt(max(1, p.shape[0] / p[0].numel())) for p in b]
    for n in range(3):
        grads(a, n)
        use = [0, 1, 2]
        if n == 1:
            a[1].grad = None
            use = [0, 2]
        opt.step()
        pick = lambda x: [x[i] for i in use]  # noqa: E731
        O.muon_step([b[i].data for i in use], [a[i].grad for i in use], pick(m), ctl, lr=pick([0.1, 0.02, 0.02]), momentum=0.8,
                    weight_decay=pick([0.2, 0.0, 0.0]), scales=pick(scale))
        for p, q in zip(a, b):
            assert torch.equal(p, q)
    assert opt.skipped_steps() == 0 and int(opt.ctl[0]) == 3


def test_saved_and_copied(O):
    a = params(2, torch.bfloat16)
    opt = O.Muon(a)
    for n in range(2):
        grads(a, n)
        opt.step()
    saved = opt.state_dict()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    other = O.Muon(b)
    other.load_state_dict(copy.deepcopy(saved))
    assert other.state[b[0]]['momentum'].dtype == torch.float32
    third = copy.deepcopy(opt)
    for n in range(2, 4):
        for ps, o in ((a, opt), (b, other), (third.param_groups[0]['params'], third)):
            grads(ps, n)
            o.step()
    for p, q, r in zip(a, b, third.param_groups[0]['params']):
        assert torch.equal(p, q) and torch.equal(p, r)
    with pytest.raises(ValueError):
        other.load_state_dict(torch.optim.SGD(b, lr=0.1).state_dict())


def test_skipped(O):
    a = params(3)
    opt = O.Muon(a)
    grads(a, 0)
    opt.step()
    before = [p.detach().clone() for p in a]
    a[2].grad[0, 0, 0] = math.nan
    opt.step()
    assert opt.skipped_steps() == 1 and all(torch.equal(p, q) for p, q in zip(a, before))


def test_captured(O):
    a, b = params(4), params(4)
    opt, plain = O.Muon(a), O.Muon(b)
    grads(a, 0)
    grads(b, 0)
    fresh = O.Muon(params(5))
    for o in (opt, plain):
        o.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
        p = fresh.param_groups[0]['params'][0]
        p.grad = a[0].grad
        with pytest.raises(RuntimeError):          # its state would be made anew by each replay
            fresh.step()
    for n in range(1, 5):
        g = torch.Generator(device=DEV).manual_seed(n)
        for p, q in zip(a, b):
            q.grad = torch.randn(p.shape, generator=g, device=DEV)
            p.grad.copy_(q.grad)
        graph.replay()
        plain.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), n


def test_beside_adamw(O):
    """The trunk's matrices are Muon's, the rest AdamW's; together they are the two alone."""
    model = importlib.import_module('dcss-auto_amd.policy').MemoryPolicy(width=32, obs=50).cuda()
    both = O.MuonAdamW(model.named_parameters(), muon=dict(lr=0.05), adamw=dict(lr=0.01))
    names = {id(p): n for n, p in model.named_parameters()}
    assert {names[id(p)] for g in both.muon.param_groups for p in g['params']} == {'l1.weight', 'cell.weight'}
    twin = copy.deepcopy(model)
    one = O.Muon([twin.l1.weight, twin.cell.weight], lr=0.05)
    two = O.AdamW([p for n, p in twin.named_parameters() if n not in ('l1.weight', 'cell.weight')], lr=0.01)
    for n in range(3):
        grads(list(model.parameters()), n)
        for p, q in zip(model.parameters(), twin.parameters()):
            q.grad = p.grad.clone()
        both.step()
        one.step()
        two.step()
    assert all(torch.equal(p, q) for p, q in zip(model.parameters(), twin.parameters()))
    again = O.MuonAdamW(model.named_parameters())
    again.load_state_dict(both.state_dict())
    assert torch.equal(again.muon.ctl, both.muon.ctl) and both.skipped_steps() == 0
    both.zero_grad()
    assert all(p.grad is None for p in model.parameters())


def test_refusals(O):
    a = params(6)
    for k in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(product_bits=8)):
        with pytest.raises(ValueError):
            O.Muon(a, **k)
    with pytest.raises(ValueError):
        O.Muon([torch.nn.Parameter(torch.zeros(5, device=DEV))])
    with pytest.raises(ValueError):
        O.Muon([dict(params=a, momentum=0.5)])
