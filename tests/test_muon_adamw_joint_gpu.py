"""MuonAdamW: a gradient that is not finite anywhere leaves all as it was, eagerly, captured and from ModulePPO and SequencePPO."""
import copy
import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'


@pytest.fixture(scope='module')
def mods(pkg):
    return pkg, *(importlib.import_module('dcss-auto_amd.' + n) for n in ('optim', 'policy', 'ppo', 'train'))


def model(P, seed=1):
    return P.MemoryPolicy(width=32, obs=50, seed=seed).cuda()


def grads(ps, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    for p in ps:
        new = torch.randn(p.shape, generator=g, device=DEV)
        if p.grad is None:
            p.grad = new
        else:
            p.grad.copy_(new)


def everything(net, both):
    return [t.clone() for t in (*net.parameters(), *(v for o in both.both for s in o.state.values() for v in s.values() if torch.is_tensor(v)))]


@pytest.mark.parametrize('clip', [0.0, 0.5])
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('where', ['l1.weight', 'cell.weight', 'head.weight', 'n1.bias'])
def test_a_bad_gradient_in_either_part(mods, where, bits, clip):
    """Without a clip AdamW looks at no norm: then a bad gradient of its own is its elements' alone, as it always was."""
    _, O, P, _, _ = mods
    nets = [model(P) for _ in range(2)]
    both, clean = (O.MuonAdamW(n.named_parameters(), adamw=dict(max_grad_norm=clip, state_bits=bits)) for n in nets)
    if clip == 0.0 and where in ('head.weight', 'n1.bias'):
        pytest.skip('no norm is looked at')
    skipped = 0
    for n, value in enumerate((0.0, math.nan, 0.0, math.inf, -math.inf, 0.0)):
        for net in nets:
            grads(list(net.parameters()), n)
        if value:
            dict(nets[0].named_parameters())[where].grad.view(-1)[7] = value
            before = everything(nets[0], both)
            both.step()
            skipped += 1
            assert all(torch.equal(a, b) for a, b in zip(before, everything(nets[0], both))), value
        else:
            both.step()
            clean.step()
            assert all(torch.equal(a, b) for a, b in zip(everything(nets[0], both), everything(nets[1], clean))), n
        assert both.skipped_steps() == skipped
        assert [int(o.ctl[0]) for o in both.both] == [n + 1 - skipped] * 2 and [int(o.ctl[1]) for o in both.both] == [skipped] * 2
    assert clean.skipped_steps() == 0


def test_captured(mods):
    _, O, P, _, _ = mods
    nets = [model(P) for _ in range(2)]
    both, plain = (O.MuonAdamW(n.named_parameters(), adamw=dict(max_grad_norm=0.5)) for n in nets)
    for net, o in zip(nets, (both, plain)):
        grads(list(net.parameters()), 0)
        o.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both.step()
    names = [None, 'l1.weight', None, 'head.bias', 'cell.weight', None]
    for n, bad in enumerate(names):
        for net in nets:
            grads(list(net.parameters()), 10 + n)
            if bad:
                dict(net.named_parameters())[bad].grad.view(-1)[3] = math.nan
        before = everything(nets[0], both)
        graph.replay()
        plain.step()
        torch.cuda.synchronize()
        now = everything(nets[0], both)
        assert all(torch.equal(a, b) for a, b in zip(now, everything(nets[1], plain))), n
        assert all(torch.equal(a, b) for a, b in zip(now, before)) == bool(bad), n
    assert both.skipped_steps() == plain.skipped_steps() == 3


def test_one_part_without_gradients(mods):
    """Either side alone still steps, and still skips."""
    _, O, P, _, _ = mods
    for trunk in (True, False):
        net = model(P)
        both = O.MuonAdamW(net.named_parameters(), adamw=dict(max_grad_norm=0.5))
        mine = [p for g in (both.muon if trunk else both.adamw).param_groups for p in g['params']]
        grads(mine, 1)
        before = [p.detach().clone() for p in net.parameters()]
        both.step()
        assert sum(not torch.equal(a, b) for a, b in zip(before, net.parameters())) == len(mine) and both.skipped_steps() == 0
        grads(mine, 2)
        mine[0].grad.view(-1)[0] = math.nan
        before = [p.detach().clone() for p in net.parameters()]
        both.step()
        assert all(torch.equal(a, b) for a, b in zip(before, net.parameters())) and both.skipped_steps() == 1


@pytest.mark.parametrize('where', ['l1.weight', 'cell.weight', 'head.weight', 'n2.weight'])
@pytest.mark.parametrize('optimizer', ['adamw', 'muon'])
def test_update_raises_on_a_whole_model(mods, where, optimizer):
    """ModulePPO's promise: a minibatch whose gradient is not finite changes nothing, wherever in the model it is."""
    pkg, _, P, ppo, train = mods
    for kind in (P.MemoryPolicy, P.NormPolicy):
        name = {'cell.weight': 'l2.weight'}.get(where, where) if kind is P.NormPolicy else where
        env = pkg.Env(64, pkg.baseline_config(), seed=8, hash=False)
        net = kind(width=32, seed=9).cuda()
        tr = train.ModuleTrainer(env, net, horizon=8, minibatch=512, epochs=1, optimizer=optimizer)
        tr.train(1)
        tr.rollout()
        before = [p.detach().clone() for p in net.parameters()]
        hook = dict(net.named_parameters())[name].register_hook(lambda g: torch.full_like(g, math.inf))
        with pytest.raises(RuntimeError, match='Non-finite'):
            tr.update()
        assert all(torch.equal(p, q) for p, q in zip(net.parameters(), before)), (kind, where)
        hook.remove()
        assert bool(torch.isfinite(tr.train(1)))
        assert not all(torch.equal(p, q) for p, q in zip(net.parameters(), before))


def test_with_states_loaded(mods):
    """Counts and moments of both go on from a saved state, with skips in either part."""
    _, O, P, _, _ = mods
    nets = [model(P) for _ in range(2)]
    a = O.MuonAdamW(nets[0].named_parameters(), adamw=dict(max_grad_norm=0.5))
    grads(list(nets[0].parameters()), 1)
    a.step()
    nets[0].head.weight.grad[0, 0] = math.nan
    a.step()
    nets[1].load_state_dict(nets[0].state_dict())
    b = O.MuonAdamW(nets[1].named_parameters(), adamw=dict(max_grad_norm=0.5))
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    assert b.skipped_steps() == a.skipped_steps() == 1
    for n in range(2, 5):
        for net, o in zip(nets, (a, b)):
            grads(list(net.parameters()), n)
            if n == 3:
                net.l1.weight.grad[0, 0] = math.nan
            o.step()
    assert all(torch.equal(x, y) for x, y in zip(nets[0].parameters(), nets[1].parameters())) and a.skipped_steps() == b.skipped_steps() == 2
