"""adamw_step tells torch what it wrote: version counters of every tensor that it changes, and of nothing
else, so that packed weights are made anew and autograd finds a saved tensor that was changed."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def mods(pkg):
    return tuple(importlib.import_module('dcss-auto_amd.' + n) for n in ('policy', 'optim'))


def observations(n, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return torch.randint(0, 4, (n, 1800), generator=g, device='cuda', dtype=torch.uint8)


def set_grads(model, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    for p in model.parameters():
        p.grad = torch.randn(p.shape, generator=g, device='cuda').to(p.dtype)


def fresh(cls, model):
    twin = cls().cuda().to(next(model.parameters()).dtype)
    twin.load_state_dict(model.state_dict())
    return twin


@pytest.mark.parametrize('bits', [32, 8])
def test_policy_forward_after_steps(mods, bits):
    """The fused forward of an fp32 Policy under autocast, before and after steps."""
    P, A = mods
    print(f'[versions] policy {bits}', flush=True)
    model, obs = P.Policy(seed=1).cuda(), observations(300, 2)
    opt = A.AdamW(model.parameters(), lr=3e-3, state_bits=bits, max_grad_norm=1.0)
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        outs = [model(obs)]
        for t in range(3):
            set_grads(model, t)
            opt.step()
            outs.append(model(obs))
            want = fresh(P.Policy, model)(obs)
            assert all(torch.equal(a, b) for a, b in zip(outs[-1], want))
            assert not torch.equal(outs[-1][0], outs[-2][0])


def test_policy_fed_by_copies(mods):
    """A bf16 Policy that serves while an fp32 one trains: its parameters are the step's copies."""
    P, A = mods
    print('[versions] copies', flush=True)
    model, obs = P.Policy(seed=3).cuda(), observations(300, 4)
    served = P.Policy(seed=3).cuda().to(torch.bfloat16)
    opt = A.AdamW(model.parameters(), lr=3e-3, copies=dict(zip(model.parameters(), served.parameters())))
    with torch.no_grad():
        before = served(obs)
        for t in range(2):
            set_grads(model, t)
            opt.step()
            got, want = served(obs), fresh(P.Policy, served)(obs)
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and not torch.equal(got[0], before[0])
            before = got


def test_ar_policy_after_steps(mods):
    P, A = mods
    print('[versions] ar policy', flush=True)
    model, obs = P.ARPolicy(seed=5).cuda().to(torch.bfloat16), observations(200, 6)

    def served(m):
        out = dict(action=torch.empty(200, dtype=torch.int64, device='cuda'), logp=torch.empty(200, device='cuda'),
                   value=torch.empty(200, device='cuda'), verb_logits=torch.empty(200, 8, device='cuda'))
        P.policy_fwd_sample_ar(obs, m.packed(), 11, 3, out['action'], out['logp'], out['value'], verb_logits=out['verb_logits'])
        return out

    opt = A.AdamW(model.parameters(), lr=1e-2)
    before = served(model)
    for t in range(2):
        set_grads(model, t)
        opt.step()
        got, want = served(model), served(fresh(P.ARPolicy, model))
        assert all(torch.equal(got[k], want[k]) for k in got) and not torch.equal(got['verb_logits'], before['verb_logits'])
        before = got


def test_backward_after_a_step_raises(mods):
    """A parameter that the graph has saved, changed by a step before the backward pass."""
    P, A = mods
    print('[versions] saved tensors', flush=True)
    w = torch.nn.Parameter(torch.randn(20, 30, device='cuda'))
    x = torch.randn(5, 30, device='cuda', requires_grad=True)
    opt = A.AdamW([w], lr=1e-2)
    loss = (x @ w.t()).square().sum()
    w.grad = torch.ones_like(w)
    opt.step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


@pytest.mark.parametrize('bits', [32, 8])
def test_what_a_step_writes(mods, bits):
    """Versions rise for what the step writes, once at least, and stay for the gradients; a refused call
    raises none; tensors made under inference mode, which have no version, are taken too."""
    P, A = mods
    print(f'[versions] written {bits}', flush=True)

    def make():
        zeros = lambda n, dtype=torch.float32: torch.zeros(n, dtype=dtype, device='cuda')  # noqa: E731
        p, g = [zeros(700), zeros(5)], [torch.ones(700, device='cuda'), torch.ones(5, device='cuda')]
        dtype = torch.uint8 if bits == 8 else torch.float32
        m, v = ([zeros(x.numel(), dtype) for x in p] for _ in range(2))
        copies = [zeros(700, torch.bfloat16), None]
        exps = tuple([zeros(A.moment_blocks(x.numel()), torch.uint8) for x in p] for _ in range(2)) if bits == 8 else None
        return p, g, m, v, copies, exps, zeros(8, torch.int32)

    p, g, m, v, copies, exps, step = make()
    written = [*p, *m, *v, copies[0], step] + ([*exps[0], *exps[1]] if exps else [])
    was, gwas = [x._version for x in written], [x._version for x in g]
    A.adamw_step(p, g, m, v, step, copies=copies, exps=exps)
    assert all(x._version > k for x, k in zip(written, was)) and [x._version for x in g] == gwas
    was = [x._version for x in written]
    with pytest.raises(ValueError):
        A.adamw_step(p, g, m, v, step, lr=-1.0, copies=copies, exps=exps)
    assert [x._version for x in written] == was
    if bits == 8:
        out = torch.empty(700, device='cuda')
        k = out._version
        A.read_moment(m[0], exps[0][0], signed=True, out=out)
        assert out._version > k
    with torch.inference_mode():
        q, h, a, b, c, e, s = make()
    A.adamw_step(q, h, a, b, s, copies=c, exps=e)
    assert torch.equal(q[0], p[0]) and int(s[0]) == 1
