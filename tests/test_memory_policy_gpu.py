"""MemoryPolicy, SequencePPO and the update's further terms: sequences against elementary operations, acting step by step
against the whole, one minibatch's loss and gradients, and whole runs with Muon, a reference and value clipping together."""
import copy
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'


@pytest.fixture(scope='module')
def mods(pkg):
    return pkg, *(importlib.import_module('dcss-auto_amd.' + n) for n in ('policy', 'ppo', 'train'))


def torch_norm(x, layer):
    d = x - x.mean(-1, keepdim=True)
    return d / torch.sqrt((d * d).mean(-1, keepdim=True) + layer.eps) * layer.weight + layer.bias


def plain(model, obs, state, reset):
    """The policy in elementary operations, step by step."""
    h = torch.relu(torch_norm(model.l1(obs.float()), model.n1))
    x, gate = model.cell(h).chunk(2, -1)
    z, m, out = torch.sigmoid(gate), state, []
    for t in range(obs.shape[0]):
        m = torch.where(reset[t][:, None].bool(), 0.0, m)
        m = (1 - z[t]) * m + z[t] * x[t]
        out.append(m)
    y = model.head(torch_norm(torch.stack(out) + h, model.n2))
    return y[..., :model.n_actions], y[..., model.n_actions], m


def sequence(pkg, P, steps=20, n=12, seed=3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    env = pkg.Env(n, pkg.baseline_config(), seed=seed, hash=False)
    obs = []
    for _ in range(steps):
        env.step(torch.randint(0, 16, (n,), device=DEV, generator=g))
        obs.append(env.obs.view(n, -1).clone())
    reset = (torch.rand(steps, n, device=DEV, generator=g) < 0.1).to(torch.uint8)
    return torch.stack(obs), torch.randint(0, 16, (steps, n), device=DEV, generator=g), reset, g


def test_evaluate_and_act(mods):
    pkg, P, ppo, _ = mods
    print('[memory] evaluate', flush=True)
    obs, actions, reset, g = sequence(pkg, P)
    model = P.MemoryPolicy(width=96, seed=1).cuda()
    state = torch.randn(12, 96, device=DEV, generator=g)
    logp, entropy, value = model.evaluate_sequence(obs, actions, state, reset)
    c = torch.randn(20, 12, device=DEV, generator=g)
    (c * logp + 0.3 * entropy + c * value).sum().backward()
    got = [p.grad.clone() for p in model.parameters()]
    model.zero_grad()
    logits, v, last = plain(model, obs, state, reset)
    lp = torch.log_softmax(logits, -1)
    want_logp, want_entropy = lp.gather(-1, actions[..., None])[..., 0], -(lp.exp() * lp).sum(-1)
    # fp32 throughout: the two differ by the order of sums of 1,800 and 96 terms
    torch.testing.assert_close(logp, want_logp, rtol=1e-5, atol=2e-5)
    torch.testing.assert_close(entropy, want_entropy, rtol=1e-5, atol=2e-5)
    torch.testing.assert_close(value, v, rtol=1e-4, atol=2e-5)
    (c * want_logp + 0.3 * want_entropy + c * v).sum().backward()
    for a, p in zip(got, model.parameters()):
        assert float((a - p.grad).norm() / p.grad.norm()) < 1e-4
    with torch.no_grad():
        m = state
        for t in range(20):
            number, action, sampled, one, m = model.act(obs[t], 9, t, m, reset[t])
            step_logits, _, _ = model(obs[t:t + 1], m, None)
            assert torch.equal(number, action) and number.shape == (12,)
            torch.testing.assert_close(one, v[t], rtol=1e-4, atol=2e-5)
        torch.testing.assert_close(m, last, rtol=1e-4, atol=2e-5)


def test_sequence_step(mods):
    """One minibatch's loss and gradients, with a reference and a value clip, against elementary operations."""
    pkg, P, ppo, _ = mods
    print('[memory] sequence step', flush=True)
    obs, actions, reset, g = sequence(pkg, P, seed=5)
    model, ref = P.MemoryPolicy(width=64, seed=2).cuda(), P.MemoryPolicy(width=64, seed=3).cuda()
    state = torch.randn(12, 64, device=DEV, generator=g)
    old, adv, ret, old_v = (torch.randn(20, 12, device=DEV, generator=g) * s for s in (0.1, 1.0, 1.0, 0.3))
    old -= 2.7
    mine = ppo.SequencePPO(copy.deepcopy(model), autocast=False, clip=(0.1, 0.3), value_clip=0.2, kl_coef=0.3, reference=ref,
                           max_grad_norm=1e9)
    loss = mine.sequence_step(obs, actions, old, adv, ret, state, reset, old_v)
    logits, v, _ = plain(model, obs, state, reset)
    lp = torch.log_softmax(logits, -1)
    logp, entropy = lp.gather(-1, actions[..., None])[..., 0], -(lp.exp() * lp).sum(-1)
    with torch.no_grad():
        ref_lp = torch.log_softmax(plain(ref, obs, torch.zeros_like(state), reset)[0], -1).gather(-1, actions[..., None])[..., 0]
    r = (logp - old).exp()
    x = ref_lp - logp
    near = old_v + (v - old_v).clamp(-0.2, 0.2)
    terms = dict(policy=-torch.minimum(r * adv, r.clamp(0.9, 1.3) * adv).mean(), kl=(x.exp() - 1 - x).mean(), entropy=entropy.mean(),
                 value=0.5 * torch.maximum((v - ret) ** 2, (near - ret) ** 2).mean())
    want = terms['policy'] + 0.5 * terms['value'] - 0.01 * terms['entropy'] + 0.3 * terms['kl']
    torch.testing.assert_close(loss, want.detach(), rtol=1e-4, atol=1e-5)
    for n, t in terms.items():
        torch.testing.assert_close(getattr(mine.terms, n), t.detach(), rtol=1e-3, atol=1e-5)
    want.backward()
    for p, q in zip(mine.model.parameters(), model.parameters()):
        assert float((p.grad - q.grad).norm()) <= 2e-4 * float(q.grad.norm()) + 1e-7


@pytest.mark.parametrize('optimizer', ['adamw', 'muon'])
@pytest.mark.parametrize('kind', ['memory', 'norm', 'ar'])
def test_training_loop(mods, kind, optimizer):
    """Two updates of a small run with all of it together; the same seeds give the same actions and all but the same weights."""
    pkg, P, ppo, train = mods
    print(f'[memory] loop {kind} {optimizer}', flush=True)
    make = dict(memory=lambda: P.MemoryPolicy(width=128, seed=6), norm=lambda: P.NormPolicy(width=128, seed=6), ar=lambda: P.ARPolicy(seed=6))

    def run():
        env = pkg.Env(128, pkg.baseline_config(), seed=5, hash=False)
        model = make[kind]().cuda()
        ref = copy.deepcopy(model)
        before = [p.detach().clone() for p in model.parameters()]
        tr = train.ModuleTrainer(env, model, horizon=8, minibatch=512, epochs=2, optimizer=optimizer, kl_coef=0.1, reference=ref,
                                 value_clip=0.2, clip=(0.2, 0.3))
        loss = tr.train(2)
        assert bool(torch.isfinite(loss)) and tr.ppo.opt.skipped_steps() == 0
        assert bool(torch.isfinite(tr.ppo.terms.terms).all()) and int(tr.ppo.terms.count) == 512
        for p, q in zip(model.parameters(), before):
            assert bool(torch.isfinite(p).all())
        assert sum(not torch.equal(p, q) for p, q in zip(model.parameters(), before)) >= len(before) - 1
        assert all(torch.equal(p, q) for p, q in zip(ref.parameters(), before))
        return [p.detach().clone() for p in model.parameters()], tr.buf.actions.clone()

    p1, a1 = run()
    p2, a2 = run()
    assert torch.equal(a1, a2)
    # the trunk's products are the library's, whose order of sums may differ between runs
    for p, q in zip(p1, p2):
        torch.testing.assert_close(p, q, rtol=1e-3, atol=2e-3)


def test_memory_goes_on(mods):
    """A rollout starts from the state that the one before left; worlds whose episode ended start from nothing."""
    pkg, P, ppo, train = mods
    print('[memory] goes on', flush=True)
    env = pkg.Env(64, pkg.baseline_config(), seed=9, hash=False)
    tr = train.ModuleTrainer(env, P.MemoryPolicy(width=32, seed=1).cuda(), horizon=16, minibatch=256, epochs=1, autocast=False)
    model = tr.model
    for n in range(3):
        first = tr.state.clone()
        buf = tr.rollout()
        assert torch.equal(buf.state, first)
        with torch.no_grad():
            logits, value, last = model(buf.obs, buf.state, buf.resets)
        torch.testing.assert_close(value, buf.values, rtol=1e-4, atol=1e-4)
        torch.testing.assert_close(last, tr.state, rtol=1e-4, atol=1e-4)
        assert torch.equal(buf.resets[1:], buf.dones[:-1]) and torch.equal(tr.reset, buf.dones[-1])
        assert torch.equal(buf.state, first)
    tr.update()


def test_not_finite_raises(mods):
    pkg, P, ppo, train = mods
    for optimizer in ('adamw', 'muon'):
        env = pkg.Env(64, pkg.baseline_config(), seed=8, hash=False)
        model = P.MemoryPolicy(width=32, seed=9).cuda()
        tr = train.ModuleTrainer(env, model, horizon=8, minibatch=512, epochs=1, optimizer=optimizer)
        tr.rollout()
        before = [p.detach().clone() for p in model.parameters()]
        tr.buf.rewards[3, 5] = float('nan')
        with pytest.raises(RuntimeError, match='Non-finite'):
            tr.update()
        assert all(torch.equal(p, q) for p, q in zip(model.parameters(), before))
        tr.train(1)
    for k in (dict(optimizer='sgd'), dict(kl_coef=0.1)):
        with pytest.raises(ValueError):
            ppo.ModulePPO(model, **k)
