"""Training with the same seeds twice."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('bits', [32, 8])
def test_optimizer_repeats_its_bits(pkg, bits):
    """The same gradients: the same parameters, moments and codes, bit for bit, through clips and a skipped step."""
    print(f'[repeat] optimizer {bits}', flush=True)
    A = importlib.import_module('dcss-auto_amd.optim')

    def run():
        gen = torch.Generator(device='cuda').manual_seed(1)
        ps = [torch.nn.Parameter(torch.randn(n, generator=gen, device='cuda')) for n in ((256, 1800), (256,), (17, 256), (300001,))]
        opt = A.AdamW(ps, lr=1e-2, state_bits=bits, max_grad_norm=0.5, seed=6)
        for t in range(6):
            for p in ps:
                p.grad = torch.randn(p.shape, generator=gen, device='cuda')
            if t == 3:
                ps[1].grad[7] = float('nan')
            opt.step()
        return [x.clone() for p in ps for x in (p.detach(), *opt.moments(p))] + [opt.ctl.clone()]

    a, b = run(), run()
    assert a[-1][:2].tolist() == [5, 1] and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('kind', ['norm', 'ar'])
def test_training_repeats(pkg, kind, bits):
    """Two updates from the same seeds end within a fiftieth of their movement of one another (the products' sums may be
    in another order, as between two implementations of a minibatch), each tensor by itself."""
    print(f'[repeat] training {kind} {bits}', flush=True)
    P, train = (importlib.import_module('dcss-auto_amd.' + n) for n in ('policy', 'train'))
    make = lambda: (P.NormPolicy(width=128, seed=6) if kind == 'norm' else P.ARPolicy(seed=6)).cuda()  # noqa: E731

    def run():
        model = make()
        tr = train.ModuleTrainer(pkg.Env(128, pkg.baseline_config(), seed=5, hash=False), model, horizon=8, minibatch=512,
                                 epochs=2, state_bits=bits)
        tr.train(2)
        return [p.detach().clone() for p in model.parameters()]

    for p, q, s in zip(run(), run(), make().parameters()):
        moved = float((q - s.detach()).norm())
        assert moved > 0 and float((p - q).norm()) <= 2e-2 * moved
