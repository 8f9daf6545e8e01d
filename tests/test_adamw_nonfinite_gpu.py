"""Gradients that are not finite (or whose square is not) without a clip: the element alone is lost."""
import importlib
import math

import pytest
import torch

from test_adamw_gpu import eight

pytestmark = pytest.mark.gpu
N, BAD = 700, (300, 699)               # elements, of them the bad ones: one inside a full block, one the last of a part


@pytest.fixture(scope='module')
def A():
    return importlib.import_module('dcss-auto_amd.optim')


@pytest.mark.parametrize('value', [math.inf, -math.inf, math.nan, 3e38, -3e38], ids=str)
@pytest.mark.parametrize('bits', [32, 8])
def test_neighbours_go_on(A, bits, value):
    """Beside a run whose bad elements have a gradient of 0 in that step: all other elements, their moments' values and
    what they do in the steps after have the same bits; 8-bit moments are finite throughout, and a lost
    element whose parameter is finite (3e38, whose square is not) takes ordinary steps again."""
    print(f'[adamw] neighbours {bits} {value}', flush=True)
    gen = torch.Generator(device='cuda').manual_seed(3)
    start = torch.randn(N, generator=gen, device='cuda')
    grads = [torch.randn(N, generator=gen, device='cuda') * 0.1 for _ in range(6)]
    for g in grads:
        g[list(BAD)] = 1e-3            # never their blocks' largest
    rest = torch.ones(N, dtype=torch.bool, device='cuda')
    rest[list(BAD)] = False

    def run(bad):
        p = [start.clone()]
        if bits == 8:
            m, v, exps = eight(A, [N])
        else:
            m, v, exps = [torch.zeros(N, device='cuda')], [torch.zeros(N, device='cuda')], None
        step = torch.zeros(8, dtype=torch.int32, device='cuda')
        for t, g in enumerate(grads):
            g = g.clone()
            if t == 2:
                g[list(BAD)] = bad
            before = p[0].clone()
            A.adamw_step(p, [g], m, v, step, lr=1e-2, exps=exps, counters=[0], seed=4)
            a, b = m[0], v[0]
            if bits == 8:
                a, b = A.read_moment(a, exps[0][0], signed=True), A.read_moment(b, exps[1][0], signed=False)
                assert torch.isfinite(a).all() and torch.isfinite(b).all()
            yield p[0].clone(), a.clone(), b.clone(), p[0] - before

    for t, (got, want) in enumerate(zip(run(value), run(0.0))):
        assert all(torch.equal(x[rest], y[rest]) for x, y in zip(got, want)), t
        if t >= 2 and not math.isfinite(value):
            assert not torch.isfinite(got[0][~rest]).any()
        elif bits == 8:
            # |m|/sqrt(v) of b1 = 0.9, b2 = 0.999 over at most 4 steps: under 0.1/sqrt(0.001) times the corrections
            assert torch.isfinite(got[0]).all() and float(got[3].abs().max()) < 1e-2 * 3.2 / 0.1
