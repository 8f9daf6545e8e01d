"""A step in two parts with another in between: what it refuses, and what a part leaves alone."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'


@pytest.fixture(scope='module')
def O():
    return importlib.import_module('dcss-auto_amd.optim')


def test_the_other_step(O):
    p, g, m, v = (torch.randn(50, device=DEV) for _ in range(4))
    v.abs_()
    step, other = (torch.zeros(8, dtype=torch.int32, device=DEV) for _ in range(2))
    before = p.clone()
    for bad in (step, other[:4], other.float(), other.cpu(), other.view(2, 4), torch.zeros(16, dtype=torch.int32, device=DEV)[::2]):
        with pytest.raises(ValueError, match='other'):
            O.adamw_step([p], [g], [m], [v], step, other=bad)
    assert torch.equal(p, before) and int(step.abs().sum()) == 0


def test_the_parts(O):
    """The first part writes the counts alone; after the second all is as from a whole step, also with another between that skips."""
    make = lambda: [torch.nn.Parameter(torch.randn(s, generator=torch.Generator(DEV).manual_seed(i), device=DEV)) for i, s in enumerate(((70, 90), (5, 300)))]  # noqa: E731
    a, b = make(), make()
    whole, parts = O.Muon(a), O.Muon(b)
    assert parts.begin() is None                     # no gradients
    for n in range(3):
        for i, (x, y) in enumerate(zip(a, b)):
            x.grad = torch.randn(x.shape, generator=torch.Generator(DEV).manual_seed(10 * n + i), device=DEV)
            y.grad = x.grad.clone()
        whole.step()
        before = [y.detach().clone() for y in b] + [parts.state[y]['momentum'].clone() for y in b if parts.state[y]]
        begun = parts.begin()
        now = [y.detach() for y in b] + [parts.state[y]['momentum'] for y in b][:len(before) - 2]
        assert all(torch.equal(x, y) for x, y in zip(before, now)) and int(parts.ctl[0]) == n + 1
        parts.finish(begun)
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(whole.ctl, parts.ctl)
    before = [y.detach().clone() for y in b]
    begun = parts.begin()
    q, zero = torch.randn(50, device=DEV), [torch.zeros(50, device=DEV) for _ in range(2)]
    step, kept = torch.zeros(8, dtype=torch.int32, device=DEV), q.clone()
    O.adamw_step([q], [torch.full((50,), float('inf'), device=DEV)], zero[:1], zero[1:], step, max_grad_norm=1.0, other=parts.ctl)
    parts.finish(begun)
    assert all(torch.equal(x, y) for x, y in zip(before, b)) and torch.equal(q, kept)
    assert parts.ctl[:2].tolist() == [3, 1] and step[:2].tolist() == [0, 1]
