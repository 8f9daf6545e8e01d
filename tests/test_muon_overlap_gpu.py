"""Gradients that lie on what muon_step writes are refused; those beside it, shared or copied first are not."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'


@pytest.fixture(scope='module')
def O():
    return importlib.import_module('dcss-auto_amd.optim')


def test_gradients_on_what_is_written(O):
    flat = torch.randn(400, device=DEV)
    at = lambda i, dtype=torch.float32: flat.view(dtype)[i:i + 72].view(8, 9)  # noqa: E731
    before, step = flat.clone(), torch.zeros(8, dtype=torch.int32, device=DEV)
    copy = at(400, torch.bfloat16)              # bytes 800 to 944
    for p, g, m, c in ((0, 0, 100, None), (0, 100, 100, None), (0, 71, 100, None), (0, 171, 100, None), (0, 200, 100, copy), (0, 150, 100, None)):
        with pytest.raises(ValueError, match='overlap'):
            O.muon_step([at(p)], [at(g)], [at(m)], step, copies=None if c is None else [c])
    # one's gradient on another's parameter
    other = [torch.zeros(8, 9, device=DEV) for _ in range(3)]
    with pytest.raises(ValueError, match='overlap'):
        O.muon_step([at(0), other[0]], [other[1], at(0)], [at(100), other[2]], step)
    assert torch.equal(flat, before) and int(step.abs().sum()) == 0


def test_gradients_beside_and_shared(O):
    """Neighbours are no overlap, one gradient may be two parameters', and one that is copied first may lie anywhere."""
    flat = torch.randn(400, device=DEV)
    at = lambda i: flat[i:i + 72].view(8, 9)  # noqa: E731
    step = torch.zeros(8, dtype=torch.int32, device=DEV)
    want = [at(0).clone(), at(72).clone(), at(144).clone()]
    O.muon_step([want[0]], [want[1]], [want[2]], step)
    O.muon_step([at(0)], [at(72)], [at(144)], step)
    assert torch.equal(at(0), want[0]) and torch.equal(at(144), want[2])
    g = torch.randn(8, 9, device=DEV)
    p, m = [torch.zeros(8, 9, device=DEV) for _ in range(2)], [torch.zeros(8, 9, device=DEV) for _ in range(2)]
    O.muon_step(p, [g, g], m, step)
    assert torch.equal(p[0], p[1]) and bool((p[0] != 0).any())
    square = torch.randn(9, 9, device=DEV)
    p, turned = square.clone(), square.clone()
    O.muon_step([p], [square.t()], [torch.zeros(9, 9, device=DEV)], step)
    O.muon_step([turned], [turned.t()], [torch.zeros(9, 9, device=DEV)], step)
    assert torch.equal(p, turned)
