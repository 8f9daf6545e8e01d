"""muon_step over nothing."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'


@pytest.fixture(scope='module')
def O():
    return importlib.import_module('dcss-auto_amd.optim')


def test_no_matrices(O):
    """A step of nothing is a step, as one of empty matrices is."""
    step = torch.zeros(8, dtype=torch.int32, device=DEV)
    O.muon_step([], [], [], step)
    assert step[:2].tolist() == [1, 0]
    none = [torch.zeros(0, 5, device=DEV) for _ in range(3)]
    O.muon_step(none[:1], none[1:2], none[2:], step)
    assert step[:2].tolist() == [2, 0]
