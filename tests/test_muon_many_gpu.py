"""orthogonalize of so many matrices that the numbers of their sums pass 32 bits."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_two_million_matrices():
    """2^21 + 70 scalars, 1,024 sums kept for each: a scalar's sign times what the quintic makes of 1."""
    O = importlib.import_module('dcss-auto_amd.optim')
    print('[muon] 2^21 matrices', flush=True)
    n = 2 ** 21 + 70
    u = torch.rand(n, 1, 1, generator=torch.Generator('cuda').manual_seed(1), device='cuda') + 0.5
    u[::3] *= -1
    out = O.orthogonalize(u, steps=1, eps=0.0)
    a, b, c = O.NEWTON_SCHULZ
    # each of X, A and B to 22 bits, coefficients and sums in fp32; the factor is a sum of terms up to 4.8
    off = float((out.double() - (a + b + c) * u.double().sign()).abs().max())
    assert off <= 64 * 2.0 ** -22, off
