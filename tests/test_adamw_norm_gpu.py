"""The global norm where a workgroup's chunks pass from one tensor to the next, where its sums come from several
launches, and where there is nothing to sum."""
import importlib
import math

import pytest
import torch

from test_adamw_gpu import B1, B2, EPS, LR, U, WD, clip_of, compare, tensors

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def A():
    return importlib.import_module('dcss-auto_amd.optim')


# more than 2,048 chunks a launch, an odd number in each tensor: chunks of 1,024 elements in one launch and two, and of 4,096
@pytest.mark.parametrize('sizes', [[70001] * 40, [70001] * 45, [290001] * 40, [290001] * 41 + [5, 0, 3]],
                         ids=lambda s: f'{len(s)}x{max(s)}')
def test_chunks_pass_from_tensor_to_tensor(A, sizes):
    print(f'[adamw] norm over {len(sizes)} tensors of {max(sizes)}', flush=True)
    p, g, m, v = tensors(sizes, len(sizes) + 1)
    for k, x in enumerate(g):
        x *= 1 + k                                    # a chunk read from the wrong tensor changes the norm
    step = torch.zeros(8, dtype=torch.int32, device='cuda')
    call = lambda: A.adamw_step(p, g, m, v, step, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, max_grad_norm=0.5)  # noqa: E731
    for t in (1, 2):
        before = [tuple(x.clone() for x in z) for z in zip(p, g, m, v)]
        call()
        coef, norm = clip_of(g, 0.5)
        compare(list(zip(p, m, v)), before, t, coef)
        assert step[:2].tolist() == [t, 0] and abs(float(step[5:6].view(torch.float32)) - norm) <= 2 * U * norm
    kept = [x.clone() for x in (*p, *m, *v)]
    for k, (at, where) in enumerate(((1, 0), (20, sizes[20] - 1), (len(sizes) - 1, 0), (39, sizes[39] - 1))):
        was = float(g[at][where])
        g[at][where] = math.inf                       # one element of one tensor
        call()
        assert step[:2].tolist() == [2, k + 1]
        g[at][where] = was
    assert all(torch.equal(a, b) for a, b in zip(kept, (*p, *m, *v)))


def test_norm_of_nothing(A):
    """A step without elements has a norm of 0, not that of the step before."""
    print('[adamw] norm of nothing', flush=True)
    step = torch.zeros(8, dtype=torch.int32, device='cuda')
    p, g, m, v = tensors([9], 1)
    A.adamw_step(p, g, m, v, step, max_grad_norm=1.0)
    assert float(step[5:6].view(torch.float32)) > 0
    A.adamw_step([], [], [], [], step, max_grad_norm=1.0)
    assert step[:2].tolist() == [2, 0] and float(step[5:6].view(torch.float32)) == 0
    A.adamw_step(p, g, m, v, step, max_grad_norm=1.0)
    p, g, m, v = tensors([0, 0], 1)
    A.adamw_step(p, g, m, v, step, max_grad_norm=1.0)
    assert step[:2].tolist() == [4, 0] and float(step[5:6].view(torch.float32)) == 0
