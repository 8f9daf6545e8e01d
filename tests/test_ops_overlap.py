"""The C calls refuse a gradient written over the logits it is made from, and each of their other arguments
by itself, all pointers being different (no GPU needed)."""
import importlib

import pytest

F = [0x10000000 * (k + 1) for k in range(9)]      # made-up device addresses: rejected calls never read them


@pytest.fixture(scope='module')
def L():
    return importlib.import_module('dcss-auto_amd._lib').load_ops()


def test_gradient_over_the_logits(L):
    good = [F[0], 0, 4, 5000, 5000, F[1], None, 0, F[2], F[3], F[4], F[5], F[6], None]
    for rows, vocab, stride in ((4, 5000, 5000), (4, 5000, 6000), (300, 9, 9), (1, 1, 0)):
        args = list(good)
        args[2], args[3], args[4], args[12] = rows, vocab, stride, F[0]
        assert L.d1_tokens_bwd(*args) == -1, (rows, vocab, stride)
    args = list(good)
    args[2], args[12] = 0, F[0]
    assert L.d1_tokens_bwd(*args) == 0            # nothing is written


def test_other_arguments(L):
    good = [F[0], 0, 4, 5000, 5000, F[1], None, 0, F[2], F[3], F[4], F[5], F[6], None]
    for at, bad in ((0, None), (1, 9), (2, -1), (3, 0), (4, -1), (5, None), (7, -1), (8, None), (9, None), (12, None)):
        args = list(good)
        args[at] = bad
        assert L.d1_tokens_bwd(*args) == -1, at
