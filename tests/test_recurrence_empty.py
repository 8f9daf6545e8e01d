"""gated_scan over an empty batch: as many steps as a sequence that is cut has, and no rows."""
import ctypes as C
import importlib
import subprocess
import sys

import pytest
import torch

from conftest import ROOT


@pytest.mark.parametrize('steps', [0, 1, 64, 192, 193, 300, 1 << 30])
def test_no_rows_need_no_memory(steps):
    """In a process of its own: a division by the number of rows ends it."""
    code = ('import ctypes as C, importlib\n'
            'lib = importlib.import_module("dcss-auto_amd._lib")\n'
            'L = lib.load_ops()\n'
            f'print(*(L.d1_scan_work_bytes(C.byref(lib.D1Scan(steps={steps}, rows=r, width=w, type=t)))'
            ' for r, w in ((0, 16), (0, 1000), (3, 0), (0, 0)) for t in range(3)))\n')
    r = subprocess.run([sys.executable, '-c', code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr)
    assert r.stdout.split() == ['0'] * 12


def test_one_row_still_needs_memory():
    lib = importlib.import_module('dcss-auto_amd._lib')
    assert lib.load_ops().d1_scan_work_bytes(C.byref(lib.D1Scan(steps=300, rows=1, width=16))) > 0


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(300, 0, 16), (300, 0, 1000), (70, 0, 3), (300, 5, 0), (300, 0)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_empty_batch(shape, dtype):
    R = importlib.import_module('dcss-auto_amd.recurrence')
    x, gate = (torch.zeros(shape, device='cuda', dtype=dtype).requires_grad_() for _ in range(2))
    state = torch.zeros(shape[1:], device='cuda').requires_grad_()
    reset = torch.zeros(shape[:-1], device='cuda', dtype=torch.bool)
    with torch.no_grad():
        h, last = R.gated_scan(x, gate, state, reset)
    assert h.shape == shape and h.dtype == dtype and last.shape == shape[1:]
    h, last = R.gated_scan(x, gate, state, reset)
    (h.sum() + last.sum()).backward()
    assert x.grad.shape == shape and gate.grad.shape == shape and state.grad.shape == shape[1:]
