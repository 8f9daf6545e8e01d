"""libd1ops.so: its exports, struct layouts and the arguments it rejects before any launch (no GPU
needed), and the rounding draws of the 8-bit moments."""
import ctypes as C
import importlib
import subprocess

import numpy as np
import pytest

import adamw_ref as R
from conftest import ROOT
from test_abi import declared_symbols

F = 1 << 20            # a made-up device address: rejected calls never read it


@pytest.fixture(scope='module')
def lib():
    return importlib.import_module('dcss-auto_amd._lib')


def test_exports(lib):
    assert declared_symbols('d1ops.h') == sorted(lib.OPS_SYMBOLS)
    L = lib.load_ops()
    for name in lib.OPS_SYMBOLS:
        assert hasattr(L, name), name


@pytest.mark.parametrize('name', ['D1AdamWTensor', 'D1AdamW'])
def test_struct_layout(lib, tmp_path, name):
    fields = [f for f, _ in getattr(lib, name)._fields_]
    src = tmp_path / 'layout.c'
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "d1ops.h"\nint main(void) {\n'
                   f'  printf("%zu\\n", sizeof({name}));\n' +
                   ''.join(f'  printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields) + '  return 0;\n}\n')
    exe = tmp_path / 'layout'
    subprocess.run(['gcc', '-I', str(ROOT / 'include'), '-o', str(exe), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(getattr(lib, name))] + [getattr(getattr(lib, name), f).offset for f in fields]


def test_tokens_arguments(lib):
    L = lib.load_ops()
    assert L.d1_tokens_work_bytes(8, 1000, 5) == 0 and L.d1_tokens_work_bytes(8, 5000, 5) == 0 and L.d1_tokens_work_bytes(8, 100000, 5) > 0
    for rows, vocab, top in ((-1, 5, 0), (1, 0, 0), (1, 5, 6), (1, 100, 65), (1, 5, -1), (1, (1 << 24) + 1, 0)):
        assert L.d1_tokens_work_bytes(rows, vocab, top) == -1
    good = [F, 0, 4, 100000, 100000, F, None, 0, 3, F, F, F, F, F, F, 1 << 20, None]     # long enough to be cut into segments
    assert L.d1_tokens_fwd(*good[:2], 0, *good[3:]) == 0
    for at, bad in ((0, None), (1, 3), (1, -1), (2, -1), (3, 0), (4, -1), (5, None), (7, -1), (8, 65), (9, None), (10, None),
                    (11, None), (12, None), (13, None), (14, None), (14, F + 4), (15, 7)):
        args = list(good)
        args[at] = bad
        assert L.d1_tokens_fwd(*args) == -1, at
    good = [F, 0, 4, 5000, 5000, F, None, 0, F, F, F, F, F, None]
    assert L.d1_tokens_bwd(*good[:2], 0, *good[3:]) == 0
    for at, bad in ((0, None), (1, 9), (2, -1), (3, 0), (4, -1), (5, None), (7, -1), (8, None), (9, None), (12, None)):
        args = list(good)
        args[at] = bad
        assert L.d1_tokens_bwd(*args) == -1, at


def test_norm_arguments(lib):
    L = lib.load_ops()
    good = [F, 1, 4, 300, 300, F, F, 0, 1e-5, F, F, F, None]
    assert L.d1_norm_fwd(*good[:2], 0, *good[3:]) == 0
    for at, bad in ((0, None), (1, 5), (2, -1), (3, 0), (3, 16385), (4, -1), (7, 2), (9, None), (10, None), (11, None)):
        args = list(good)
        args[at] = bad
        assert L.d1_norm_fwd(*args) == -1, at
    need = L.d1_norm_work_bytes(4, 300, 1)
    assert need > 0 and L.d1_norm_work_bytes(4, 16385, 1) == -1 and L.d1_norm_work_bytes(4, 30, 7) == -1
    good = [F, 300, F, 1, 4, 300, 300, F, 0, F, F, F, F, F, F, need, None]
    for at, bad in ((0, None), (1, -1), (2, None), (3, 4), (4, -1), (5, 0), (6, -1), (8, 2), (9, None), (10, None), (11, None),
                    (14, None), (15, need - 1)):
        args = list(good)
        args[at] = bad
        assert L.d1_norm_bwd(*args) == -1, at
    assert L.d1_norm_bwd(None, 0, None, 1, 0, 300, 0, None, 0, None, None, None, None, None, None, 0, None) == 0


def test_adamw_arguments(lib):
    L = lib.load_ops()

    def call(hyper=(), count=1, ctl=F, work=F, size=1 << 20, **fields):
        t = lib.D1AdamWTensor(p=F, g=F, m=F, v=F, m_exp=F, v_exp=F, n=1000, lr=1e-3, weight_decay=0.1)
        for name, value in fields.items():
            setattr(t, name, value)
        h = lib.D1AdamW(0.9, 0.999, 1e-8, 1.0, 0, 8)
        for name, value in hyper:
            setattr(h, name, value)
        return L.d1_adamw_step(C.byref(t), count, C.byref(h), ctl, work, size, None), L.d1_adamw_work_bytes(C.byref(t), count, C.byref(h))

    for fields in (dict(p=None), dict(g=None), dict(m=None), dict(v=None), dict(m_exp=None), dict(v_exp=None), dict(n=-1),
                   dict(n=(4096 << 23) + 1), dict(lag=-1), dict(lr=-1.0), dict(lr=float('nan')), dict(weight_decay=-1.0),
                   dict(ptype=2), dict(gtype=2), dict(count=-1)):
        assert call(**fields) == (-1, -1), fields
    for hyper in ((('bits', 16),), (('beta1', 1.0),), (('beta2', -0.5),), (('eps', -1.0),), (('max_norm', -1.0),),
                  (('max_norm', float('nan')),)):
        assert call(hyper=hyper) == (-1, -1), hyper
    for more in (dict(ctl=None), dict(work=None), dict(size=7), dict(work=F + 4)):
        code, need = call(**more)
        assert code == -1 and need == 8, more
    h = lib.D1AdamW(0.9, 0.999, 1e-8, 0.0, 0, 8)
    assert L.d1_adamw_work_bytes(None, 0, C.byref(h)) == 0 and L.d1_adamw_work_bytes(None, 1, C.byref(h)) == -1
    assert L.d1_adamw_read(None, None, 0, 1, None, None) == 0
    for args in ((None, F, 4, 1, F), (F, None, 4, 1, F), (F, F, 4, 1, None), (F, F, -1, 1, F), (F, F, 4, 2, F)):
        assert L.d1_adamw_read(*args, None) == -1


def test_cpu_tensors_are_refused():
    import torch
    T, N, A = (importlib.import_module('dcss-auto_amd.' + n) for n in ('tokens', 'norm', 'optim'))
    with pytest.raises(ValueError, match='CUDA'):
        T.token_logprobs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match='CUDA'):
        N.layer_norm(torch.zeros(2, 3))
    with pytest.raises(ValueError, match='CUDA'):
        A.adamw_step([torch.zeros(3)], [torch.zeros(3)], [torch.zeros(3)], [torch.zeros(3)], torch.zeros(8, dtype=torch.int32))


def test_missing_library_raises(monkeypatch, tmp_path, lib):
    monkeypatch.setattr(lib, '_OPS', None)
    monkeypatch.setattr(lib, 'HERE', tmp_path)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        lib.load_ops()
    monkeypatch.setattr(lib, '_OPS_TORCH', None)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        lib.load_ops_torch()


def test_torch_module_loads(lib):
    """The binding finds libd1ops.so beside it and offers every call that the Python surface makes."""
    m = lib.load_ops_torch()
    for name in ('tokens_fwd', 'tokens_bwd', 'norm_fwd', 'norm_bwd', 'adamw_step', 'adamw_read'):
        assert callable(getattr(m, name)), name


def test_draws_are_uniform_and_independent():
    """2^20 draws of neighbouring counters: both 16-bit halves uniform over 256 bins (chi-square of 255
    degrees, mean 255, deviation 22.6: under 255 + 6 x 22.6), neighbours, steps and halves uncorrelated
    (a correlation of n draws deviates by 1/sqrt(n) = 1e-3: under 6e-3)."""
    n = 1 << 20
    words = {step: R.draws(77, step, np.arange(n)) for step in (1, 2)}
    high = {s: (w >> np.uint64(16)).astype(np.int64) for s, w in words.items()}
    low = {s: (w & np.uint64(0xFFFF)).astype(np.int64) for s, w in words.items()}
    for d in (high[1], low[1], high[2], low[2]):
        for part in (d >> 8, d & 255):
            count = np.bincount(part, minlength=256)
            assert ((count - n / 256) ** 2 / (n / 256)).sum() < 255 + 6 * 22.6
    corr = lambda a, b: abs(np.corrcoef(a, b)[0, 1])  # noqa: E731
    for a, b in ((high[1][:-1], high[1][1:]), (low[1][:-1], low[1][1:]), (high[1], high[2]), (low[1], low[2]),
                 (high[1], low[1]), (low[1][:-256], low[1][256:])):
        assert corr(a, b) < 6e-3


def test_codes_of_every_value():
    """Each code stands for a value that encodes to itself whatever the draw; a value between two codes
    becomes one of them, the upper with the share of the way there; the largest never overflows."""
    for top, count in ((15, 128), (31, 256)):
        code = np.arange(count, dtype=np.uint8)
        x = R.decode(code, np.array([130], np.uint8), top)
        assert (np.diff(x) > 0).all()
        for draw in (0, 1, 40000, 65535):
            c, e = R.encode(x, top, np.full(count, draw))
            # the largest code's value has the mantissa that keeps the block's exponent
            assert e[0] == 130 and np.array_equal(c, code)
        between = np.float32(0.75) * x[50] + np.float32(0.25) * x[51]
        block = np.full(256, between, np.float32)
        block[0] = x[-1]
        up = [R.encode(block, top, np.full(256, d))[0][1] for d in range(0, 65536, 64)]
        assert set(up) == {50, 51} and abs(np.mean(np.array(up) == 51) - 0.25) < 2e-3
        huge = np.full(256, np.float32(1.99999988), np.float32)
        for draw in (0, 65535):
            c, e = R.encode(huge, top, np.full(256, draw))
            assert abs(R.decode(c, e, top) / 2 - 1).max() <= 1 / 16
