"""libd1ops.so: struct layouts and rejected arguments of the policy loss, the gated recurrence and the orthogonalised
updates (no GPU needed: rejected calls never launch)."""
import ctypes as C
import importlib
import subprocess

import pytest

from conftest import ROOT

F = 1 << 20            # a made-up device address: rejected calls never read it


@pytest.fixture(scope='module')
def lib():
    return importlib.import_module('dcss-auto_amd._lib')


@pytest.mark.parametrize('name', ['D1LossInput', 'D1PolicyLoss', 'D1Scan', 'D1MuonTensor', 'D1Muon'])
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


def test_loss_arguments(lib):
    L = lib.load_ops()
    flat = lambda type=0: lib.D1LossInput(data=F, row=100, step=1, type=type)  # noqa: E731

    def loss(**k):
        base = dict(logp=flat(), old_logp=flat(), advantages=flat(), rows=20, length=100, clip_low=0.2, clip_high=0.2)
        return lib.D1PolicyLoss(**dict(base, **k))
    good = loss()
    need = L.d1_policy_loss_work_bytes(C.byref(good))
    assert need == 0                           # 2,000 tokens are one workgroup's
    many = loss(rows=1000)
    assert L.d1_policy_loss_work_bytes(C.byref(many)) > 0
    masked = loss(rows=1000, mask=flat(), sequence=1)
    assert L.d1_policy_loss_work_bytes(C.byref(masked)) > L.d1_policy_loss_work_bytes(C.byref(many)) + 4 * 1000
    bad = [dict(rows=-1), dict(length=-1), dict(clip_low=-0.1), dict(clip_low=1.1), dict(clip_high=-1.0), dict(clip_high=float('nan')),
           dict(value_clip=-1.0), dict(kl_coef=float('inf')), dict(value_coef=float('nan')), dict(sequence=2), dict(logp=flat(3)),
           dict(old_logp=lib.D1LossInput()), dict(advantages=lib.D1LossInput()), dict(values=flat()), dict(returns=flat()),
           dict(values=flat(), returns=flat(), value_clip=0.1), dict(ref_logp=flat(-1)), dict(rows=1 << 30, length=1 << 30),
           dict(mask=lib.D1LossInput(data=F, row=-1, step=1)), dict(entropy=lib.D1LossInput(data=F, row=1, step=-1))]
    for k in bad:
        h = loss(**k)
        assert L.d1_policy_loss_work_bytes(C.byref(h)) == -1, k
        assert L.d1_policy_loss(C.byref(h), F, None, None, None, F, 1 << 30, None) == -1, k
    assert L.d1_policy_loss(C.byref(good), None, None, None, None, None, 0, None) == -1
    assert L.d1_policy_loss(C.byref(good), F, None, F, None, None, 0, None) == -1        # an entropy gradient without an entropy
    assert L.d1_policy_loss(C.byref(many), F, None, None, None, None, 0, None) == -1
    assert L.d1_policy_loss(C.byref(many), F, None, None, None, F, 8, None) == -1
    assert L.d1_policy_loss(None, F, None, None, None, None, 0, None) == -1
    assert L.d1_scale(F, F, 9, 4, F, None) == -1 and L.d1_scale(None, F, 0, 4, F, None) == -1 and L.d1_scale(F, F, 0, -1, F, None) == -1
    assert L.d1_scale(F, None, 0, 4, F, None) == -1 and L.d1_scale(None, None, 0, 0, None, None) == 0


def test_scan_arguments(lib):
    L = lib.load_ops()

    def scan(**k):
        return lib.D1Scan(**dict(dict(x=F, gate=F, x_t=64, gate_t=64, steps=1000, rows=1, width=64), **k))
    good = scan()
    assert L.d1_scan_marks(C.byref(good)) == 15 and L.d1_scan_marks(C.byref(scan(steps=64))) == 0
    need = L.d1_scan_work_bytes(C.byref(good))
    assert need > 0 and L.d1_scan_work_bytes(C.byref(scan(steps=8))) == 0
    for k in (dict(steps=-1), dict(rows=-1), dict(width=-1), dict(type=3), dict(width=(1 << 24) + 1), dict(steps=(1 << 30) + 1),
              dict(rows=1 << 43)):
        h = scan(**k)
        assert L.d1_scan_marks(C.byref(h)) == -1 and L.d1_scan_work_bytes(C.byref(h)) == -1, k
        assert L.d1_scan_fwd(C.byref(h), F, 64, 0, F, F, 1 << 30, None) == -1, k
    for k in (dict(x=None), dict(gate=None)):
        assert L.d1_scan_fwd(C.byref(scan(**k)), F, 64, 0, F, F, need, None) == -1
    assert L.d1_scan_fwd(C.byref(good), None, 64, 0, F, F, need, None) == -1
    assert L.d1_scan_fwd(C.byref(good), F, 64, 0, F, None, need, None) == -1
    assert L.d1_scan_fwd(C.byref(good), F, 64, 0, F, F, need - 1, None) == -1
    assert L.d1_scan_fwd(None, F, 64, 0, F, F, need, None) == -1
    back = [F, 64, 0, None, F, 64, 0, F, 64, 0, None, F, need, None]
    assert L.d1_scan_bwd(C.byref(good), *back) == -1              # no marks
    marked = scan(marks=F)
    for at, value in ((0, None), (4, None), (7, None), (11, None), (12, 7)):
        args = list(back)
        args[at] = value
        assert L.d1_scan_bwd(C.byref(marked), *args) == -1, at
    for k in (dict(steps=0), dict(rows=0), dict(width=0)):
        assert L.d1_scan_fwd(C.byref(scan(**k)), None, 0, 0, None, None, 0, None) == 0


def test_muon_arguments(lib):
    L = lib.load_ops()

    def settings(**k):
        return lib.D1Muon(**dict(dict(a=3.4445, b=-4.775, c=2.0315, eps=1e-7, steps=5), **k))

    def matrix(**k):
        return (lib.D1MuonTensor * 1)(lib.D1MuonTensor(**dict(dict(g=F, out=F, rows=100, cols=300), **k)))
    h = settings()
    assert L.d1_muon_check(C.byref(h)) == 0 and L.d1_muon_check(C.byref(settings(a=1.5, b=-0.5, c=0.0, steps=32))) == 0
    for k in (dict(steps=0), dict(steps=33), dict(eps=-1.0), dict(momentum=1.0), dict(terms=2), dict(a=20.0), dict(a=float('nan')),
              dict(a=3.0, b=-3.0, c=5.0)):
        assert L.d1_muon_check(C.byref(settings(**k))) == -1, k
    need = L.d1_muon_work_bytes(matrix(), 1, C.byref(h))
    assert need > 0 and L.d1_muon_work_bytes(matrix(type=1), 1, C.byref(h)) < need
    for k in (dict(rows=-1), dict(cols=1 << 18), dict(g=None), dict(out=None), dict(type=5), dict(gtype=-1), dict(lr=float('nan')),
              dict(momentum=F, type=2), dict(copy=F)):
        assert L.d1_muon_work_bytes(matrix(**k), 1, C.byref(h)) == -1, k
        assert L.d1_muon_step(matrix(**k), 1, C.byref(h), None, F, 1 << 40, None) == -1, k
    for args in ((None, need), (F, need - 1), (F + 8, need)):
        assert L.d1_muon_step(matrix(), 1, C.byref(h), None, *args, None) == -1
    assert L.d1_muon_step(matrix(), 1, C.byref(h), 3, F, need, None) == -1
    assert L.d1_muon_step(matrix(), -1, C.byref(h), None, F, need, None) == -1 and L.d1_muon_step(None, 1, C.byref(h), None, F, need, None) == -1
