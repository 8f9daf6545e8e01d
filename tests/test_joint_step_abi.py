"""libd1ops.so: a step in two parts and one made together with it, rejected arguments (no GPU needed: rejected calls never launch)."""
import ctypes as C
import importlib

F = 1 << 20            # a made-up device address: rejected calls never read it


def test_arguments():
    lib = importlib.import_module('dcss-auto_amd._lib')
    L = lib.load_ops()
    settings = lambda part: lib.D1Muon(a=3.4445, b=-4.775, c=2.0315, eps=1e-7, steps=5, part=part)  # noqa: E731
    t = (lib.D1MuonTensor * 1)(lib.D1MuonTensor(g=F, momentum=F, out=F, rows=100, cols=300))
    need = [L.d1_muon_work_bytes(t, 1, C.byref(settings(part))) for part in (0, 1, 2)]
    assert need[0] > 0 and need == need[:1] * 3               # one buffer for both parts
    for part in (1, 2):                                       # without the counts there is nothing to decide by
        assert L.d1_muon_step(t, 1, C.byref(settings(part)), None, F, need[0], None) == -1
    for part in (-1, 3):
        assert L.d1_muon_check(C.byref(settings(part))) == -1 and L.d1_muon_work_bytes(t, 1, C.byref(settings(part))) == -1
        assert L.d1_muon_step(t, 1, C.byref(settings(part)), F, F, need[0], None) == -1
    a = (lib.D1AdamWTensor * 1)(lib.D1AdamWTensor(p=F, g=F, m=F, v=F, n=100))
    h = lib.D1AdamW(beta1=0.9, beta2=0.999, eps=1e-8, bits=32)
    for ctl, other in ((None, F), (F, F), (F, F + 1026)):
        assert L.d1_adamw_step_with(a, 1, C.byref(h), ctl, other, None, 0, None) == -1
