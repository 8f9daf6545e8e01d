"""adamw_step and AdamW (csrc/d1_optim.hip): 32-bit moments and parameters against the definition in
64 bits (u = 2^-24: a moment is two products and a sum, 3 u of its terms; the step lr m/den adds about
12 u of itself, the parameter 2 u), 8-bit moments bit for bit against a numpy restatement, the clip,
the skip of a step that is not finite, many tensors, steps that tensors miss, graphs, checkpoints."""
import copy
import importlib
import math

import numpy as np
import pytest
import torch

import adamw_ref as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
LR, B1, B2, EPS, WD = 3e-3, 0.9, 0.999, 1e-6, 0.05


@pytest.fixture(scope='module')
def A():
    return importlib.import_module('dcss-auto_amd.optim')


def tensors(sizes, seed, pdtype=torch.float32, gdtype=torch.float32):
    g = torch.Generator(device='cuda').manual_seed(seed)
    rand = lambda n, s: torch.randn(n, generator=g, device='cuda') * s  # noqa: E731
    return ([rand(n, 0.5).to(pdtype) for n in sizes], [rand(n, 1e-2).to(gdtype) for n in sizes],
            [rand(n, 1e-3) for n in sizes], [rand(n, 1e-2).square() for n in sizes])


def formula(p, g, m, v, t, coef=1.0):
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * coef
    m1, v1 = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    step = LR / (1 - B1 ** t) * m1 / (torch.sqrt(v1 / (1 - B2 ** t)) + EPS)
    return p * (1 - LR * WD) - step, m1, v1, step


def clip_of(grads, most):
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    return min(1.0, most / (norm + 1e-6)), norm


def compare(got, before, t, coef=1.0):
    for (p, m, v), (p0, g0, m0, v0) in zip(got, before):
        if not p.numel():
            continue
        wp, wm, wv, step = formula(p0, g0, m0, v0, t, coef)
        gc = g0.double() * coef
        assert float(((m.double() - wm).abs() - 4 * U * ((B1 * m0.double()).abs() + ((1 - B1) * gc).abs()) - 1e-44).max()) <= 0
        assert float(((v.double() - wv).abs() - 6 * U * wv - 1e-44).max()) <= 0
        # what m's own rounding moves in the step: m may be a difference of its terms
        loose = 4 * U * ((B1 * m0.double()).abs() + gc.abs()) / (wm.abs() + 1e-300) * step.abs()
        tol = 2 * U * wp.abs() + 2 * U * p0.double().abs() + 16 * U * step.abs() + loose
        if p.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * wp.abs()
        assert float(((p.double() - wp).abs() - tol).max()) <= 0


SIZES = [[1], [3], [255], [256], [257], [4095], [4096], [4097], [5, 0, 1023, 70000, 1, 16, 12289],
         [17 * k + 1 for k in range(97)]]


@pytest.mark.parametrize('clip', [0.0, 0.05])
@pytest.mark.parametrize('pdtype,gdtype', [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                           (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)],
                         ids=['f32', 'f32-b16', 'b16', 'b16-f32'])
@pytest.mark.parametrize('sizes', SIZES, ids=[f'{len(s)}x{max(s)}' for s in SIZES])
def test_32_bit(A, sizes, pdtype, gdtype, clip):
    print(f'[adamw] {len(sizes)} tensors up to {max(sizes)} {pdtype} {gdtype} clip {clip}', flush=True)
    p, g, m, v = tensors(sizes, len(sizes) + max(sizes), pdtype, gdtype)
    copies = [torch.zeros(n, dtype=torch.bfloat16, device='cuda') for n in sizes] if pdtype == torch.float32 else None
    step = torch.zeros(8, dtype=torch.int32, device='cuda')
    for t in (1, 2, 3):
        before = [tuple(x.clone() for x in z) for z in zip(p, g, m, v)]
        A.adamw_step(p, g, m, v, step, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, max_grad_norm=clip, copies=copies)
        coef, norm = clip_of(g, clip) if clip else (1.0, 0.0)
        compare(list(zip(p, m, v)), before, t, coef)
        assert int(step[0]) == t and int(step[1]) == 0
        if clip:
            assert abs(float(step[5:6].view(torch.float32)) - norm) <= 2 * U * norm
        if copies:
            assert all(torch.equal(c, x.to(torch.bfloat16)) for c, x in zip(copies, p))


# partial sums of the norm up to where the step's workgroups add them (1,024 of 1,024 elements) and past it, one and
# several launches of up to 40 tensors, and the long chunks from 4 M elements on
@pytest.mark.parametrize('sizes', [[1 << 20], [(1 << 20) + 1], [26000] * 40, [26000] * 41, [4194303], [4194304, 9]],
                         ids=lambda s: f'{len(s)}x{max(s)}')
def test_clip_over_many_elements(A, sizes):
    print(f'[adamw] clip {len(sizes)} tensors up to {max(sizes)}', flush=True)
    p, g, m, v = tensors(sizes, len(sizes))
    step = torch.zeros(8, dtype=torch.int32, device='cuda')
    call = lambda: A.adamw_step(p, g, m, v, step, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, max_grad_norm=0.5)  # noqa: E731
    for t in (1, 2):
        before = [tuple(x.clone() for x in z) for z in zip(p, g, m, v)]
        call()
        coef, norm = clip_of(g, 0.5)
        compare(list(zip(p, m, v)), before, t, coef)
        assert step[:2].tolist() == [t, 0] and abs(float(step[5:6].view(torch.float32)) - norm) <= 2 * U * norm
    kept = [x.clone() for x in (*p, *m, *v)]
    g[-1][-1] = math.inf
    call()
    assert all(torch.equal(a, b) for a, b in zip(kept, (*p, *m, *v))) and step[:2].tolist() == [2, 1]


def eight(A, sizes):
    zeros = lambda n: torch.zeros(n, dtype=torch.uint8, device='cuda')  # noqa: E731
    return ([zeros(n) for n in sizes], [zeros(n) for n in sizes],
            ([zeros(A.moment_blocks(n)) for n in sizes], [zeros(A.moment_blocks(n)) for n in sizes]))


@pytest.mark.parametrize('sizes', [[1], [255, 256, 257], [4099, 7, 0, 513], [40000]], ids=str)
@pytest.mark.parametrize('gdtype', [torch.float32, torch.bfloat16], ids=['f32', 'b16'])
def test_8_bit_codes(A, sizes, gdtype):
    """Codes and exponents of several steps bit for bit, parameters from the unrounded moments."""
    print(f'[adamw] 8 bits {sizes} {gdtype}', flush=True)
    p, g, _, _ = tensors(sizes, 4, torch.float32, gdtype)
    for k, x in enumerate(g):                        # magnitudes from denormal to large, zeros, whole zero blocks
        if x.numel() > 200:
            x[::7] *= 1e-6
            x[1::11] *= 1e-18
            x[2::13] = 0
            x[3::17] *= 1e3
        if x.numel() > 600:
            x[256:512] = 0
    codes_m, codes_v, exps = eight(A, sizes)
    step = torch.zeros(8, dtype=torch.int32, device='cuda')
    counters = [(5 << 32) - 100 + 100000 * k for k in range(len(sizes))]       # draws whose counters pass 2^32
    seed = 0x123456789ABCDEF0
    for t in range(1, 5):
        host = [(x.cpu().numpy(), y.float().cpu().numpy(), a.cpu().numpy(), b.cpu().numpy(), ea.cpu().numpy(), eb.cpu().numpy())
                for x, y, a, b, ea, eb in zip(p, g, codes_m, codes_v, *exps)]
        A.adamw_step(p, g, codes_m, codes_v, step, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, exps=exps,
                     counters=counters, seed=seed)
        for k, (p0, g0, cm, cv, em, ev) in enumerate(host):
            n = len(p0)
            if not n:
                continue
            m0, v0 = R.decode(cm, em, 15), R.decode(cv, ev, 31)
            m1, v1 = R.moments(m0, v0, g0, 1.0)
            word = R.draws(seed, t, counters[k] + np.arange(n))
            wm, we = R.encode(m1, 15, word >> np.uint64(16))
            assert np.array_equal(codes_m[k].cpu().numpy(), wm) and np.array_equal(exps[0][k].cpu().numpy(), we)
            wv, we = R.encode(v1, 31, word & np.uint64(0xFFFF))
            assert np.array_equal(codes_v[k].cpu().numpy(), wv) and np.array_equal(exps[1][k].cpu().numpy(), we)
            read = A.read_moment(codes_m[k], exps[0][k], signed=True).cpu().numpy()
            assert np.array_equal(read, R.decode(wm, exps[0][k].cpu().numpy(), 15))
            read = A.read_moment(codes_v[k], exps[1][k], signed=False).cpu().numpy()
            assert np.array_equal(read, R.decode(wv, exps[1][k].cpu().numpy(), 31))
            assert not ((read == 0) & (v1 > 0)).any()
            want = formula(*(torch.from_numpy(x) for x in (p0, g0, m0, v0)), t)
            off = np.abs(p[k].cpu().numpy().astype(np.float64) - want[0].numpy())
            tol = 4 * U * np.abs(p0) + 16 * U * want[3].abs().numpy() + 4 * U * (np.abs(0.9 * m0) + np.abs(g0)) / (
                np.abs(want[1].numpy()) + 1e-300) * want[3].abs().numpy()
            assert (off <= tol).all()


def test_8_bit_rounding_follows_the_mean(A):
    """v moves by (1 - b2)(g^2 - v) a step, less than its code's resolution: rounding by chance
    still takes it to g^2. 65,536 elements, each rounding off by up to an eighth of v, independent:
    after the steps v's mean is within 1% of the 32-bit run's (a standard error under 0.1%)."""
    print('[adamw] 8 bits mean', flush=True)
    n, steps = 65536, 400
    g = [torch.full((n,), 0.1, device='cuda')]
    p8, p32 = [torch.zeros(n, device='cuda')], [torch.zeros(n, device='cuda')]
    m8, v8, exps = eight(A, [n])
    m32, v32 = [torch.zeros(n, device='cuda')], [torch.zeros(n, device='cuda')]
    s8, s32 = (torch.zeros(8, dtype=torch.int32, device='cuda') for _ in range(2))
    for k in range(steps):
        g[0].fill_(0.1 if k < 100 else 0.3)
        g[0][::256] = 1.0                          # each block's largest element: the others sit lower in the range
        A.adamw_step(p8, g, m8, v8, s8, lr=LR, exps=exps, counters=[0], seed=5)
        A.adamw_step(p32, g, m32, v32, s32, lr=LR)
    rest = torch.arange(n, device='cuda') % 256 != 0
    for code, e, want, signed in ((m8[0], exps[0][0], m32[0], True), (v8[0], exps[1][0], v32[0], False)):
        got = A.read_moment(code, e, signed=signed)
        assert abs(float(got[rest].double().mean() / want[rest].double().mean()) - 1) < 0.01
    assert abs(float(p8[0].double().mean() / p32[0].double().mean()) - 1) < 0.02


@pytest.mark.parametrize('bits', [32, 8])
def test_not_finite(A, bits):
    print(f'[adamw] not finite {bits}', flush=True)
    sizes = [300, 5000]
    for bad in (math.nan, math.inf):
        p, g, m, v = tensors(sizes, 3)
        exps = None
        if bits == 8:
            m, v, exps = eight(A, sizes)
        step = torch.zeros(8, dtype=torch.int32, device='cuda')
        call = lambda clip: A.adamw_step(p, g, m, v, step, lr=LR, max_grad_norm=clip, exps=exps)  # noqa: E731
        call(1.0)
        kept = [x.clone() for x in (*p, *m, *v)]
        g[1][4321] = bad
        call(1.0)
        call(1.0)
        assert all(torch.equal(a, b) for a, b in zip(kept, (*p, *m, *v))) and step[:2].tolist() == [1, 2]
        g[1][4321] = 0.5
        call(1.0)
        assert step[:2].tolist() == [2, 2] and not torch.equal(kept[1], p[1])
        g[1][4321] = bad
        call(0.0)                                  # without a clip nothing is looked at
        assert step[:2].tolist() == [3, 2]
        assert not math.isfinite(float(p[1][4321])) and int((~torch.isfinite(p[1])).sum()) == 1 and torch.isfinite(p[0]).all()


def test_offsets_past_32_bits(A):
    """A tensor of more than 2^32 elements: its last ones, in both kinds of moments."""
    print('[adamw] offsets', flush=True)
    n, tail = 2 ** 32 + 1031, 2000
    p, g = torch.zeros(n, dtype=torch.bfloat16, device='cuda'), torch.zeros(n, dtype=torch.bfloat16, device='cuda')
    last, lastg, m0, v0 = (x[0] for x in tensors([tail], 12, torch.bfloat16, torch.bfloat16))
    zero = torch.zeros_like(m0)
    for bits in (32, 8):
        p[-tail:], g[-tail:] = last, lastg
        dtype = torch.uint8 if bits == 8 else torch.float32
        m, v = torch.zeros(n, dtype=dtype, device='cuda'), torch.zeros(n, dtype=dtype, device='cuda')
        exps = tuple([torch.zeros(A.moment_blocks(n), dtype=torch.uint8, device='cuda')] for _ in range(2)) if bits == 8 else None
        step = torch.zeros(8, dtype=torch.int32, device='cuda')
        A.adamw_step([p], [g], [m], [v], step, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, max_grad_norm=0.05, exps=exps)
        coef, norm = clip_of([lastg], 0.05)
        assert abs(float(step[5:6].view(torch.float32)) - norm) <= 2 * U * norm
        if bits == 32:
            compare([(p[-tail:], m[-tail:], v[-tail:])], [(last, lastg, zero, zero)], 1, coef)
        else:
            q = [x.clone() for x in (last, lastg)]
            one = A.adamw_step
            state = eight(A, [tail])
            twin = torch.zeros(8, dtype=torch.int32, device='cuda')
            one([q[0]], [q[1]], state[0], state[1], twin, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, max_grad_norm=0.05, exps=state[2])
            assert torch.equal(p[-tail:], q[0])          # the step is made before moments are rounded
            read = A.read_moment(m, exps[0][0], signed=True)
            wide = formula(last, lastg, zero, zero, 1, coef)[1]
            block = wide.abs().max()
            assert float(((read[-tail:].double() - wide).abs() - wide.abs() / 8 - block * 2.0 ** -16).max()) <= 0
            del read
        assert not bool(p[:tail].any()) and not bool(m[:tail].any())
        del m, v, exps
    del p, g
    torch.cuda.empty_cache()


def test_strides_and_streams(A):
    print('[adamw] strides', flush=True)
    flat = torch.randn(5000, device='cuda')
    flat2 = flat.clone()
    p = [flat[1:1000], flat[1003:4000]]            # unaligned views
    g = [torch.randn(999, device='cuda'), torch.randn(37, 81, device='cuda').t().expand(81, 37)]
    m, v = [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p]
    step = torch.zeros(8, dtype=torch.int32, device='cuda')
    A.adamw_step(p, g, m, v, step, lr=LR)
    q = [flat2[1:1000].clone(), flat2[1003:4000].clone()]
    m2, v2 = [torch.zeros_like(x) for x in q], [torch.zeros_like(x) for x in q]
    step2 = torch.zeros(8, dtype=torch.int32, device='cuda')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        A.adamw_step(q, [g[0].clone(), g[1].contiguous()], m2, v2, step2, lr=LR)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*p, *m, *v), (*q, *m2, *v2)))
    untouched = [0, 1000, 1001, 1002, *range(4000, 5000)]
    assert torch.equal(flat[untouched], flat2[untouched])


@pytest.mark.parametrize('bits', [32, 8])
def test_optimizer(A, bits):
    """Groups with their own lr and decay, a parameter that misses steps, one that never has a
    gradient; a saved state continues bit for bit."""
    print(f'[adamw] optimizer {bits}', flush=True)

    def make(seed):
        gen = torch.Generator(device='cuda').manual_seed(seed)
        ps = [torch.nn.Parameter(torch.randn(n, generator=gen, device='cuda')) for n in ((40, 30), (7,), (300,), (5,))]
        copies = {ps[0]: torch.zeros(40, 30, dtype=torch.bfloat16, device='cuda')}
        opt = A.AdamW([dict(params=ps[:2], lr=LR, weight_decay=WD), dict(params=ps[2:])], lr=1e-2, weight_decay=0.0,
                      betas=(B1, B2), eps=EPS, state_bits=bits, max_grad_norm=0.5, copies=copies, seed=9)
        return ps, opt, copies

    def grads(ps, t):
        gen = torch.Generator(device='cuda').manual_seed(100 + t)
        for k, p in enumerate(ps):
            p.grad = torch.randn(p.shape, generator=gen, device='cuda') * 0.1
        ps[3].grad = None
        if t in (0, 3):
            ps[1].grad = None

    ps, opt, copies = make(1)
    if bits == 32:
        ref = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        plain = torch.optim.AdamW([dict(params=ref[:2], lr=LR, weight_decay=WD), dict(params=ref[2:], lr=1e-2, weight_decay=0.0)],
                                  betas=(B1, B2), eps=EPS)
    start = ps[3].detach().clone()
    saved = None
    for t in range(8):
        grads(ps, t)
        opt.step()
        if bits == 32:
            grads(ref, t)
            norm = torch.nn.utils.clip_grad_norm_([p for p in ref if p.grad is not None], 0.5)
            plain.step()
            torch.testing.assert_close(opt.grad_norm(), norm, rtol=1e-6, atol=0)
            for a, b in zip(ps, ref):
                torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)
        if t == 4:
            saved = (opt.state_dict(), [p.detach().clone() for p in ps])
            saved[0]['state'] = {k: {n: x.clone() if torch.is_tensor(x) else x for n, x in s.items()} for k, s in saved[0]['state'].items()}
    assert torch.equal(ps[3], start) and torch.equal(copies[ps[0]], ps[0].to(torch.bfloat16))
    assert opt.skipped_steps() == 0 and opt.state[ps[1]]['lag'] == 2
    qs, again, _ = make(2)
    with torch.no_grad():
        for q, p in zip(qs, saved[1]):
            q.copy_(p)
    again.load_state_dict(saved[0])
    for t in range(5, 8):
        grads(qs, t)
        again.step()
    assert all(torch.equal(a, b) for a, b in zip(ps, qs))
    for a, b in zip(ps[:3], qs[:3]):
        assert all(torch.equal(x, y) for x, y in zip(opt.moments(a), again.moments(b)))
    with pytest.raises(ValueError):
        A.AdamW(qs, state_bits=40 - bits).load_state_dict(saved[0])


def test_own_step_counts(A):
    """A parameter's count holds the steps that were made with it alone: not those it missed, nor
    those skipped while it was there or away, and it follows steps replayed from a graph."""
    print('[adamw] own step counts', flush=True)
    gen = torch.Generator(device='cuda').manual_seed(8)
    ps = [torch.nn.Parameter(torch.randn(n, generator=gen, device='cuda')) for n in (50, 70, 90)]
    ref = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt = A.AdamW(ps, lr=LR, weight_decay=WD, betas=(B1, B2), eps=EPS, max_grad_norm=1e9)
    plain = torch.optim.AdamW(ref, lr=LR, weight_decay=WD, betas=(B1, B2), eps=EPS)
    # parameters with a gradient, and whether the step's gradients are finite
    plan = [('a', True), ('ab', False), ('ab', True), ('a', False), ('a', True), ('a', False), ('abc', True), ('bc', False), ('abc', True)]

    def step(who, finite):
        for k, (p, q) in enumerate(zip(ps, ref)):
            here = 'abc'[k] in who
            p.grad = torch.randn(p.shape, generator=gen, device='cuda') if here else None
            q.grad = p.grad.clone() if here else None
        if not finite:
            ps['abc'.index(who[0])].grad[3] = math.inf
        opt.step()
        if finite:
            plain.step()

    for t, (who, finite) in enumerate(plan):
        step(who, finite)
        for a, b in zip(ps, ref):
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)
        if t == 5:
            opt = copy.deepcopy(opt)             # a copy has parameters of its own: go on with those
            ps = opt.param_groups[0]['params']
    assert opt.ctl[:2].tolist() == [5, 4] and [opt.state[p]['lag'] for p in ps] == [0, 2, 3]
    ps[1].grad = ps[2].grad = ref[1].grad = ref[2].grad = None
    opt.step()
    plain.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
        plain.step()
    step('abc', True)
    for a, b in zip(ps, ref):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)
    assert int(opt.ctl[0]) == 10 and [opt.state[p]['lag'] for p in ps] == [0, 6, 7]


def test_capture_needs_a_step_before(A, monkeypatch):
    """Moments made, or a count taken, inside a capture would be made again at each replay."""
    print('[adamw] before a capture', flush=True)
    ps = [torch.nn.Parameter(torch.ones(5, device='cuda')) for _ in range(2)]
    opt = A.AdamW(ps, lr=LR)
    with pytest.raises(ValueError):
        opt.moments(ps[0])

    def step(first, second, captured):
        for p, here in zip(ps, (first, second)):
            p.grad = torch.ones(5, device='cuda') if here else None
        with monkeypatch.context() as patch:
            patch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: captured)
            opt.step()

    with pytest.raises(RuntimeError):
        step(True, False, True)
    opt = A.AdamW(ps, lr=LR)
    step(True, True, False)
    step(True, True, True)
    with pytest.raises(RuntimeError):
        step(True, False, True)
    step(True, False, False)
    step(True, False, True)
    with pytest.raises(RuntimeError):
        step(True, True, True)
    step(True, True, False)
    assert int(opt.ctl[0]) == 5 and [opt.state[p]['lag'] for p in ps] == [0, 2]


@pytest.mark.parametrize('bits', [32, 8])
def test_graph_replays(A, bits):
    """The step count advances on the device: each replay is the next step."""
    print(f'[adamw] graph {bits}', flush=True)
    sizes = [1000, 77, 9000]
    p, g, m, v = tensors(sizes, 6)
    exps = None
    if bits == 8:
        m, v, exps = eight(A, sizes)
    step = torch.zeros(8, dtype=torch.int32, device='cuda')
    twin = [[x.clone() for x in z] for z in (p, m, v)]
    texps = None if exps is None else tuple([x.clone() for x in z] for z in exps)
    tstep = step.clone()
    args = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, max_grad_norm=0.5, counters=[0, 1024, 1280], seed=3)
    A.adamw_step(p, g, m, v, step, exps=exps, **args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.adamw_step(p, g, m, v, step, exps=exps, **args)
    A.adamw_step(twin[0], g, twin[1], twin[2], tstep, exps=texps, **args)
    for k in range(4):
        g[2].mul_(1.5)
        graph.replay()
        A.adamw_step(twin[0], g, twin[1], twin[2], tstep, exps=texps, **args)
        assert all(torch.equal(a, b) for z, w in zip((p, m, v), twin) for a, b in zip(z, w))
        assert int(step[0]) == k + 2
        torch.cuda.synchronize()


def test_refusals(A):
    print('[adamw] refusals', flush=True)
    step = torch.zeros(8, dtype=torch.int32, device='cuda')

    def call(change=None, **more):
        p, g, m, v = tensors([10, 20], 1)
        lists = dict(p=p, g=g, m=m, v=v)
        if change:
            name, k, value = change
            lists[name][k] = value(lists[name][k])
        A.adamw_step(lists['p'], lists['g'], lists['m'], lists['v'], more.pop('step', step), **more)

    call()
    for change in (('p', 0, lambda x: x.double()), ('p', 1, lambda x: x.half()), ('g', 0, lambda x: x.half()),
                   ('g', 0, lambda x: x[:9]), ('m', 1, lambda x: x[:19]), ('v', 1, lambda x: x.bfloat16()),
                   ('p', 0, lambda x: torch.zeros(20, device='cuda')[::2]), ('m', 0, lambda x: torch.zeros(20, device='cuda')[::2]),
                   ('g', 0, lambda x: x.cpu()), ('p', 0, lambda x: x.cpu())):
        with pytest.raises(ValueError):
            call(change)
    for more in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(lr=-1.0), dict(weight_decay=[0.1, -0.1]),
                 dict(lr=[1.0]), dict(max_grad_norm=-1.0), dict(max_grad_norm=math.nan), dict(step=step[:7]),
                 dict(step=step.float()), dict(step=step.cpu()), dict(copies=[None]), dict(counters=[0]), dict(lags=[0]),
                 dict(copies=[torch.zeros(10, device='cuda'), None]),
                 dict(exps=([step], [step]))):
        with pytest.raises(ValueError):
            call(**more)
    assert int(step[0]) == 1
    with pytest.raises(ValueError):
        A.AdamW([torch.nn.Parameter(torch.zeros(3, device='cuda'))], state_bits=16)
    with pytest.raises(ValueError):
        A.read_moment(torch.zeros(300, dtype=torch.uint8, device='cuda'), torch.zeros(1, dtype=torch.uint8, device='cuda'), True)
