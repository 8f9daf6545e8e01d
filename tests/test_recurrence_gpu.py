"""gated_scan against its definition step by step in 64 bits, with bounds that follow every rounding along the
sequence; lengths from nothing to segments, resets, strides, refusals, streams and graphs."""
import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'
U = 2.0 ** -24
TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
# A step's roundings: z and a 4 halves of a step each (exponential with its correction, sum, reciprocal, product), a
# multiply-add 1, the products of composites 2 a step; what it adds has the size of what is added
STEP = 12


@pytest.fixture(scope='module')
def R():
    return importlib.import_module('dcss-auto_amd.recurrence')


def data(steps, rows, width, dtype=torch.float32, seed=0, state=True, reset=0.05, slow=5.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    return dict(x=normal(steps, rows, width).to(dtype), gate=(normal(steps, rows, width) - slow * torch.rand(width, generator=g, device=DEV)).to(dtype),
                state=normal(rows, width) if state else None,
                reset=torch.rand(steps, rows, generator=g, device=DEV) < reset if reset else None), \
        dict(dh=normal(steps, rows, width).to(dtype), dlast=normal(rows, width))


def definition(x, gate, state, reset, dh=None, dlast=None):
    """-> {name: (value, bound on the kernels' error before its last rounding)} in 64 bits."""
    x, gate = x.double(), gate.double()
    steps, rows, width = x.shape
    z, a = torch.sigmoid(gate), torch.sigmoid(-gate)
    m = torch.ones(steps, rows, 1, dtype=torch.float64, device=DEV) if reset is None else (~reset.bool()).double()[:, :, None]
    a = torch.where(m > 0, a, 0.0)
    h = torch.zeros(rows, width, dtype=torch.float64, device=DEV) if state is None else state.double()
    size, err = h.abs(), torch.zeros_like(h)
    hs, before, bsize, berr, errs = [], [], [], [], []
    for t in range(steps):
        keep = m[t] > 0
        before.append(torch.where(keep, h, 0.0))
        bsize.append(torch.where(keep, size, 0.0))
        berr.append(torch.where(keep, err, 0.0))
        h, size = torch.where(keep, a[t] * h, 0.0) + z[t] * x[t], torch.where(keep, a[t] * size, 0.0) + z[t] * x[t].abs()
        err = torch.where(keep, a[t] * err, 0.0) + STEP * U * size
        hs.append(h)
        errs.append(err)
    stack = lambda v: torch.stack(v) if v else torch.zeros_like(x)  # noqa: E731
    out = dict(h=(stack(hs), stack(errs)), last=(h, err))
    if dh is None:
        return out
    zero = torch.zeros(rows, width, dtype=torch.float64, device=DEV)
    c = zero if dlast is None else dlast.double()
    csize, cerr = c.abs(), zero
    slope = torch.sigmoid(gate) * torch.sigmoid(-gate)
    dx, dxe, dg, dge = [], [], [], []
    for t in reversed(range(steps)):
        gr, gs = dh[t].double() + c, dh[t].double().abs() + csize
        ge = cerr + 2 * U * gs
        dx.append(z[t] * gr)
        dxe.append(z[t] * (ge + STEP * U * gs))
        span = x[t].abs() + bsize[t]
        dg.append(gr * (x[t] - before[t]) * slope[t])
        dge.append(slope[t] * (ge * span + gs * berr[t] + STEP * U * gs * span))
        c, csize, cerr = a[t] * gr, a[t] * gs, a[t] * ge + STEP * U * a[t] * gs
    out['dx'], out['dgate'] = [(stack(v[::-1]), stack(e[::-1])) for v, e in ((dx, dxe), (dg, dge))]
    out['dstate'] = (c, cerr)
    return out


def check(got, want, name):
    value, bound = want
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    bound = bound + torch.finfo(got.dtype).eps / 2 * (value.abs() + bound) + tiny
    off = (got.double() - value).abs()
    bad = ~(off <= bound) & ~(off.isnan() & value.isnan())
    assert not bool(bad.any()), (name, int(bad.sum()), float((off - bound)[bad].max()))


def run(R, k, g):
    h, last, marks = R.gated_scan_fwd(**k)
    dx, dgate, dstate = R.gated_scan_bwd(g['dh'], g['dlast'], **k, marks=marks)
    return dict(h=h, last=last, dx=dx, dgate=dgate, dstate=dstate)


def compare(R, k, g):
    got, want = run(R, k, g), definition(**k, **g)
    for name in want:
        if name == 'dstate' and k['state'] is None:
            assert got[name] is None
            continue
        assert got[name].dtype == (torch.float32 if name in ('last', 'dstate') else k['x'].dtype)
        check(got[name], want[name], name)
    return got


@pytest.mark.parametrize('steps', [1, 2, 7, 8, 9, 33, 63, 64, 65, 127, 129, 200])
@pytest.mark.parametrize('rows,width', [(3, 1), (1, 64), (2, 65), (3, 97), (2, 191), (5, 200), (1, 257), (2, 1001)])
def test_sizes(R, steps, rows, width):
    print(f'[scan] {steps} {rows} {width}', flush=True)
    compare(R, *data(steps, rows, width, seed=steps + width))


@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('state', [False, True])
@pytest.mark.parametrize('reset', [0, 0.02, 0.7, 1.0])
def test_types_states_resets(R, dtype, state, reset):
    print(f'[scan] {dtype} {state} {reset}', flush=True)
    for steps, rows, width in ((1, 4, 130), (50, 3, 66), (150, 2, 260)):
        compare(R, *data(steps, rows, width, TYPES[dtype], 3, state, reset))


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
@pytest.mark.parametrize('steps,rows,width', [(257, 1, 8), (1000, 1, 64), (1500, 2, 300), (4096, 1, 130), (2049, 37, 33)])
def test_segments(R, steps, rows, width, dtype):
    """Sequences that are cut, with memories longer than a segment."""
    print(f'[scan] segments {steps} {rows} {width} {dtype}', flush=True)
    for reset in (0, 0.001):
        compare(R, *data(steps, rows, width, TYPES[dtype], steps, True, reset, slow=9.0))


def test_strides(R):
    """Batch-first sequences, rows apart from each other, channels that are not adjacent, broadcast gates and gradients."""
    print('[scan] strides', flush=True)
    k, g = data(90, 6, 70, seed=5)
    want = run(R, k, g)
    first = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    wide = torch.zeros(90, 6, 150, device=DEV)
    wide[..., 5:75] = k['gate']
    s = dict(k, x=first(k['x']), gate=wide[..., 5:75], reset=first(k['reset']), state=k['state'].t().contiguous().t())
    got = run(R, s, dict(dh=first(g['dh']), dlast=g['dlast']))
    for name in want:
        assert torch.equal(got[name], want[name]), name
    assert got['h'].stride() == s['x'].stride() and got['dx'].stride() == s['x'].stride()
    s = dict(k, x=k['x'].permute(2, 0, 1).contiguous().permute(1, 2, 0))
    assert torch.equal(run(R, s, g)['dgate'], want['dgate'])
    same = dict(k, x=k['x'][:, :1].expand(90, 6, 70))
    copied = dict(k, x=same['x'].contiguous())
    a, b = run(R, same, dict(g, dh=torch.ones((), device=DEV).expand(90, 6, 70))), run(R, copied, dict(g, dh=torch.ones(90, 6, 70, device=DEV)))
    for name in a:
        assert torch.equal(a[name], b[name]), name


def test_two_dimensions_and_steps(R):
    """[steps, width] is a row of its own; a sequence in pieces or step by step is the whole."""
    k, g = data(130, 1, 70, seed=6)
    flat = {n: (t[:, 0] if n in ('x', 'gate', 'reset') else t[0]) for n, t in k.items()}
    want, got = run(R, k, g), run(R, flat, dict(dh=g['dh'][:, 0], dlast=g['dlast'][0]))
    assert torch.equal(got['h'], want['h'][:, 0]) and torch.equal(got['dstate'], want['dstate'][0]) and got['last'].shape == (70,)
    state, out = k['state'], []
    for t in range(130):
        h, state = R.gated_scan(k['x'][t:t + 1], k['gate'][t:t + 1], state, k['reset'][t:t + 1])
        out.append(h)
    whole = definition(**k)
    check(torch.cat(out), whole['h'], 'steps')
    check(state, whole['last'], 'steps')
    assert torch.equal(out[-1][0], state)


def test_a_reset_drops_anything(R):
    """Infinite and NaN states and inputs before a reset leave nothing behind it, within and across segments and waves."""
    print('[scan] not finite', flush=True)
    for steps, at in ((3, 1), (40, 17), (300, 200), (3000, 2500)):
        k, g = data(steps, 2, 70, seed=steps, reset=0)
        k['reset'] = torch.zeros(steps, 2, dtype=torch.bool, device=DEV)
        k['reset'][at, 0] = True
        clean = run(R, k, g)
        k['state'][0] = math.nan
        k['x'][at - 1, 0, :35] = math.inf
        k['gate'][at - 1, 0, 35:] = math.nan
        got = run(R, k, g)
        assert torch.equal(got['h'][at:, 0], clean['h'][at:, 0]) and torch.equal(got['h'][:, 1], clean['h'][:, 1])
        assert torch.equal(got['last'], clean['last']) and torch.equal(got['dx'][at:], clean['dx'][at:])
        assert torch.equal(got['dgate'][at:], clean['dgate'][at:]) and bool(got['h'][:at, 0].isnan().any())


def test_extreme_gates(R):
    """Gates at the ends of their range: the state is kept or replaced exactly."""
    x = torch.randn(20, 1, 64, device=DEV)
    state = torch.randn(1, 64, device=DEV)
    for value, want in ((-math.inf, state.expand(20, 1, 64)), (math.inf, x), (-1e30, state.expand(20, 1, 64)), (200.0, x)):
        h, last = R.gated_scan(x, torch.full_like(x, value), state)
        assert torch.equal(h, want) and torch.equal(last, want[-1])
    for dtype in TYPES.values():
        k, g = data(30, 2, 70, dtype, 7, slow=40.0)
        compare(R, k, g)


@pytest.mark.parametrize('shape', [(0, 3, 5), (4, 0, 5), (4, 3, 0), (0, 5)])
def test_nothing(R, shape):
    x = torch.zeros(shape, device=DEV)
    state = torch.randn(shape[1:], device=DEV)
    h, last, marks = R.gated_scan_fwd(x, x, state)
    assert h.shape == shape
    if shape[0] == 0:
        assert torch.equal(last, state)
        assert float(R.gated_scan(x, x)[1].abs().sum()) == 0
    dx, dgate, dstate = R.gated_scan_bwd(x, state, x, x, state, None, marks)
    assert dx.shape == shape and dgate.shape == shape and dstate.shape == state.shape
    if shape[0] == 0:
        assert torch.equal(dstate, state)


def test_autograd(R):
    """Through autograd: both results, either alone, against differences of the definition in 64 bits."""
    k, g = data(70, 2, 40, seed=9)
    leaves = [k[n].requires_grad_() for n in ('x', 'gate', 'state')]
    h, last = R.gated_scan(**k)
    want = run(R, {n: t.detach() for n, t in k.items()}, g)
    got = torch.autograd.grad((h * g['dh']).sum() + (last * g['dlast']).sum(), leaves, retain_graph=True)
    for a, n in zip(got, ('dx', 'dgate', 'dstate')):
        assert torch.equal(a, want[n])
    zero = torch.zeros_like(g['dh'])
    only = torch.autograd.grad((last * g['dlast']).sum(), leaves, retain_graph=True)
    for a, n in zip(only, ('dx', 'dgate', 'dstate')):
        assert torch.equal(a, run(R, {n: t.detach() for n, t in k.items()}, dict(g, dh=zero))[n])
    h.sum().backward()
    assert all(t.grad is not None for t in leaves)
    d = {n: t.detach().double() if n != 'reset' else t for n, t in k.items()}
    gen = torch.Generator(device=DEV).manual_seed(4)
    f = lambda k: float((definition(**k)['h'][0] * g['dh'].double()).sum() + (definition(**k)['last'][0] * g['dlast'].double()).sum())  # noqa: E731
    for n, grad in zip(('x', 'gate', 'state'), got):
        v = torch.randn(d[n].shape, generator=gen, device=DEV, dtype=torch.float64)
        slope = (f(dict(d, **{n: d[n] + 1e-5 * v})) - f(dict(d, **{n: d[n] - 1e-5 * v}))) / 2e-5
        # O(h^2) of the difference, and fp32 in the gradient
        assert abs(slope - float((grad.double() * v).sum())) <= 1e-5 * float((grad.double() * v).abs().sum())


def test_stream_and_graph(R):
    print('[scan] graph', flush=True)
    k, g = data(700, 2, 100, torch.bfloat16, 10)
    run(R, k, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(R, k, g)
    torch.cuda.current_stream().wait_stream(side)
    want = run(R, k, g)
    assert all(torch.equal(again[n], want[n]) for n in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(R, k, g)
    for i in range(4):
        k2, g2 = data(700, 2, 100, torch.bfloat16, 30 + i)
        for d, s in ((k, k2), (g, g2)):
            for n in d:
                d[n].copy_(s[n])
        want = run(R, k2, g2)
        graph.replay()
        torch.cuda.synchronize()
        for n in want:
            assert torch.equal(out[n], want[n]), (i, n)


def test_refusals(R):
    k, g = data(100, 3, 8, seed=11)
    for change in (dict(x=k['x'].cpu()), dict(x=k['x'].double()), dict(x=k['x'][0, 0]), dict(gate=k['gate'].bfloat16()), dict(gate=k['gate'][:50]),
                   dict(state=k['state'].double()), dict(state=k['state'][:2]), dict(reset=k['reset'].float()), dict(reset=k['reset'][:9]),
                   dict(reset=k['reset'].cpu())):
        with pytest.raises(ValueError):
            R.gated_scan(**dict(k, **change))
    marks = R.gated_scan_fwd(**k)[2]
    assert marks is not None
    for bad in (None, marks[:0], marks.double()):
        with pytest.raises(ValueError):
            R.gated_scan_bwd(g['dh'], None, **k, marks=bad)
    with pytest.raises(ValueError):
        R.gated_scan_bwd(g['dh'].double(), None, **k, marks=marks)
    with pytest.raises(ValueError):
        R.gated_scan_bwd(g['dh'], g['dlast'].half(), **k, marks=marks)
