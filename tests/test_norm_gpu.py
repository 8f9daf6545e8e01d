"""layer_norm (csrc/d1_norm.hip) against the definition in 64 bits, forward, backward and the weight's
and bias's gradients, over widths on both sides of every row shape, element types, strides and row counts.
With u = 2^-24 and a sum of about width/64 + 16 terms a lane, the mean is off by at most
K max|x|, K = u (width/64 + 64), so xh by K A with A = (max|x| + |mean|) rstd + |xh|; products and sums after
it carry these over (the tolerances spell that out), and a result is rounded once to its type."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}


@pytest.fixture(scope='module')
def N():
    return importlib.import_module('dcss-auto_amd.norm')


def inputs(rows, width, dtype, wdtype, seed, pad=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731
    x = (rand(rows, width + pad) * 1.5 + 0.7).to(dtype)[:, :width]
    dy = rand(rows, width + pad).to(dtype)[:, :width]
    return x, dy, (1 + 0.2 * rand(width)).to(wdtype), (0.3 * rand(width)).to(wdtype)


def within(got, want, tol, what):
    off = (got.double() - want).abs() - tol - ROUND[got.dtype] * want.abs() - TINY[got.dtype]
    assert got.numel() == 0 or float(off.max()) <= 0, f'{what}: {float((got.double() - want).abs().max()):.3g} off'


def check(N, x, dy, w, b, eps=1e-5):
    width, rows = x.shape[-1], x.numel() // x.shape[-1]
    y, mean, rstd = N.layer_norm_fwd(x, w, b, eps)
    dx, dw, db = N.layer_norm_bwd(dy, x, w, b, mean, rstd)
    X, D = x.double().reshape(rows, width), dy.double().reshape(rows, width)
    W = torch.ones(width, dtype=torch.float64, device='cuda') if w is None else w.double()
    B = torch.zeros(width, dtype=torch.float64, device='cuda') if b is None else b.double()
    mu = X.mean(1, keepdim=True)
    var = (X - mu).square().mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = (X - mu) * r
    K = U * (width / 64 + 64)
    A = (X.abs().amax(1, keepdim=True) + mu.abs()) * r + xh.abs()
    within(mean.reshape(rows, 1), mu, K * X.abs().amax(1, keepdim=True), 'mean')
    within(rstd.reshape(rows, 1), r, K * r * (1 + A.amax(1, keepdim=True)), 'rstd')
    # the variance is about a mean that is K max|x| off: second order; r is off by K (1 + A K)
    within(y.reshape(rows, width), xh * W + B, K * (A + xh.abs()) * W.abs() + U * B.abs(), 'y')
    u = D * W
    c1, c2 = u.mean(1, keepdim=True), (u * xh).mean(1, keepdim=True)
    a1, a2 = u.abs().mean(1, keepdim=True), (u * xh).abs().mean(1, keepdim=True)
    off2 = a2 + (u.abs() * A).mean(1, keepdim=True)               # of c2: its terms' errors and the sum's
    tol = K * r * (u.abs() + a1 + xh.abs() * off2 + A * (c2.abs() + a2) + (u - c1 - xh * c2).abs() * (1 + A))
    within(dx.reshape(rows, width), r * (u - c1 - xh * c2), tol, 'dx')
    deep = U * (rows + 64)                                        # no more terms than rows are added in a row
    if w is not None:
        within(dw, (D * xh).sum(0), deep * (D * xh).abs().sum(0) + K * (D.abs() * A).sum(0), 'dweight')
    else:
        assert dw is None
    if b is not None:
        within(db, D.sum(0), deep * D.abs().sum(0), 'dbias')
    else:
        assert db is None
    assert y.dtype == dx.dtype == x.dtype and y.shape == dx.shape == x.shape
    return y, dx, dw, db


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float32), (torch.float16, torch.float16)]


@pytest.mark.parametrize('dtype,wdtype', TYPES, ids=['fp32', 'bf16-fp32', 'bf16', 'fp16-fp32', 'fp16'])
@pytest.mark.parametrize('rows,width,pad', [
    (1, 1, 0), (5, 2, 0), (33, 7, 1), (100, 16, 0), (65, 17, 0), (70, 32, 0), (50, 33, 0), (129, 64, 3), (31, 65, 0),
    (64, 128, 0), (20, 129, 0), (300, 256, 0), (18, 257, 0), (9, 511, 1), (7, 512, 8), (6, 513, 0), (11, 1000, 0),
    (5, 1024, 0), (3, 1025, 0), (4, 1800, 0), (3, 2049, 0), (2, 4096, 0), (3, 4097, 5), (2, 8192, 0), (3, 8193, 0),
    (2, 16383, 0), (1, 16384, 0), (2100, 300, 0), (1111, 5000, 0)])
def test_sizes(N, rows, width, pad, dtype, wdtype):
    print(f'[norm] {rows} x {width}+{pad} {dtype} {wdtype}', flush=True)
    check(N, *inputs(rows, width, dtype, wdtype, rows + 3 * width, pad))


@pytest.mark.parametrize('weight,bias', [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize('width', [40, 5000])
def test_without_weight_or_bias(N, width, weight, bias):
    print(f'[norm] {width} weight {weight} bias {bias}', flush=True)
    x, dy, w, b = inputs(21, width, torch.float32, torch.float32, 3)
    check(N, x, dy, w if weight else None, b if bias else None)


def test_values(N):
    """Constant rows, a large mean beside a small spread, large and small magnitudes; a row with a
    NaN or an infinity spoils itself alone."""
    print('[norm] values', flush=True)
    x, dy, w, b = inputs(8, 256, torch.float32, torch.float32, 5)
    x[0] = 3.25
    x[1] = 0.0
    x[2] = 1000.0 + x[2]
    x[3] *= 1e15
    x[4] *= 1e-12
    y, dx, dw, db = check(N, x, dy, w, b)
    assert torch.equal(y[0], b) and torch.equal(y[1], b)
    bad = x.clone()
    bad[5, 17], bad[6, 200] = float('nan'), float('inf')
    y2, mean, rstd = N.layer_norm_fwd(bad, w, b)
    dx2, dw2, db2 = N.layer_norm_bwd(dy, bad, w, b, mean, rstd)
    keep = [0, 1, 2, 3, 4, 7]
    assert torch.equal(y2[keep], y[keep]) and torch.equal(dx2[keep], dx[keep]) and torch.equal(db2, db)
    assert torch.isnan(y2[5]).all() and torch.isnan(y2[6]).all() and torch.isnan(dx2[5]).all() and torch.isnan(dw2).all()


def test_shapes_strides_streams_and_repeats(N):
    print('[norm] shapes', flush=True)
    x, dy, w, b = inputs(24, 300, torch.bfloat16, torch.float32, 6)
    y, mean, rstd = N.layer_norm_fwd(x, w, b)
    back = N.layer_norm_bwd(dy, x, w, b, mean, rstd)
    y3, mean3, rstd3 = N.layer_norm_fwd(x.view(2, 3, 4, 300), w, b)
    assert mean3.shape == (2, 3, 4) and torch.equal(y3.view(24, 300), y)
    for a, c in zip(N.layer_norm_bwd(dy.view(2, 3, 4, 300), x.view(2, 3, 4, 300), w, b, mean3, rstd3), back):
        assert torch.equal(a.reshape(c.shape), c)
    turned, spread = x.t().contiguous().t(), torch.stack([x, x], 1)[:, 1]
    for z in (turned, spread):
        assert torch.equal(N.layer_norm_fwd(z, w, b)[0], y)
        for a, c in zip(N.layer_norm_bwd(dy.t().contiguous().t(), z, w, b, mean, rstd), back):
            assert torch.equal(a, c)
    row = N.layer_norm_fwd(x[3], w, b)
    assert row[1].shape == () and torch.equal(row[0], y[3])
    same = N.layer_norm_bwd(dy[:1].expand(24, 300), x[:1].expand(24, 300), w, b, mean[:1].expand(24), rstd[:1].expand(24))
    assert torch.equal(same[0], back[0][:1].expand(24, 300))
    none = N.layer_norm_fwd(x[:0], w, b)
    dx, dw, db = N.layer_norm_bwd(dy[:0], x[:0], w, b, none[1], none[2])
    assert none[0].shape == dx.shape == (0, 300) and not dw.any() and not db.any()
    assert not N.layer_norm_bwd(dy[:0], x[:0], None, b, none[1], none[2])[2].any()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys, ms, rs = N.layer_norm_fwd(x, w, b)
        bs = N.layer_norm_bwd(dy, x, w, b, ms, rs)
    side.synchronize()
    assert torch.equal(ys, y) and all(torch.equal(p, q) for p, q in zip(bs, back))
    big, dbig, w2, b2 = inputs(20000, 256, torch.bfloat16, torch.float32, 7)
    _, m2, r2 = N.layer_norm_fwd(big, w2, b2)
    first = N.layer_norm_bwd(dbig, big, w2, b2, m2, r2)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, N.layer_norm_bwd(dbig, big, w2, b2, m2, r2)))


@pytest.mark.parametrize('width', [48, 2000])
def test_gradient_against_differences(N, width):
    """Directional derivatives of sum(dy y) from the forward pass alone: a step of 0.02 leaves 1e-4 of
    truncation and rounding of 1e-6 / 0.02 a term, averaged over the row."""
    print(f'[norm] differences {width}', flush=True)
    x, dy, w, b = inputs(30, width, torch.float32, torch.float32, 8)
    x, w, b = (t.requires_grad_() for t in (x.contiguous(), w, b))
    (N.layer_norm(x, w, b) * dy).sum().backward()
    gen = torch.Generator(device='cuda').manual_seed(9)
    for t, k in ((x, 0), (w, 1), (b, 2)):
        v = torch.randn(t.shape, generator=gen, device='cuda')

        def f(step):
            args = [a.detach() + (step * v if i == k else 0) for i, a in enumerate((x, w, b))]
            return (N.layer_norm(*args).double() * dy.double()).sum()
        diff = float((f(0.01) - f(-0.01)) / 0.02)
        along = float((t.grad.double() * v.double()).sum())
        scale = float(t.grad.double().norm())
        assert abs(diff - along) < 2e-3 * scale * 3


def test_module_and_autograd(N):
    print('[norm] module', flush=True)
    layer = N.LayerNorm(96).cuda()
    x = torch.randn(40, 96, device='cuda').to(torch.bfloat16).requires_grad_()
    y = layer(x)
    assert y.dtype == torch.bfloat16 and layer.weight.dtype == torch.float32
    y.float().sum().backward()                         # a broadcast gradient
    dy = torch.ones_like(x)
    _, mean, rstd = N.layer_norm_fwd(x.detach(), layer.weight.detach(), layer.bias.detach())
    dx, dw, db = N.layer_norm_bwd(dy, x.detach(), layer.weight.detach(), layer.bias.detach(), mean, rstd)
    assert torch.equal(x.grad, dx) and torch.equal(layer.weight.grad, dw) and torch.equal(layer.bias.grad, db)
    assert N.LayerNorm(8, bias=False).bias is None
    frozen = N.layer_norm(x.detach(), layer.weight, None)      # the weight alone needs a gradient
    frozen.float().sum().backward()
    with torch.no_grad():
        assert not layer(x).requires_grad


def test_graph_replays(N):
    print('[norm] graph', flush=True)
    x, dy, w, b = inputs(3000, 256, torch.bfloat16, torch.float32, 10)
    static = x.clone()
    N.layer_norm_fwd(static, w, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = N.layer_norm_fwd(static, w, b)
        back = N.layer_norm_bwd(dy, static, w, b, mean, rstd)
    for k in range(4):
        static.copy_(x * (k + 1))
        graph.replay()
        e, m, r = N.layer_norm_fwd((x * (k + 1)).contiguous(), w, b)
        assert torch.equal(e, y)
        for p, q in zip(back, N.layer_norm_bwd(dy, (x * (k + 1)).contiguous(), w, b, m, r)):
            assert torch.equal(p, q)
        torch.cuda.synchronize()


def test_far_rows(N):
    """Rows 2^30 elements apart: offsets beyond 2^31."""
    print('[norm] far rows', flush=True)
    wide = torch.zeros(4, 1 << 30, dtype=torch.float16, device='cuda')
    x = wide[:, :500]
    x.copy_(torch.randn(4, 500, device='cuda'))
    check(N, x, x, torch.ones(500, dtype=torch.float16, device='cuda'), None)


def test_refusals(N):
    print('[norm] refusals', flush=True)
    x, dy, w, b = inputs(4, 64, torch.bfloat16, torch.float32, 1)
    for args in ((x.cpu(), None, None), (x.double(), None, None), (x, w[:63], None), (x, w.half(), None), (x, w, b.bfloat16()),
                 (x, w.cpu(), None), (x[:, :0], None, None), (x[0, 0], None, None),
                 (torch.zeros(1, 16385, device='cuda'), None, None)):
        with pytest.raises(ValueError):
            N.layer_norm_fwd(*args)
    _, mean, rstd = N.layer_norm_fwd(x, w, b)
    for args in ((dy.float(), x, w, b, mean, rstd), (dy[:3], x, w, b, mean, rstd), (dy, x, w, b, mean[:3], rstd),
                 (dy, x, w, b, mean.double(), rstd)):
        with pytest.raises(ValueError):
            N.layer_norm_bwd(*args)


def test_offsets_past_32_bits(N):
    """Rows 2^31 elements apart, and results of more than 2^32 elements."""
    print('[norm] offsets', flush=True)
    rows, width, apart = 3, 1031, 2 ** 31 + 8
    x, dy, w, b = inputs(rows, width, torch.bfloat16, torch.float32, 5)
    far, fardy = (torch.empty((rows - 1) * apart + width, dtype=torch.bfloat16, device='cuda').as_strided((rows, width), (apart, 1))
                  for _ in range(2))
    far.copy_(x)
    fardy.copy_(dy)
    check(N, far, fardy, w, b)
    del far, fardy
    rows, width = 262400, 16384
    x, dy, w, b = inputs(1, width, torch.bfloat16, torch.float32, 6)
    y, mean, rstd = N.layer_norm_fwd(x.expand(rows, width), w, b)
    one = N.layer_norm_fwd(x, w, b)
    assert torch.equal(y[rows - 1:], one[0]) and torch.equal(y[rows - 2:rows - 1], one[0]) and bool((mean == one[1]).all())
    del y
    dx, dw, db = N.layer_norm_bwd(dy.expand(rows, width), x.expand(rows, width), w, b, mean, rstd)
    one = N.layer_norm_bwd(dy, x, w, b, *one[1:])
    assert torch.equal(dx[rows - 1:], one[0]) and torch.equal(dx[rows - 2:rows - 1], one[0])
    # rows equal terms of a column: partial sums of a workgroup's rows one after the other, then of the workgroups
    assert float(((db.double() - rows * one[2].double()).abs() - U * (rows / 256 + 64) * rows * dy[0].double().abs()).max()) <= 0
    del dx
    torch.cuda.empty_cache()
