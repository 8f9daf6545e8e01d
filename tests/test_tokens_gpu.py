"""token_logprobs (csrc/d1_tokens.hip) against the definition in 64 bits: log probability, entropy,
alternatives (exactly, lowest index first among equal values) and the gradient, over row lengths on
both sides of every kernel's range, element types, row strides, masks and the values where a softmax
goes wrong. With u = 2^-24 a lane adds about V/256 terms in a row (V/64 in the short kernels), each
with a relative error of a few u, and a term e^d carries an error of about 1.5 |d| u from the
product d log2(e): the tolerances below are these sums, taken with the data's own p and d."""
import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}


@pytest.fixture(scope='module')
def T():
    return importlib.import_module('dcss-auto_amd.tokens')


def reference(logits, tokens, mask, top):
    """In 64 bits; (logp, entropy, ids, top_logp, p, lp, tolerance pieces)."""
    x = logits.double()
    allowed = torch.ones_like(x, dtype=torch.bool) if mask is None else mask.bool().expand(x.shape)
    x = torch.where(allowed, x, -math.inf)
    m = x.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    d = x - m
    e = d.exp()
    s = e.sum(1, keepdim=True)
    p = e / torch.where(s > 0, s, 1.0)
    lp = torch.where(s > 0, d - torch.where(s > 0, s, 1.0).log(), -math.inf)
    entropy = -torch.where(p > 0, p * lp, torch.where(p == 0, 0.0, p)).sum(1)
    inside = (tokens >= 0) & (tokens < x.shape[1])
    at = torch.where(inside, tokens, 0)
    logp = torch.where(tokens < 0, 0.0, torch.where(inside, lp.gather(1, at[:, None])[:, 0], math.nan))
    far = torch.where(p > 0, d, 0.0)
    depth = x.shape[1] / 64 + 24
    spread = (p * far.abs()).sum(1), (p * far * far).sum(1)
    h_tol = U * (depth * (1 + spread[0]) + 2 * spread[1])
    ids = vals = None
    if top:
        order = torch.sort(torch.where(allowed, logits.float(), -math.inf), dim=1, descending=True, stable=True).indices
        # allowed entries first: a masked one is never an alternative, an allowed -inf is
        order = order.gather(1, torch.sort((~allowed).gather(1, order).to(torch.uint8), dim=1, stable=True).indices)
        ids = order[:, :top]
        vals = lp.gather(1, ids)
        here = allowed.gather(1, ids)
        ids, vals = torch.where(here, ids, -1), torch.where(here, vals, -math.inf)
    return dict(logp=logp, entropy=entropy, ids=ids, vals=vals, p=p, lp=lp, d=far, s=s[:, 0], allowed=allowed, depth=depth,
                h_tol=h_tol, lp_tol=lambda v: U * (depth + 3 * v.abs()))


def grad_reference(r, tokens, g, h):
    live = (r['s'] > 0)[:, None]
    lp = torch.where(r['p'] > 0, r['lp'], 0.0)
    g = torch.where(tokens < 0, 0.0, g.double())[:, None]
    h = h.double()[:, None]
    hot = torch.zeros_like(r['p'])
    inside = (tokens >= 0) & (tokens < r['p'].shape[1])
    hot[torch.arange(len(tokens), device=hot.device)[inside], tokens[inside]] = 1.0
    want = g * (hot - r['p']) - h * r['p'] * (lp + r['entropy'][:, None])
    want = torch.where(r['allowed'] & live, want, 0.0)
    tol = U * (2 * r['depth'] + 24 + 3 * r['d'].abs()) * r['p'] * (g.abs() + 2 * h.abs() * (lp.abs() + r['entropy'][:, None] + 1))
    return want, tol + 2 * U * g.abs() * hot


def close(got, want, tol, what):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f'{what}: NaN in other places'
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), f'{what}: infinities differ'
    ok = torch.isfinite(want)
    off = ((got - want).abs() - tol)[ok]
    assert off.numel() == 0 or float(off.max()) <= 0, f'{what}: {float((got - want).abs()[ok].max()):.3g} off'


def check(T, logits, tokens, mask=None, top=0, g=None, h=None):
    r = reference(logits, tokens, mask, top)
    out = T.token_logprobs(logits, tokens, mask=mask, top=top)
    close(out.logp, r['logp'], r['lp_tol'](torch.nan_to_num(r['logp'], neginf=0.0)), 'logp')
    close(out.entropy, r['entropy'], r['h_tol'], 'entropy')
    if top:
        assert torch.equal(out.top_ids, r['ids']), 'alternatives'
        close(out.top_logp, r['vals'], r['lp_tol'](torch.nan_to_num(r['vals'], neginf=0.0)), 'top_logp')
    else:
        assert out.top_ids is None and out.top_logp is None
    if g is not None:
        want, tol = grad_reference(r, tokens, g, h)
        got = T.token_logprobs_bwd(logits, tokens, out, g, h, mask=mask)
        assert got.dtype == logits.dtype and got.shape == logits.shape and got.is_contiguous()
        close(got, want, tol + ROUND[logits.dtype] * want.abs() + TINY[logits.dtype], 'dlogits')
    return out


def inputs(rows, vocab, dtype, seed, pad=0, scale=3.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    logits = (torch.randn(rows, vocab + pad, generator=g, device='cuda') * scale).to(dtype)[:, :vocab]
    tokens = torch.randint(0, vocab, (rows,), generator=g, device='cuda')
    return logits, tokens, torch.randn(rows, generator=g, device='cuda'), torch.randn(rows, generator=g, device='cuda') * 0.1


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('rows,vocab,pad', [
    (1, 1, 0), (3, 2, 0), (65, 3, 1), (300, 16, 1), (257, 17, 0), (1000, 25, 0), (130, 33, 2), (67, 64, 0), (66, 65, 0),
    (9, 255, 1), (5, 256, 0), (6, 257, 0), (7, 1000, 24), (3, 1023, 0), (4, 1024, 0), (3, 1025, 0), (5, 2047, 1),
    (2, 2048, 0), (2, 2049, 3), (1, 4097, 0), (700, 1300, 0), (3, 8191, 0), (1, 50001, 0), (33, 16385, 1)])
def test_sizes(T, rows, vocab, pad, dtype):
    print(f'[tokens] {rows} x {vocab}+{pad} {dtype}', flush=True)
    logits, tokens, g, h = inputs(rows, vocab, dtype, 7 * rows + vocab, pad)
    tokens[::3] = logits.float().argmax(1)[::3]
    for top in sorted({0, 1, min(5, vocab), min(64, vocab)}):
        check(T, logits, tokens, top=top, g=g, h=h)


@pytest.mark.parametrize('vocab', [19, 300, 1500, 20000])
@pytest.mark.parametrize('kind', ['full', 'row', 'bytes', 'strided'])
def test_masks(T, vocab, kind):
    print(f'[tokens] masks {vocab} {kind}', flush=True)
    rows = 37
    logits, tokens, g, h = inputs(rows, vocab, torch.float32, vocab)
    gen = torch.Generator(device='cuda').manual_seed(vocab + 1)
    mask = torch.rand(rows, vocab, generator=gen, device='cuda') < 0.5
    mask[3] = False                                        # nothing allowed
    mask[4] = False
    mask[4, vocab - 1] = True                              # one entry
    tokens[4] = vocab - 1
    tokens[5], tokens[6] = -1, -100                        # padding
    mask[6] = False                                        # padding and nothing allowed
    tokens[7] = vocab                                      # not a token
    # what stands in masked places is not looked at
    logits[~mask] = torch.tensor([math.nan, math.inf, -math.inf, 3e38], device='cuda')[
        torch.randint(0, 4, (int((~mask).sum()),), generator=gen, device='cuda')]
    if kind == 'row':
        logits, tokens, g, h = inputs(rows, vocab, torch.float32, vocab)
        mask = mask[9]
    elif kind == 'bytes':
        mask = mask.to(torch.uint8) * 255
    elif kind == 'strided':
        wide = torch.zeros(rows, vocab + 5, dtype=torch.bool, device='cuda')
        wide[:, :vocab] = mask
        mask = wide[:, :vocab]
    check_rows = torch.arange(rows, device='cuda') != 7 if kind != 'row' else torch.ones(rows, dtype=torch.bool, device='cuda')
    top = min(20, vocab)
    out = T.token_logprobs(logits, tokens, mask=mask, top=top)
    back = T.token_logprobs_bwd(logits, tokens, out, g, h, mask=mask)
    if kind != 'row':
        assert math.isnan(out.logp[7]) and torch.isnan(back[7][mask[7].bool()]).all() and (back[7][~mask[7].bool()] == 0).all()
        assert out.logp[3] == -math.inf and out.entropy[3] == 0 and (out.top_ids[3] == -1).all() and (back[3] == 0).all()
        assert out.logp[6] == 0 and out.entropy[6] == 0 and (back[6] == 0).all()
        assert out.logp[4] == 0 and out.top_ids[4, 0] == vocab - 1 and (out.top_ids[4, 1:] == -1).all()
    keep = check_rows
    check(T, logits[keep], tokens[keep], mask=mask if mask.dim() == 1 else mask[keep], top=top, g=g[keep], h=h[keep])


@pytest.mark.parametrize('vocab', [5, 40, 700, 3000, 9000])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['fp32', 'bf16', 'fp16'])
def test_special_values(T, vocab, dtype):
    print(f'[tokens] values {vocab} {dtype}', flush=True)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    rows = 12
    logits, tokens, g, h = inputs(rows, vocab, dtype, 11)
    logits[0] = low                                        # a mask of the type's lowest value everywhere
    logits[1] = low
    logits[1, vocab // 2] = 1.0                            # and everywhere but one
    tokens[1] = vocab // 2
    logits[2] = -math.inf
    logits[3, 1:] = -math.inf
    tokens[3] = 0
    logits[4] = 0.0                                        # ties: 0 and -0 are equal
    logits[4, 1::2] = -0.0
    logits[5] = high
    logits[6, ::2] = low
    logits[7, ::2] = -math.inf
    tokens[7] = 1
    tokens[8] = -5
    logits[9] = 88.0                                       # equal entries: the lowest indices, in order
    logits[10] *= 8.0
    logits[11, 2] = high
    check(T, logits, tokens, top=min(vocab, 33), g=g, h=h)
    for bad in (math.nan, math.inf):
        x = logits.clone()
        x[10, vocab - 1] = bad
        out = T.token_logprobs(x, tokens, top=2)
        assert torch.isnan(out.logp[10]) and torch.isnan(out.entropy[10]) and torch.isnan(out.top_logp[10]).all()
        assert out.top_ids[10, 0] == vocab - 1
        assert torch.isnan(T.token_logprobs_bwd(x, tokens, out, g, h)[10]).all()
        good = T.token_logprobs(logits, tokens, top=2)
        keep = torch.arange(rows, device='cuda') != 10
        for a, b in zip(out, good):
            assert torch.equal(a[keep], b[keep])
    x = torch.full((2, vocab), math.nan, dtype=dtype, device='cuda')
    out = T.token_logprobs(x, tokens[:2], top=1)
    assert torch.isnan(out.logp).all() and (out.top_ids == 0).all()


@pytest.mark.parametrize('vocab', [60, 1024, 5000, 40000])
def test_order_among_ties(T, vocab):
    """Few distinct values, rising and falling rows: lists that overflow and lists of equal keys."""
    print(f'[tokens] ties {vocab}', flush=True)
    g = torch.Generator(device='cuda').manual_seed(vocab)
    x = torch.randint(0, 3, (6, vocab), generator=g, device='cuda').to(torch.bfloat16)
    x[1] = 1.0
    x[2] = torch.arange(vocab, device='cuda').float() / 64      # rising, many equal after rounding
    x[3] = -torch.arange(vocab, device='cuda').float() / 64
    x[4] = (torch.arange(vocab, device='cuda') % 256).float()
    check(T, x, torch.zeros(6, dtype=torch.int64, device='cuda'), top=min(64, vocab))
    check(T, torch.arange(2 * vocab, device='cuda', dtype=torch.float32).view(2, vocab) * 1e-3,
          torch.zeros(2, dtype=torch.int64, device='cuda'), top=min(64, vocab))


def test_shapes_strides_and_streams(T):
    print('[tokens] shapes', flush=True)
    logits, tokens, _, _ = inputs(24, 50, torch.float32, 3)
    want = T.token_logprobs(logits, tokens, top=4)
    three = T.token_logprobs(logits.view(2, 3, 4, 50), tokens.view(2, 3, 4), top=4)
    assert three.logp.shape == (2, 3, 4) and three.top_ids.shape == (2, 3, 4, 4) and three.stats.shape == (2, 3, 4, 2)
    for a, b in zip(three, want):
        assert torch.equal(a.reshape(b.shape), b)
    turned = logits.t().contiguous().t()                    # columns adjacent: taken as a copy
    cut = torch.stack([logits, logits + 1], 1)[:, 0]        # rows 100 apart
    for x in (turned, cut):
        for a, b in zip(T.token_logprobs(x, tokens, top=4), want):
            assert torch.equal(a, b)
    one = T.token_logprobs(logits[5], tokens[5], top=4)     # a single row without a batch dimension
    assert one.logp.shape == () and torch.equal(one.logp, want.logp[5]) and torch.equal(one.top_ids, want.top_ids[5])
    same = T.token_logprobs(logits[5].expand(24, 50), tokens[5].expand(24), top=4)
    assert torch.equal(same.logp, want.logp[5].expand(24))
    torch.testing.assert_close(want.lse, torch.logsumexp(logits.double(), 1).float(), rtol=0, atol=1e-5)
    empty = T.token_logprobs(logits[:0], tokens[:0], top=4)
    assert empty.logp.shape == (0,) and empty.top_ids.shape == (0, 4)
    assert T.token_logprobs_bwd(logits[:0], tokens[:0], empty, tokens[:0].float(), None).shape == (0, 50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    long, t2, g, h = inputs(3, 9001, torch.bfloat16, 4)
    a = T.token_logprobs(long, t2, top=9)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = T.token_logprobs(long, t2, top=9)
        gb = T.token_logprobs_bwd(long, t2, b, g, h)
    side.synchronize()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    assert torch.equal(gb, T.token_logprobs_bwd(long, t2, a, g, h))


@pytest.mark.parametrize('vocab', [25, 3001])
def test_gradient_against_differences(T, vocab):
    """The directional derivative of sum(c logp + d entropy) from the forward pass alone. The step
    0.02 leaves a truncation of order 0.02^2 / 6 times third derivatives (at most about 1 a row here) and a
    rounding of 1e-6 / 0.02 a row: 2e-4 of the 2-norm of the rows' parts."""
    print(f'[tokens] differences {vocab}', flush=True)
    x, tokens, c, d = inputs(40, vocab, torch.float32, 5, scale=1.5)
    gen = torch.Generator(device='cuda').manual_seed(6)
    v = torch.randn(x.shape, generator=gen, device='cuda')
    v /= v.norm(dim=1, keepdim=True) / 2.0
    x.requires_grad_()
    out = T.token_logprobs(x, tokens)
    (c * out.logp + d * out.entropy).sum().backward()

    def f(y):
        o = T.token_logprobs(y, tokens)
        return c.double() * o.logp.double() + d.double() * o.entropy.double()
    with torch.no_grad():
        diff = (f(x + 0.01 * v) - f(x - 0.01 * v)) / 0.02
        along = (x.grad.double() * v.double()).sum(1)
    assert float((diff - along).norm() / along.norm()) < 1e-3


def test_autograd(T):
    print('[tokens] autograd', flush=True)
    x, tokens, g, h = inputs(31, 77, torch.float32, 8)
    mask = torch.rand(31, 77, device='cuda') < 0.8
    x.requires_grad_()
    out = T.token_logprobs(x, tokens, mask=mask, top=3)
    assert out.logp.requires_grad and not out.top_logp.requires_grad and not out.stats.requires_grad
    (a,) = torch.autograd.grad((out.logp * g).sum() + (out.entropy * h).sum(), x, retain_graph=True)
    assert torch.equal(a, T.token_logprobs_bwd(x.detach(), tokens, out, g, h, mask=mask))
    (b,) = torch.autograd.grad(out.logp.sum(), x, retain_graph=True)        # a broadcast gradient, one output alone
    assert torch.equal(b, T.token_logprobs_bwd(x.detach(), tokens, out, torch.ones_like(g), None, mask=mask))
    (e,) = torch.autograd.grad(out.entropy.mean(), x)
    want = T.token_logprobs_bwd(x.detach(), tokens, out, None, torch.full_like(h, 1 / 31), mask=mask)
    torch.testing.assert_close(e, want, rtol=1e-6, atol=0)
    with torch.no_grad():
        assert not T.token_logprobs(x, tokens).logp.requires_grad


def test_graph_replays(T):
    """A captured forward and backward, replayed with eager work between the replays."""
    print('[tokens] graph', flush=True)
    x, tokens, g, h = inputs(5, 6000, torch.bfloat16, 9)
    static = x.clone().contiguous()
    T.token_logprobs(static, tokens, top=8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = T.token_logprobs(static, tokens, top=8)
        back = T.token_logprobs_bwd(static, tokens, out, g, h)
    for k in range(4):
        new = (x.float() * (1 + k)).to(torch.bfloat16)
        static.copy_(new)
        graph.replay()
        eager = T.token_logprobs(new.contiguous(), tokens, top=8)
        for p, q in zip(out, eager):
            assert torch.equal(p, q)
        assert torch.equal(back, T.token_logprobs_bwd(new.contiguous(), tokens, eager, g, h))
        torch.cuda.synchronize()


def test_many_rows(T):
    """More rows than a launch has workgroups, and an offset beyond 2^31 elements."""
    print('[tokens] many rows', flush=True)
    n = (1 << 20) * 64 + 77
    x = torch.zeros(n, 2, dtype=torch.float16, device='cuda')
    x[-1, 1] = 3.0
    tokens = torch.ones(n, dtype=torch.int64, device='cuda')
    out = T.token_logprobs(x, tokens)
    assert abs(float(out.logp[-1]) - math.log(1 / (1 + math.exp(-3.0)))) < 1e-6
    assert float((out.logp[:-1] - math.log(0.5)).abs().max()) < 1e-6
    del x, tokens, out
    wide = torch.zeros(3, 1 << 30, dtype=torch.float16, device='cuda')   # rows 2^30 elements apart
    x = wide[:, :1500]
    x.copy_(torch.randn(3, 1500, device='cuda'))
    check(T, x, torch.tensor([0, 7, 1499], device='cuda'), top=5, g=torch.ones(3, device='cuda'), h=torch.ones(3, device='cuda'))


def test_refusals(T):
    print('[tokens] refusals', flush=True)
    x, tokens, g, h = inputs(4, 10, torch.float32, 1)
    for args in ((x.double(), tokens), (x.cpu(), tokens.cpu()), (x, tokens.int()), (x, tokens[:3]), (x, tokens.cpu()),
                 (x[:, :0], tokens), (x[0, 0], tokens[0])):
        with pytest.raises(ValueError):
            T.token_logprobs(*args)
    for top in (-1, 11, 65, True, 2.0):
        with pytest.raises(ValueError):
            T.token_logprobs(x, tokens, top=top)
    for mask in (torch.ones(4, 9, device='cuda', dtype=torch.bool), torch.ones(4, 10, device='cuda'),
                 torch.ones(4, 10, dtype=torch.bool), torch.ones(4, 1, device='cuda', dtype=torch.bool)):
        with pytest.raises(ValueError):
            T.token_logprobs(x, tokens, mask=mask)
    out = T.token_logprobs(x, tokens)
    for dl, de in ((g.double(), h), (g[:3], h), (g, h.cpu())):
        with pytest.raises(ValueError):
            T.token_logprobs_bwd(x, tokens, out, dl, de)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('rows,vocab', [(1, 120001), (5, 60008), (37, 53251), (200, 57344), (1030, 70001)])
def test_rows_in_segments(T, rows, vocab, dtype):
    """Rows long enough to be cut: masks that empty whole segments, ties over the cuts, NaN, infinities."""
    print(f'[tokens] segments {rows} x {vocab} {dtype}', flush=True)
    logits, tokens, g, h = inputs(rows, vocab, dtype, 2 * rows + vocab, pad=1)
    gen = torch.Generator(device='cuda').manual_seed(rows)
    mask = torch.rand(rows, vocab, generator=gen, device='cuda') < 0.6
    check(T, logits, tokens, top=20, g=g, h=h)
    check(T, logits, tokens, mask=mask, top=64, g=g, h=h)
    mask[:, vocab // 9:] = False                            # all later segments empty
    mask[rows // 2] = False
    mask[rows // 2, vocab - 2:] = True                      # the last two entries alone
    tokens[0] = -1
    check(T, logits, tokens, mask=mask, top=5, g=g, h=h)
    ties = (torch.arange(vocab, device='cuda') % 50 == 49).to(dtype).expand(rows, vocab)
    check(T, ties, tokens, top=33)
    odd = logits.clone()
    odd[:, 7::1001] = -math.inf
    odd[rows - 1] = torch.finfo(dtype).min
    check(T, odd, tokens, top=3, g=g, h=h)
    odd[rows - 1, vocab - 1] = math.nan
    out = T.token_logprobs(odd, tokens, top=1)
    assert torch.isnan(out.entropy[rows - 1]) and out.top_ids[rows - 1, 0] == vocab - 1
    assert not torch.isnan(out.entropy[:rows - 1]).any()


@pytest.mark.parametrize('rows,vocab,dtype', [(rows, vocab, dtype) for rows, vocab in ((2050, 3001), (4100, 5000), (1100, 9001), (800, 33001))
                                              for dtype in (torch.float32, torch.bfloat16, torch.float16)]
                         + [(127000, 1100, torch.bfloat16), (64100, 2111, torch.bfloat16)],
                         ids=lambda x: str(x).replace('torch.', ''))
def test_many_rows(T, rows, vocab, dtype):
    """Whole rows on a wave and on workgroups; results past what the caches hold."""
    print(f'[tokens] many rows {rows} x {vocab} {dtype}', flush=True)
    logits, tokens, g, h = inputs(rows, vocab, dtype, rows + vocab, pad=3)
    check(T, logits, tokens, top=4, g=g, h=h)
    mask = torch.rand(vocab, device='cuda', generator=torch.Generator(device='cuda').manual_seed(vocab)) < 0.4
    check(T, logits, tokens, mask=mask, g=g, h=h)


def test_offsets_past_32_bits(T):
    """Rows 2^31 elements apart, masks too, and a gradient of more than 2^32 elements."""
    print('[tokens] offsets', flush=True)
    rows, vocab, apart = 3, 1031, 2 ** 31 + 8
    logits, tokens, g, h = inputs(rows, vocab, torch.float16, 77)
    mask = torch.rand(rows, vocab, device='cuda', generator=torch.Generator(device='cuda').manual_seed(3)) < 0.5
    far = torch.empty((rows - 1) * apart + vocab, dtype=torch.float16, device='cuda').as_strided((rows, vocab), (apart, 1))
    far_mask = torch.empty((rows - 1) * apart + vocab, dtype=torch.bool, device='cuda').as_strided((rows, vocab), (apart, 1))
    far.copy_(logits)
    far_mask.copy_(mask)
    check(T, far, tokens, mask=far_mask, top=5, g=g, h=h)
    check(T, far[:, :200], tokens.clamp(max=199), mask=far_mask[:, :200], top=5, g=g, h=h)
    del far, far_mask
    rows, vocab = 260, 1 << 24
    one = torch.randn(1, vocab, device='cuda', generator=torch.Generator(device='cuda').manual_seed(4)).to(torch.bfloat16)
    logits, tokens = one.expand(rows, vocab), torch.full((rows,), vocab - 5, device='cuda')
    g, h = torch.ones(rows, device='cuda'), torch.ones(rows, device='cuda')
    out = T.token_logprobs(logits, tokens)
    first = T.token_logprobs(one, tokens[:1])
    close(out.logp, first.logp.double().expand(rows), 1e-5, 'logp')
    d = T.token_logprobs_bwd(logits, tokens, out, g, h)
    assert torch.equal(d[rows - 1], d[0]) and torch.equal(d[rows - 2], d[0]) and float(d[rows - 1, vocab - 5]) > 0.9
    del d
    torch.cuda.empty_cache()
