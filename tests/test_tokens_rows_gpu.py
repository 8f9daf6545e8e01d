"""More rows than a launch has workgroups (2^20): the row loops' second round."""
import importlib
import math

import pytest
import torch

import test_tokens_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def T():
    return importlib.import_module('dcss-auto_amd.tokens')


def test_more_short_rows_than_workgroups(T):
    """64 rows a workgroup; and rows 2^30 elements apart."""
    print('[tokens] more short rows than workgroups', flush=True)
    n = (1 << 20) * 64 + 77
    x = torch.zeros(n, 2, dtype=torch.float16, device='cuda')
    x[-1, 1] = 3.0
    tokens = torch.ones(n, dtype=torch.int64, device='cuda')
    out = T.token_logprobs(x, tokens, top=1)
    assert abs(float(out.logp[-1]) - math.log(1 / (1 + math.exp(-3.0)))) < 1e-6
    assert float((out.logp[:-1] - math.log(0.5)).abs().max()) < 1e-6
    assert int(out.top_ids[-1, 0]) == 1 and not bool(out.top_ids[:-1].any())
    d = T.token_logprobs_bwd(x, tokens, out, torch.ones(n, device='cuda'), None)
    p = 1 / (1 + math.exp(-3.0))
    assert abs(float(d[-1, 1]) - (1 - p)) < 2.0 ** -11 * (1 - p) + 1e-6 and bool((d[:-1, 0] == -0.5).all())
    del x, tokens, out, d
    wide = torch.zeros(3, 1 << 30, dtype=torch.float16, device='cuda')
    x = wide[:, :1500]
    x.copy_(torch.randn(3, 1500, device='cuda'))
    test_tokens_gpu.check(T, x, torch.tensor([0, 7, 1499], device='cuda'), top=5, g=torch.ones(3, device='cuda'),
                          h=torch.ones(3, device='cuda'))


@pytest.mark.parametrize('masked', [False, True])
def test_more_long_rows_than_workgroups(T, masked):
    """A row a workgroup (1,100 entries), alternatives and gradients: the last row of the first round and those of the
    second have the bits of the same rows in a small call, which is checked against 64 bits."""
    print(f'[tokens] more long rows than workgroups {masked}', flush=True)
    n, vocab = (1 << 20) + 300, 1100
    gen = torch.Generator(device='cuda').manual_seed(2)
    x = torch.randn(n, vocab, generator=gen, device='cuda', dtype=torch.bfloat16).mul_(3)
    tokens = torch.randint(-1, vocab, (n,), generator=gen, device='cuda')
    g, h = torch.randn(n, generator=gen, device='cuda'), torch.randn(n, generator=gen, device='cuda')
    mask = None
    if masked:
        mask = torch.randint(0, 3, (n, vocab), generator=gen, device='cuda', dtype=torch.uint8)
        mask[(1 << 20) - 3] = 0
        mask[(1 << 20) + 5] = 0
    out = T.token_logprobs(x, tokens, mask=mask, top=20)
    d = T.token_logprobs_bwd(x, tokens, out, g, h, mask=mask)
    for rows in (slice(0, 300), slice((1 << 20) - 300, 1 << 20), slice(1 << 20, n)):
        part = None if mask is None else mask[rows]
        few = T.token_logprobs(x[rows], tokens[rows], mask=part, top=20)
        assert all(torch.equal(a[rows], b) for a, b in zip(out, few))
        assert torch.equal(d[rows], T.token_logprobs_bwd(x[rows], tokens[rows], few, g[rows], h[rows], mask=part))
        test_tokens_gpu.check(T, x[rows], tokens[rows], mask=part, top=20, g=g[rows], h=h[rows])
    del x, mask, out, d
    torch.cuda.empty_cache()
