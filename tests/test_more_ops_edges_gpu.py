"""The policy loss, the gated recurrence and the orthogonalised updates at their edges: offsets past 32 bits, more rows than
one launch takes, graphs that are kept or share their memory, tangents, transforms and traces."""
import importlib

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24


@pytest.fixture(scope='module')
def mods(pkg):
    return tuple(importlib.import_module('dcss-auto_amd.' + n) for n in ('losses', 'recurrence', 'optim'))


def rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV).to(dtype)


def far(x):
    """x [a, b, ...] with its first dimension's stride past 2^31 elements."""
    stride = 2 ** 31 + 24
    base = torch.empty(stride * (x.shape[0] - 1) + x[0].numel(), dtype=x.dtype, device=DEV)
    y = base.as_strided(x.shape, (stride, *x[0].contiguous().stride()))
    y.copy_(x)
    return y


def test_loss_far_rows(mods):
    print('[loss] rows past 2^31 elements apart', flush=True)
    L = mods[0]
    logp, old = rand(3, 700, seed=1, dtype=torch.bfloat16), rand(3, 700, seed=2)
    adv, mask = rand(3, seed=3), rand(3, 700, seed=4) > 0
    for level in ('token', 'sequence'):
        want = L.policy_loss_grads(logp, old, adv, mask=mask, level=level)
        got = L.policy_loss_grads(far(logp), old, adv, mask=far(mask.byte()), level=level)
        # the same tokens in sums of 64 bits, whose order may differ
        torch.testing.assert_close(got[0].terms, want[0].terms, rtol=2 * U, atol=1e-12)
        assert torch.equal(got[1], want[1])


@pytest.mark.parametrize('steps', [3, 130])
def test_scan_far_steps(mods, steps):
    print(f'[scan] strides past 2^31 elements {steps}', flush=True)
    R = mods[1]
    x, gate, dh = (rand(3, steps, 70, seed=s, dtype=torch.bfloat16) for s in range(3))     # sequences first
    turn = (lambda t: t) if steps == 3 else (lambda t: t.transpose(0, 1))                # steps or rows far apart
    k = [turn(t) for t in (x, gate, dh)]
    f = turn(far(x)), turn(far(gate)), turn(far(dh))
    want, got = R.gated_scan_fwd(*k[:2]), R.gated_scan_fwd(*f[:2])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    want, got = (R.gated_scan_bwd(t[2], None, t[0], t[1], None, None, r[2]) for t, r in ((k, want), (f, got)))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize('steps', [1, 12])
def test_scan_many_rows(mods, steps):
    print(f'[scan] more rows than a launch takes {steps}', flush=True)
    R = mods[1]
    rows = 2 ** 22 + 37
    x, gate, state = rand(steps, rows, 1), rand(steps, rows, 1, seed=1), rand(rows, 1, seed=2)
    reset = rand(steps, rows, seed=3) > 1
    h, last, marks = R.gated_scan_fwd(x, gate, state, reset)
    dx, dgate, dstate = R.gated_scan_bwd(h, last, x, gate, state, reset, marks)
    for part in (slice(0, 1000), slice(2 ** 22 - 1000, rows)):          # the same rows in a call of their own
        k = x[:, part], gate[:, part], state[part], reset[:, part]
        want = R.gated_scan_fwd(*k)
        assert torch.equal(h[:, part], want[0]) and torch.equal(last[part], want[1])
        want = R.gated_scan_bwd(h[:, part], last[part], *k, want[2])
        assert torch.equal(dx[:, part], want[0]) and torch.equal(dgate[:, part], want[1]) and torch.equal(dstate[part], want[2])


def test_muon_far_elements(mods):
    """A matrix of more than 2^31 elements with one entry of 1 a row, all in different columns: with every singular value
    s = 1 / sqrt(rows), a result is p(s) where an entry is and 0 elsewhere."""
    print('[muon] past 2^31 elements', flush=True)
    O = mods[2]
    rows, cols = 16500, 131072
    u = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    at = torch.randperm(cols, generator=torch.Generator(DEV).manual_seed(1), device=DEV)[:rows]
    r = torch.arange(rows, device=DEV)
    u[r, at] = 1.0
    out = O.orthogonalize(u, steps=2)
    s = rows ** -0.5
    a, b, c = O.NEWTON_SCHULZ
    want = s
    for _ in range(2):
        want = a * want + b * want ** 3 + c * want ** 5
    got = out[r, at]
    # a step rounds X, A and B to fp16 (2^-11 each, of terms that are at most the result here) and the result to bf16 (2^-8)
    assert float((got.double() - want).abs().max()) <= want * (2 ** -8 + 8 * 2 ** -11)
    out[r, at] = 0
    assert all(int(torch.count_nonzero(part)) == 0 for part in out.split(2048))


def test_graph_kept(mods):
    """Gradients of a graph that is kept are the same at each pass, and those handed out stay as they are."""
    L, R, _ = mods
    logp, old, adv = rand(40, 90, seed=1).requires_grad_(), rand(40, 90, seed=2), rand(40, 90, seed=3)
    x, gate = rand(90, 40, 33, seed=4).requires_grad_(), rand(90, 40, 33, seed=5)
    loss = L.policy_loss(logp, old, adv).loss
    h, last = R.gated_scan(x, gate)
    plain = L.policy_loss_grads(logp.detach(), old, adv)[1]
    for out, leaf, by in ((loss, logp, plain), ((h * h.detach()).sum() + last.sum(), x, None)):
        seen = [torch.autograd.grad(f * out, leaf, retain_graph=True)[0] for f in (2.0, 1.0, 2.0, 4.0)]
        assert torch.equal(seen[0], seen[2])
        if by is not None:
            assert torch.equal(seen[1], by) and torch.equal(seen[0], 2 * by) and torch.equal(seen[3], 4 * by)


def test_graphs_share_memory(mods):
    """Two graphs from one pool, replayed in turn, with eager calls between."""
    print('[graphs] one pool', flush=True)
    L, R, O = mods
    logp, old, adv = (rand(300, 90, seed=s) for s in range(3))
    x, gate = rand(900, 2, 64, seed=4), rand(900, 2, 64, seed=5)
    u = [rand(300, 700, seed=6), rand(90, 20, seed=7)]

    def one():
        return L.policy_loss_grads(logp, old, adv, mask=adv > 0)[1], O.orthogonalize(u)[0]

    def two():
        h, last, marks = R.gated_scan_fwd(x, gate)
        return (*R.gated_scan_bwd(h, last, x, gate, None, None, marks)[:2], O.orthogonalize(u[::-1])[0])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(), two()
    torch.cuda.current_stream().wait_stream(side)
    a, b = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(a):
        got_one = one()
    with torch.cuda.graph(b, pool=a.pool()):
        got_two = two()
    for i in range(3):
        for k, t in enumerate((logp, old, adv, x, gate, *u)):
            t.copy_(rand(*t.shape, seed=50 + 10 * i + k))
        for graph, got, f in ((a, got_one, one), (b, got_two, two), (a, got_one, one)):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, f()))


@pytest.mark.parametrize('grad', [False, True])
def test_tangents_are_refused(mods, grad):
    L, R, O = mods
    logp, old, adv = (rand(6, 40, seed=s) for s in range(3))
    x, gate, state = rand(70, 3, 8), rand(70, 3, 8, seed=1), rand(3, 8, seed=2)
    marks = R.gated_scan_fwd(x, gate, state)[2]
    p, step = rand(8, 9), torch.zeros(8, dtype=torch.int32, device=DEV)
    with forward_ad.dual_level():
        dual = lambda a: forward_ad.make_dual(a.clone().requires_grad_(grad), torch.ones_like(a))  # noqa: E731
        with torch.set_grad_enabled(grad):
            calls = [lambda: L.policy_loss(dual(logp), old, adv), lambda: L.policy_loss(logp, old, dual(adv)),
                     lambda: L.policy_loss(logp, old, dual(adv[:, 0])), lambda: L.policy_loss_grads(logp, old, adv, entropy=dual(old)),
                     lambda: R.gated_scan(dual(x), gate), lambda: R.gated_scan(x, dual(gate), state), lambda: R.gated_scan(x, gate, dual(state)),
                     lambda: R.gated_scan_bwd(dual(x), None, x, gate, state, None, marks),
                     lambda: R.gated_scan_bwd(x, dual(state), x, gate, state, None, marks), lambda: O.orthogonalize(dual(p))]
            with torch.no_grad():
                tangent = forward_ad.make_dual(p.clone(), torch.ones_like(p))
            calls += [lambda: O.muon_step([tangent], [p], [torch.zeros_like(p)], step), lambda: O.muon_step([p], [tangent], [torch.zeros_like(p)], step)]
            for k, call in enumerate(calls):
                with pytest.raises(NotImplementedError):
                    call()
                    print('not refused:', k)


def test_transforms_and_traces_are_refused(mods):
    L, R, O = mods
    logp, old, adv = (rand(6, 40, seed=s) for s in range(3))
    x, gate = rand(70, 3, 8), rand(70, 3, 8, seed=1)
    for call, at in ((lambda z: L.policy_loss(z, old, adv).loss, logp), (lambda z: R.gated_scan(z, gate)[0], x), (O.orthogonalize, logp)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(call, (at,), (at,))
        with pytest.raises(RuntimeError, match='trace'):
            torch.jit.trace(call, (at,), check_trace=False)


def test_orthogonalize_takes_the_same_matrix_twice(mods):
    O = mods[2]
    u = rand(60, 100)
    a, b = O.orthogonalize([u, u])
    assert torch.equal(a, b) and torch.equal(a, O.orthogonalize(u)) and a.data_ptr() != b.data_ptr()


def test_orthogonalize_has_no_gradient(mods):
    """A result outside of autograd is not taken for one within it."""
    u = rand(60, 100).requires_grad_()
    assert not mods[2].orthogonalize(u).requires_grad
