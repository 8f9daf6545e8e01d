"""gated_scan with finite gates up to the largest that their type holds: z and 1 - z are 0 and 1 exactly, forward and backward."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def values(dtype):
    """Gates of which e^-|gate| is 0 in fp32: past 104; some whose product with log2 e passes fp32's range."""
    top = torch.finfo(dtype).max
    return [g for g in (150.0, 1e4, 1e30, 2.3e38, 2.4e38, 3.3e38, top) if g <= top]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('steps,rows,width', [(1, 3, 70), (7, 3, 70), (40, 2, 130), (70, 2, 65), (600, 1, 70)])
def test_the_state_is_kept(dtype, steps, rows, width):
    """A gate masked with its type's lowest value keeps the state: h and last are it, bit for bit in fp32, and its gradient is the sum."""
    R = importlib.import_module('dcss-auto_amd.recurrence')
    gen = torch.Generator(DEV).manual_seed(steps)
    x = torch.randn(steps, rows, width, generator=gen, device=DEV).to(dtype)
    state = torch.randn(rows, width, generator=gen, device=DEV)
    dh, dlast = torch.ones_like(x), torch.full_like(state, 3.0)
    for value in values(dtype):
        print(f'[scan] gate {-value} {dtype} {steps}', flush=True)
        gate = torch.full_like(x, -value)
        h, last, marks = R.gated_scan_fwd(x, gate, state)
        assert torch.equal(last, state) and torch.equal(h, state.to(dtype).expand_as(h))
        dx, dgate, dstate = R.gated_scan_bwd(dh, dlast, x, gate, state, None, marks)
        # whole numbers up to 603: their sum has no rounding
        assert torch.equal(dstate, torch.full_like(state, 3.0 + steps))
        assert float(dx.abs().max()) == 0 and float(dgate.abs().max()) == 0


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('steps,rows,width', [(1, 3, 70), (40, 2, 130), (600, 1, 70)])
def test_the_state_is_replaced(dtype, steps, rows, width):
    R = importlib.import_module('dcss-auto_amd.recurrence')
    gen = torch.Generator(DEV).manual_seed(steps)
    x, dh = (torch.randn(steps, rows, width, generator=gen, device=DEV).to(dtype) for _ in range(2))
    state = torch.randn(rows, width, generator=gen, device=DEV)
    for value in values(dtype):
        gate = torch.full_like(x, value)
        h, last, marks = R.gated_scan_fwd(x, gate, state)
        assert torch.equal(h, x) and torch.equal(last, x[-1].float())
        dx, dgate, dstate = R.gated_scan_bwd(dh, None, x, gate, state, None, marks)
        assert torch.equal(dx, dh) and float(dgate.abs().max()) == 0 and float(dstate.abs().max()) == 0


def test_masked_steps_among_others():
    """masked_fill with the lowest value: the steps that it leaves give what they give alone."""
    R = importlib.import_module('dcss-auto_amd.recurrence')
    gen = torch.Generator(DEV).manual_seed(3)
    x, gate = (torch.randn(300, 2, 33, generator=gen, device=DEV) for _ in range(2))
    live = torch.rand(300, generator=gen, device=DEV) < 0.3
    h, last = R.gated_scan(x, gate.masked_fill(~live[:, None, None], torch.finfo(torch.float32).min))
    want = torch.zeros(2, 33, dtype=torch.float64, device=DEV)
    z = torch.sigmoid(gate.double())
    size, err = want.abs(), torch.zeros_like(want)
    for t in range(300):
        if live[t]:
            want = (1 - z[t]) * want + z[t] * x[t]
            size = (1 - z[t]) * size + z[t] * x[t].abs()
            # 4 halves of a step for z and 1 - z each, a multiply-add, 2 for a composite's product
            err = (1 - z[t]) * err + 12 * 2.0 ** -24 * size
        assert bool(((h[t].double() - want).abs() <= err + 2.0 ** -24 * want.abs()).all()), t
    assert torch.equal(last, h[-1])


def test_not_finite_stays_not_finite():
    """A NaN gate is still NaN, an infinite one is its limit."""
    R = importlib.import_module('dcss-auto_amd.recurrence')
    for dtype in TYPES:
        x, state = torch.ones(20, 1, 64, device=DEV, dtype=dtype), torch.full((1, 64), 5.0, device=DEV)
        for steps in (1, 20):
            nan = torch.full_like(x[:steps], float('nan'))
            assert bool(R.gated_scan(x[:steps], nan, state)[1].isnan().all())
            low = torch.full_like(x[:steps], -float('inf'))
            assert torch.equal(R.gated_scan(x[:steps], low, state)[1], state)
