"""A gated linear recurrence over long sequences, forward and backward (csrc/d1_scan.hip).

`gated_scan` is the differentiable function, for whole sequences and for single steps; `gated_scan_fwd` and
`gated_scan_bwd` are the two passes for code that runs without autograd. `policy.MemoryPolicy` is built on it.
"""
import torch
from torch.autograd.function import once_differentiable

from .ops import call


def gated_scan_fwd(x, gate, state=None, reset=None):
    """-> (h, last, marks): gated_scan's results, and the states that the backward pass starts from (None where it
    needs none)."""
    return call('scan_fwd', x, x, gate, state, reset, True)


def gated_scan_bwd(dh, dlast, x, gate, state, reset, marks):
    """-> (dx, dgate, dstate) from gated_scan_fwd's arguments and its marks; dh is like x, dlast like the state, either
    may be None (zero). dstate is None where the state is."""
    return call('scan_bwd', x, dh, dlast, x, gate, state, reset, marks)


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, state, reset):
        h, last, marks = gated_scan_fwd(x, gate, state, reset)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, gate, state, reset, marks)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dlast):
        if dh is None and dlast is None:
            return None, None, None, None
        return (*gated_scan_bwd(dh, dlast, *ctx.saved_tensors), None)


def gated_scan(x, gate, state=None, reset=None):
    """h[t] = (1 - z[t]) h[t-1] + z[t] x[t] with z = sigmoid(gate), along the first dimension -> (h, last).

    x, gate: [steps, rows, width] or [steps, width], fp32, bf16 or fp16 of the same type, any strides (batch-first
    sequences as their transpose(0, 1)). state: fp32 [rows, width] (or [width]), h before the first step (None: zeros).
    reset: bool or uint8 [steps, rows] (or [steps]); where it is true the step starts from zero, whatever was before: an
    episode that begins, or the next of several sequences in a row. h has x's type, last is the fp32 state after the last
    step. A single step is x[None]. States are fp32 throughout. A state that is not finite stays so until a reset (an infinite one
    may become NaN, where the factors of many steps together are under fp32's range)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, gate, state)):
        return _GatedScan.apply(x, gate, state, reset)
    return call('scan_fwd', x, x, gate, state, reset, False)[:2]
