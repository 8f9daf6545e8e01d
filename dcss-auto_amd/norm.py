"""Layer norm over the last dimension, forward and backward (csrc/d1_norm.hip).

`layer_norm` is the differentiable function, `LayerNorm` the module; `layer_norm_fwd` and
`layer_norm_bwd` are the two passes for code that runs without autograd. The weight's and the
bias's gradients are summed over rows in fp32 in a fixed order.
"""
import torch
from torch import nn
from torch.autograd.function import once_differentiable

from .ops import call, is_tracing


def layer_norm_fwd(x, weight=None, bias=None, eps=1e-5):
    """-> (y like x, mean fp32 [...], rstd fp32 [...]): y = (x - mean) * rstd * weight + bias."""
    return call('norm_fwd_alone', x, x, weight, bias, eps)


def layer_norm_bwd(dy, x, weight, bias, mean, rstd):
    """-> (dx, dweight, dbias) from layer_norm_fwd's arguments and its mean and rstd; dweight and
    dbias are None where the weight or the bias is."""
    return call('norm_bwd', x, dy, x, weight, bias, mean, rstd)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = call('norm_fwd', x, x, weight, bias, eps)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return (*layer_norm_bwd(dy, *ctx.saved_tensors), None)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of x [..., width] (fp32, bf16 or fp16; rows of any stride, up to 16,384 elements)
    with an optional weight and bias [width] in fp32 or x's type; statistics in fp32."""
    if is_tracing() or torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return call('norm_fwd', x, x, weight, bias, eps)[0]


class LayerNorm(nn.Module):
    """layer_norm with its parameters; they stay fp32 where the activations are bf16 or fp16 unless
    the module is cast."""

    def __init__(self, width, eps=1e-5, bias=True):
        super().__init__()
        self.width, self.eps = width, eps
        self.weight = nn.Parameter(torch.ones(width))
        self.bias = nn.Parameter(torch.zeros(width)) if bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f'{self.width}, eps={self.eps}, bias={self.bias is not None}'
