"""Layer norm over the last dimension, forward and backward (csrc/d1_norm.hip).

`layer_norm` is the differentiable function, `LayerNorm` the module; `layer_norm_fwd` and
`layer_norm_bwd` are the two passes for code that runs without autograd. The weight's and the
bias's gradients are summed over rows in fp32 in a fixed order.
"""
import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .rows import TYPES, as_rows, call, like, type_of

MAX_WIDTH = 16384


def _check(x, weight, bias):
    """-> (x's type code, the weights' type code, x as rows, weight, bias)."""
    code = type_of(x, 'x')
    width, index, dtype = x.shape[-1], x.get_device(), x.dtype
    if width > MAX_WIDTH:
        raise ValueError(f'x: rows of at most {MAX_WIDTH} elements')
    first = bias if weight is None else weight
    if first is not None:
        dtype = first.dtype
        if dtype != x.dtype and dtype != torch.float32:
            raise ValueError(f"weight and bias must be fp32 or of x's type, not {dtype}")
        if weight is not None:
            weight = like(weight, (width,), index, 'weight', dtype)
        if bias is not None:
            bias = like(bias, (width,), index, 'bias', dtype)
    return code, TYPES[dtype], as_rows(x), weight, bias


def _ptr(t):
    return None if t is None else t.data_ptr()


def layer_norm_fwd(x, weight=None, bias=None, eps=1e-5):
    """-> (y like x, mean fp32 [...], rstd fp32 [...]): y = (x - mean) * rstd * weight + bias."""
    code, wcode, rows, weight, bias = _check(x, weight, bias)
    n, width = rows.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    call(_lib.load_ops().d1_norm_fwd, x.get_device(), rows.data_ptr(), code, n, width, rows.stride(0), _ptr(weight), _ptr(bias),
         wcode, eps, y.data_ptr(), mean.data_ptr(), rstd.data_ptr())
    return y, mean, rstd


def layer_norm_bwd(dy, x, weight, bias, mean, rstd):
    """-> (dx, dweight, dbias) from layer_norm_fwd's arguments and its mean and rstd; dweight and
    dbias are None where the weight or the bias is."""
    code, wcode, rows, weight, bias = _check(x, weight, bias)
    index, shape, (n, width) = x.get_device(), x.shape[:-1], rows.shape
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.get_device() != index:
        raise ValueError(f'dy must be {x.dtype} of shape {tuple(x.shape)} on {x.device}')
    drows = as_rows(dy)
    mean, rstd = like(mean, shape, index, 'mean'), like(rstd, shape, index, 'rstd')
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = None if weight is None else torch.empty_like(weight)
    db = None if bias is None else torch.empty_like(bias)
    L = _lib.load_ops()
    need = 0 if dw is None and db is None else L.d1_norm_work_bytes(n, width, code)
    work = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    call(L.d1_norm_bwd, index, drows.data_ptr(), drows.stride(0), rows.data_ptr(), code, n, width, rows.stride(0),
         _ptr(weight), wcode, mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), _ptr(dw), _ptr(db), _ptr(work), need)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return (*layer_norm_bwd(dy, *ctx.saved_tensors), None)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of x [..., width] (fp32, bf16 or fp16; rows of any stride, up to 16,384 elements)
    with an optional weight and bias [width] in fp32 or x's type; statistics in fp32."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm_fwd(x, weight, bias, eps)[0]


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
