"""What the row operators' Python surfaces (tokens.py, norm.py) and the optimizer share: element
types, the view of a tensor as rows, and a call of libd1ops.so on a tensor's device and stream.

The small calls (a minibatch of action logits, a narrow layer) take a few microseconds on the GPU,
so what stands here and in the callers is kept short: plain comparisons, no views, no context
managers on the usual path."""
import torch

from . import _lib

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # D1_FP32, D1_BF16, D1_FP16
# the stream's handle without a Stream object around it (0.1 us against 2.5)
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def type_of(x, name):
    if not x.is_cuda:
        raise ValueError(f'{name} must be a CUDA tensor (there is no CPU fallback)')
    code = TYPES.get(x.dtype)
    if code is None:
        raise ValueError(f'{name} must be fp32, bf16 or fp16, not {x.dtype}')
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f'{name} must have a last dimension of at least one element')
    return code


def as_rows(x):
    """x as [rows, width] with adjacent elements in a row, a view where its strides allow it."""
    width = x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(x.numel() // width, width)
    if width > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x


def like(t, shape, index, name, dtype=torch.float32):
    """t as a contiguous tensor of `dtype` and `shape` on GPU `index`, or an error that names it."""
    if t.dtype != dtype or t.shape != shape or t.get_device() != index:
        raise ValueError(f'{name} must be {dtype} of shape {tuple(shape)} on cuda:{index}, '
                         f'not {t.dtype} of {tuple(t.shape)} on {t.device}')
    return t if t.is_contiguous() else t.contiguous()


def call(function, index, *args):
    """A libd1ops.so entry point on GPU `index` and its current stream (the last argument)."""
    if index == torch.cuda.current_device():
        code = function(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = function(*args, _raw_stream(index))
    if code:
        _lib.check(code, function.__name__)
