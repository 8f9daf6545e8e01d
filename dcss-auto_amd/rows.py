"""What the row operators' Python surfaces (tokens.py, norm.py) share: element types, the view of a
tensor as rows, and the stream a call runs on."""
import torch

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # D1_FP32, D1_BF16, D1_FP16


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


def like(t, shape, device, name, dtype=torch.float32):
    """t as a contiguous tensor of `dtype` and `shape` on `device`, or an error that names it."""
    if t.dtype != dtype or t.shape != shape or t.device != device:
        raise ValueError(f'{name} must be {dtype} of shape {tuple(shape)} on {device}, '
                         f'not {t.dtype} of {tuple(t.shape)} on {t.device}')
    return t.contiguous()


class on_device:
    """Makes a tensor's device the current one for a launch and gives its current stream."""

    def __init__(self, device):
        self.index, self.guard = device.index, None

    def __enter__(self):
        if self.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *error):
        if self.guard is not None:
            self.guard.__exit__(*error)
