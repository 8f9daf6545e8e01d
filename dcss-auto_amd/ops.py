"""The call into libd1ops.so that tokens.py, norm.py and optim.py share.

The small calls (a minibatch of action logits, a narrow layer) take a few microseconds on the GPU, so
arguments are checked and outputs made on the C++ side (csrc/d1_ops_torch.cpp), and what stands
here is kept short."""
import torch

from . import _lib

# the stream's handle without a Stream object around it (0.1 us against 2.5)
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)
# whether torch.jit.trace is recording (0.09 us against 0.19)
is_tracing = getattr(torch._C, '_is_tracing', None) or torch.jit.is_tracing


def call(name, x, *args):
    """An operator's C++ call with x's GPU as the current device and its current stream."""
    function = getattr(_lib.load_ops_torch(), name)
    index = x.get_device()
    if index < 0:
        raise ValueError('the operators take CUDA tensors (there is no CPU fallback)')
    if index == torch.cuda.current_device():
        return function(*args, _raw_stream(index))
    with torch.cuda.device(index):
        return function(*args, _raw_stream(index))
