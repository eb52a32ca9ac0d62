"""What the modules share to hand torch tensors to the C ABI: addresses, the current stream, checks."""
import ctypes

import torch

from . import _lib

is_capturing = torch._C._cuda_isCurrentStreamCapturing   # what torch.cuda.is_current_stream_capturing() returns

TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def _stream():
    # the address alone: torch.cuda.current_stream() makes an object for it, which took 2.5 us of a call of 8.7 us
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def signature(*tensors):
    """What a call's argument checks and descriptors depend on: equal signatures need neither again."""
    try:
        return [(t.shape, t.stride(), t.dtype, t.get_device()) for t in tensors]
    except AttributeError:
        raise TypeError("CUDA tensors are needed") from None


def stream_on(index, device=torch._C._cuda_getDevice, stream=torch._C._cuda_getCurrentRawStream):
    """The current stream, if device `index` is the current one."""
    if device() != index:
        raise ValueError("the tensors are not on the current device")
    return stream(index)


def _check_tensor(t, name, ndim=None, strided=False):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s: CUDA support only!" % name)   # the reference's assert message
    if t.dtype != torch.float32:
        raise TypeError("%s must be float32" % name)
    if ndim is not None and t.dim() != ndim:
        raise ValueError("%s must be %d-D" % (name, ndim))
    if not strided and not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)


class Workspace:
    """Device memory that a module hands to its calls, grown as they need more.  Each stream has its own, and so has each
    call that is captured into a graph, for as long as the module lives: calls that run at the same time share none."""

    def __init__(self):
        self._of, self._captured = {}, []

    def take(self, nbytes, device, stream=None, capturing=False):
        last = None if capturing else self._of.get(stream)
        if last is None or last.numel() < nbytes or last.device != device:
            size = max(nbytes, 2 * last.numel() if last is not None and last.device == device else 0, 256)
            last = torch.empty(size, dtype=torch.uint8, device=device)
            if capturing:
                self._captured.append(last)
            else:
                self._of[stream] = last
        return last
