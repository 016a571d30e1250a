"""What the operators over rows of several types share (``norm``, ``experts``):
calls of the library on a tensor's device, and their checks."""
import torch
from torch.autograd import forward_ad

from . import int8
from .sphops import _native

TYPES = int8.TYPES  # float32, bfloat16, float16
check_rows, rows_view, first_order = int8._check_rows, int8._rows_view, int8.first_order


def address(t):
    return None if t is None else t.data_ptr()


def call(function, device, *args):
    """The entry point on the device's current stream, whichever device is current."""
    if device.index == torch.cuda.current_device():
        _native.check(function(*args, torch._C._cuda_getCurrentRawStream(device.index)))
        return
    with torch.cuda.device(device):
        _native.check(function(*args, torch._C._cuda_getCurrentRawStream(device.index)))


def wants_grad(*tensors):
    """Whether a call goes through its autograd function: for gradients, and
    wherever tensors may hold tangents (whatever the grad mode), which the function
    refuses and a kernel would lose."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
            or forward_ad._current_level >= 0)


def check_weight(t, shape, types, device, what):
    """None, or a contiguous tensor of the given shape, one of the types and the device."""
    if t is None:
        return None
    if t.dtype not in types or t.device != device:
        names = " or ".join(str(d).replace("torch.", "") for d in types)
        raise TypeError(f"{what} must be a {names} tensor on {device}")
    if tuple(t.shape) != tuple(shape):
        raise RuntimeError(f"{what} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()
