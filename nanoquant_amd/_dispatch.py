"""When a call may run a kernel of the HIP library directly, and how it is launched."""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib


def only_eager(*tensors) -> bool:
    """Whether a kernel may take the tensors' memory: nothing traces, transforms or differentiates them."""
    for t in tensors:
        if type(t) is not torch.Tensor and type(t) is not nn.Parameter:
            return False
    if torch.compiler.is_compiling() or torch.jit.is_tracing() or torch._C._len_torch_dispatch_stack() > 0:
        return False
    if torch._C._functorch.peek_interpreter_stack() is not None or torch.autograd.forward_ad._current_level >= 0:
        return False
    return not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors))


def only_eager_many(many, *tensors) -> bool:
    """:func:`only_eager` of a list as well: for 64 tensors 4 us instead of 9, more than what the kernel takes."""
    if not set(map(type, many)) <= {torch.Tensor, nn.Parameter} or not only_eager(*tensors):
        return False
    return not (torch.is_grad_enabled() and any(t.requires_grad for t in many))


def launch(what, fn, x, *args) -> None:
    """``fn(*args, stream)`` on the device of x and its current stream. A small call is bound by this path: torch's device
    guard and stream object took three of eleven microseconds."""
    index = x.get_device()
    if index == torch.cuda.current_device():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, what)
