"""Launches of kernels that take their arguments as one structure: small calls are bound by the host, so pointers are
plain integers and the constant part of a structure is made once per shape and copied."""
import ctypes as _c

import torch

from . import fl_ops

MAX_THREADS = 2 ** 32 - 1        # of a launch: workgroups · threads of a workgroup


def ptr(t):
    """Address of an operand the kernel writes (None: null)."""
    if t is None or fl_ops._SC is None:
        return None if t is None else t.data_ptr()
    return fl_ops._p(t).value


def ptr_read(t):
    """Address of an operand the kernel only reads (None: null)."""
    if t is None or fl_ops._SC is None:
        return None if t is None else t.data_ptr()
    return fl_ops._pr(t).value


def launch(name, args, ints, device, refusal=None):
    """Calls ``name(&args, *ints, stream)`` on the device's current stream. False where it returned ``refusal``, with
    nothing launched."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = fl_ops._fn(name)(_c.byref(args), *ints, _c.c_void_p(torch._C._cuda_getCurrentRawStream(index)))
    else:
        with torch.cuda.device(device):
            rc = fl_ops._fn(name)(_c.byref(args), *ints, _c.c_void_p(torch._C._cuda_getCurrentRawStream(index)))
    if rc == refusal:
        return False
    fl_ops._check(rc, name)
    return True
