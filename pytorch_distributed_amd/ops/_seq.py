"""What the sequence-policy operators (logprob.py, scan.py, dropout.py) share: element types, native dispatch, errors."""
import contextlib

import torch

from . import lib, native_error

TYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # csrc/seq.h SEQ_*


def check_floating(t, what):
    if not isinstance(t, torch.Tensor) or t.dtype not in TYPE_CODES:
        raise ValueError("%s must be a float32, bfloat16 or float16 tensor, not %s"
                         % (what, t.dtype if isinstance(t, torch.Tensor) else type(t).__name__))
    if t.device.type not in ("cuda", "cpu"):
        raise ValueError("%s is on %s: the operator runs on a GPU (HIP kernels) or on the CPU" % (what, t.device))


def check_int(t, what, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError("%s must be an int32 or int64 tensor" % what)
    if tuple(t.shape) != tuple(shape):
        raise ValueError("%s has shape %s, expected %s" % (what, tuple(t.shape), tuple(shape)))
    if t.device != device:
        raise ValueError("%s is on %s, not on %s" % (what, t.device, device))


def native(name):
    """The C entry `name`; raises when the library is not there (a GPU tensor never falls back to eager torch)."""
    try:
        return getattr(lib(), name)
    except RuntimeError:
        raise RuntimeError("%s on a GPU needs the HIP library: %s" % (name, native_error()))


def ptr(t):
    return t.data_ptr() if t is not None else None


@contextlib.contextmanager
def _other_device(device):
    with torch.cuda.device(device):
        yield


_SAME = contextlib.nullcontext()


def on_device(t):
    """Context in which `t`'s device is the current one (kernels launch on the current device)."""
    return _SAME if t.device.index == torch.cuda.current_device() else _other_device(t.device)


def stream_of(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def launched(rc, name):
    if rc == 0:
        return
    if rc < 0:
        raise ValueError("%s refused its arguments" % name)
    raise RuntimeError("%s: the launch failed with HIP error %d" % (name, rc))
