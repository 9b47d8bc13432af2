"""What the sequence-policy operators (logprob.py, scan.py, dropout.py) share: element types, native dispatch, errors."""
import ctypes

import torch
from torch.autograd import forward_ad

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


_is_tracing, _dispatch_modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack
_in_dispatch, _PRE_DISPATCH = torch._C._dispatch_tls_is_dispatch_key_included, torch._C.DispatchKey.PreDispatch
_ENTRIES = {}


def _proxied():
    from torch.fx.experimental.proxy_tensor import get_proxy_mode
    return get_proxy_mode() is not None


def native(name, whole=False):
    """The C entry `name`; raises when the library is not there (a GPU tensor never falls back to eager torch), and where a
    tracer (torch.jit.trace, make_fx) records the call: a launch is no torch operation, so the program would hold the outputs'
    allocation and no launch.  whole: an autograd function runs the call, which torch.jit.trace records as one operation."""
    if (_is_tracing() and not whole) or ((_dispatch_modes() or _in_dispatch(_PRE_DISPATCH)) and _proxied()):
        raise RuntimeError("%s on a GPU cannot be recorded into a traced program" % name)
    entry = _ENTRIES.get(name)
    if entry is None:
        try:
            entry = _ENTRIES[name] = getattr(lib(), name)
        except RuntimeError:
            raise RuntimeError("%s on a GPU needs the HIP library: %s" % (name, native_error()))
    return entry


def differentiable_once(backward):
    """torch's once_differentiable, without its wrapper (5 us a call) where no graph of the gradient is asked for."""
    with_graph = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return (with_graph if torch.is_grad_enabled() else backward)(ctx, *grads)
    return run


def wants_graph(*tensors):
    """Whether a call has to go through autograd: a gradient may be asked of it, or tangents are being carried forward (which
    the operators' functions refuse)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return getattr(forward_ad, "_current_level", -1) >= 0


def refuse_tangents(name, *tensors):
    """For operators without an autograd function, which would drop them."""
    if getattr(forward_ad, "_current_level", -1) >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("%s carries no tangents forward" % name)


def ptr(t):
    return t.data_ptr() if t is not None else None


def run_on(t, entry, name, args):
    """entry(args, type code, stream) on t's device and its current stream."""
    index = t.device.index
    if index == torch.cuda.current_device():
        rc = entry(ctypes.byref(args), TYPE_CODES[t.dtype], _raw_stream(index))
    else:       # kernels launch on the current device
        with torch.cuda.device(index):
            rc = entry(ctypes.byref(args), TYPE_CODES[t.dtype], _raw_stream(index))
    if rc != 0:
        launched(rc, name)


def _raw_stream(index):
    return ctypes.c_void_p(torch.cuda.current_stream(index).cuda_stream)


if hasattr(torch._C, "_cuda_getCurrentRawStream"):      # the same handle without building a Stream object (3 us a call)
    def _raw_stream(index):     # noqa: F811
        return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(index))


def launched(rc, name):
    if rc == 0:
        return
    if rc < 0:
        raise ValueError("%s refused its arguments" % name)
    raise RuntimeError("%s: the launch failed with HIP error %d" % (name, rc))
