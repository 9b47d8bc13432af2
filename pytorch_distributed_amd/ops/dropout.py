"""Dropout from a counter-based generator: the mask is a function of (seed, step counter, site, element), never stored,
and regenerated in the backward pass (csrc/dropout.hip).  It stands beside the counter-hash draws of the replay
(csrc/replay_kernels.hip): like them it reads its step counter from DEVICE memory, so a captured hipGraph draws a new
mask in every replay once the counter is bumped inside it or between replays.

`dropout(x, p, seed, counter)` is the operator, `CounterDropout` the module the models use (model_params.dropout).
On CPU tensors the same functions run in torch with the same masks, bit for bit.
"""
import ctypes

import torch
import torch.nn as nn

from ._seq import check_floating, differentiable_once, native, ptr, run_on, wants_graph

_M64 = (1 << 64) - 1
_GOLDEN = 0x9E3779B97F4A7C15
_vp, _u32 = ctypes.c_void_p, ctypes.c_uint


class _Args(ctypes.Structure):      # mirrors DropoutArgs in csrc/dropout.hip
    _fields_ = [("x", _vp), ("residual", _vp), ("y", _vp), ("counter", _vp), ("used", _vp), ("seed", ctypes.c_ulonglong),
                ("site", _u32), ("hi", _u32), ("lo", _u32), ("scale", ctypes.c_float), ("n", ctypes.c_longlong)]


def _signed(v):
    v &= _M64
    return v - (1 << 64) if v >> 63 else v


def _mix(z):
    """csrc/seq.h hash_u64 on an int64 tensor (products wrap)."""
    def down(v):
        return (v >> 33) & 0x7FFFFFFF
    z = (z ^ down(z)) * _signed(0xFF51AFD7ED558CCD)
    z = (z ^ down(z)) * _signed(0xC4CEB9FE1A85EC53)
    return z ^ down(z)


def keep_mask(n, p, seed, counter, site=0):
    """The mask of n elements as a bool tensor, in torch (the CPU path, and what the tests compare the kernels with)."""
    hi, lo = _threshold(p)
    g = _signed(_GOLDEN)
    dev = counter.device
    key = _mix(_mix(_signed(seed) + g * (1 + counter)) + _signed(_GOLDEN * (1 + site)))
    words = _mix(key + g * (1 + torch.arange((n + 3) // 4, device=dev)))
    u = torch.stack([(words >> (16 * j)) & 0xFFFF for j in range(4)], 1).reshape(-1)[:n]
    tie = (_mix(_mix(key) + g * (1 + torch.arange(n, device=dev))) >> 32) & 0xFFFFFFFF
    return (u > hi) | ((u == hi) & (tie >= lo))


def _threshold(p):
    thr = min(int(round(p * 2.0 ** 48)), 1 << 48)
    return thr >> 32, thr & 0xFFFFFFFF


def _run(x, residual, p, seed, site, counter, used):
    """y = x scaled where kept (+ residual); used: int64[1] that receives the counter's value on a GPU (None: backward pass)."""
    scale = 1.0 / (1.0 - p) if p < 1.0 else 0.0
    if x.device.type == "cpu":
        keep = keep_mask(x.numel(), p, seed, counter, site).reshape(x.shape)
        y = torch.where(keep, x.float() * scale, torch.zeros(()))
        return (y if residual is None else y + residual.float()).to(x.dtype)
    entry = native("pda_dropout", whole=used is not None)
    hi, lo = _threshold(p)
    y = torch.empty_like(x)
    args = _Args(ptr(x), ptr(residual), ptr(y), ptr(counter), ptr(used), seed & _M64, site, hi, lo, scale, x.numel())
    run_on(x, entry, "dropout", args)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, site, counter):
        x, residual = x.contiguous(), residual.contiguous() if residual is not None else None
        if x.device.type == "cpu":
            used = counter.clone()
            y = _run(x, residual, p, seed, site, used, None)
        else:
            used = torch.empty_like(counter)
            y = _run(x, residual, p, seed, site, counter, used)
        ctx.save_for_backward(used)
        ctx.how = (p, seed, site)
        return y

    @staticmethod
    @differentiable_once
    def backward(ctx, dy):
        used, = ctx.saved_tensors
        dx = _run(dy.contiguous(), None, *ctx.how, used, None) if ctx.needs_input_grad[0] else None
        return dx, (dy if ctx.needs_input_grad[1] else None), None, None, None, None


def dropout(x, p, seed, counter, site=0, residual=None):
    """y = x / (1 - p) where an element is kept, 0 where it is dropped (probability p), + residual; any shape, float32,
    bfloat16 or float16, computed in 32 bits and rounded once.  A dropped element gives 0 even where x is not finite.

    seed      int; the mask is a function of seed, *counter, site and the element's row-major index alone
    counter   int64 tensor of one element on x's device, read when the kernel RUNS (bump it between steps; the backward
              pass uses the value that its forward pass read, whatever the counter holds by then)
    site      0 .. 2^32 - 1: tells apart the dropouts of one step
    residual  added behind the dropout: x's shape, type and device (its gradient is y's)

    p = 1 drops everything; no rounding of p above 2^-48.  Gradients flow to x and residual (not twice)."""
    check_floating(x, "x")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must be in [0, 1], not %r" % p)
    if isinstance(seed, bool) or not isinstance(seed, int) or isinstance(site, bool) or not isinstance(site, int):
        raise ValueError("seed and site must be ints")
    if not 0 <= site < 1 << 32:
        raise ValueError("site must be in [0, 2^32), not %d" % site)
    if not isinstance(counter, torch.Tensor) or counter.dtype != torch.int64 or counter.numel() != 1:
        raise ValueError("counter must be an int64 tensor of one element")
    if counter.device != x.device:
        raise ValueError("counter is on %s, x on %s" % (counter.device, x.device))
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.dtype != x.dtype or residual.shape != x.shape or \
                residual.device != x.device:
            raise ValueError("residual must have x's shape, type and device")
    counter = counter if counter.dim() == 1 else counter.reshape(1)
    if wants_graph(x, residual):
        return _Dropout.apply(x, residual, p, seed, site, counter)
    return _run(x.contiguous(), residual.contiguous() if residual is not None else None, p, seed, site, counter, None)


class CounterDropout(nn.Module):
    """Dropout layer on `dropout`: keeps its own step counter (a buffer that is no part of the state dict) and bumps it
    behind every call that dropped.  Active in training mode and where gradients are recorded, so action selection and
    target values, which run under no_grad, never drop.

    Not for parts of a model that are computed again in the backward pass (activation checkpointing): the second computation
    would read a counter that has gone on, so it is refused.  `dropout` with a counter of the caller's, bumped once per step
    behind the backward pass, gives both computations the same mask.  (For the same check torch.compile breaks its graph here.)"""

    def __init__(self, p, seed=0, site=0):
        super().__init__()
        self.p, self.seed, self.site = float(p), int(seed), int(site)
        if not 0.0 <= self.p <= 1.0:
            raise ValueError("p must be in [0, 1], not %r" % p)
        self.register_buffer("counter", torch.zeros(1, dtype=torch.int64), persistent=False)

    def forward(self, x, residual=None):
        if self.p == 0.0 or not self.training or not torch.is_grad_enabled():
            return x if residual is None else x + residual
        if torch._C._current_graph_task_id() != -1:         # (inside a running backward pass)
            raise RuntimeError("CounterDropout cannot be computed again in a backward pass (activation checkpointing): its "
                               "counter has gone on; use ops.dropout.dropout with a counter bumped once per step")
        y = dropout(x, self.p, self.seed, self.counter, site=self.site, residual=residual)
        self.counter.add_(1)
        return y

    def extra_repr(self):
        return "p=%g, seed=%d, site=%d" % (self.p, self.seed, self.site)
