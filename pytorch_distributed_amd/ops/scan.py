"""Gated linear recurrence h_t = a_t h_{t-1} + u_t over sequences, its backward pass and its single-token step
(csrc/scan.hip).  It stands beside the n-step return assembly (agents/nstep.py, which walks one episode step by step on the
host): discounted returns are this recurrence with gate = gamma, run backwards, and so is a recurrent layer's memory.
The evaluator's return report (agent_params.evaluate_returns) runs on it.

On CPU tensors the same functions compute the same formulas in torch, step by step.
"""
import ctypes
import functools

import torch

from ._seq import TYPE_CODES, check_floating, check_int, differentiable_once, launched, native, ptr, refuse_tangents, run_on, \
    wants_graph

GATES = ("decay", "logit")
_written = torch._C._increment_version      # torch.autograd.graph.increment_version without its look at the argument's type
_vp, _i64, _int = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int


class _Args(ctypes.Structure):      # mirrors ScanArgs in csrc/scan.hip
    _fields_ = [("x", _vp), ("gate", _vp), ("dh", _vp), ("xs0", _i64), ("xs1", _i64), ("xs2", _i64),
                ("gs0", _i64), ("gs1", _i64), ("gs2", _i64), ("ds0", _i64), ("ds1", _i64), ("ds2", _i64), ("h0", _vp),
                ("dlast", _vp), ("lengths", _vp), ("len64", _int), ("h", _vp), ("last", _vp), ("carry", _vp),
                ("sums", _vp), ("dx", _vp), ("dg", _vp), ("dh0", _vp), ("B", _int), ("T", _int), ("D", _int),
                ("logit", _int), ("mix", _int), ("reverse", _int), ("chunks", _int), ("chunk_len", _int),
                ("carry_len", _int), ("carries", _int)]


class _StepArgs(ctypes.Structure):  # mirrors ScanStepArgs
    _fields_ = [("x", _vp), ("gate", _vp), ("state", _vp), ("state_out", _vp), ("h", _vp), ("xs0", _i64),
                ("xs1", _i64), ("gs0", _i64), ("gs1", _i64), ("ss0", _i64), ("ss1", _i64), ("os0", _i64), ("os1", _i64),
                ("B", _int), ("D", _int), ("logit", _int), ("mix", _int)]


def _gate(g, logit):
    """-> (a, 1 - a) in 32 bits"""
    g = g.float()
    return (torch.sigmoid(g), torch.sigmoid(-g)) if logit else (g, 1 - g)


def _advance(h, x, g, logit, mix):
    a, c = _gate(g, logit)
    x = x.float()
    return _decayed(h, a, c, logit) + (c * x if mix else x)


def _decayed(h, a, c, logit):
    """a h (csrc/scan.hip: from 1 - a where a gate is above 1/2)"""
    return torch.where(c <= 0.5, h - c * h, a * h) if logit else a * h


def _steps(T, n, reverse, dev):
    """Yields, for every step of the recurrence, the position it reads per sequence and whether that step exists."""
    for i in range(T):
        pos = (n - 1 - i).clamp_min(0) if reverse else torch.full_like(n, i)
        yield pos, (i < n)[:, None]


def _forward_torch(x, gate, h0, n, logit, mix, reverse, hist=None):
    """-> (h, last); hist: a list that receives the state in front of every step"""
    B, T, D = x.shape
    row = torch.arange(B)
    h = h0.clone() if h0 is not None else torch.zeros(B, D)
    out = torch.zeros(B, T, D, dtype=x.dtype)
    for pos, on in _steps(T, n, reverse, x.device):
        if hist is not None:
            hist.append(h)
        h = torch.where(on, _advance(h, x[row, pos], gate[row, pos], logit, mix), h)
        out[row, pos] = torch.where(on, h.to(x.dtype), out[row, pos])
    return out, h


def _backward_torch(x, gate, h0, n, logit, mix, reverse, dh, dlast):
    B, T, D = x.shape
    row = torch.arange(B)
    hist = []
    _forward_torch(x, gate, h0, n, logit, mix, reverse, hist)
    dx, dg = torch.zeros(B, T, D, dtype=x.dtype), torch.zeros(B, T, D, dtype=x.dtype)
    carry = dlast.clone() if dlast is not None else torch.zeros(B, D)
    for prev, (pos, on) in reversed(list(zip(hist, _steps(T, n, reverse, x.device)))):
        a, c = _gate(gate[row, pos], logit)
        xv = x[row, pos].float()
        gr = carry + (dh[row, pos].float() if dh is not None else 0.0)
        da = gr * (prev - xv if mix else prev)
        if logit:
            da = da * a * c
        dx[row, pos] = torch.where(on, (gr * c if mix else gr).to(x.dtype), dx[row, pos])
        dg[row, pos] = torch.where(on, da.to(x.dtype), dg[row, pos])
        carry = torch.where(on, _decayed(gr, a, c, logit), carry)
    return dx, dg, carry


@functools.lru_cache(maxsize=1024)
def _plan(B, T, D, code):
    """-> (carries, chunks): how the kernels cut the steps (csrc/scan.hip scan_plan), a function of the sizes"""
    out = (ctypes.c_int * 2)()
    launched(native("pda_scan_plan")(B, T, D, code, ctypes.byref(out, 0), ctypes.byref(out, 4)), "linear_scan")
    return out[0], out[1]


def _lengths(lengths, B, T):
    return torch.full((B,), T) if lengths is None else lengths.long().clamp(0, T)


def _cube(t):
    """[B, T] (or a state [B]) as one channel"""
    return t.unsqueeze(-1) if t is not None else None


def _sizes(x):
    """-> (B, T, D), x's strides and whether it has a channel dimension"""
    return (x.shape, x.stride(), True) if x.dim() == 3 else ((*x.shape, 1), (*x.stride(), 1), False)


def _forward(x, gate, h0, lengths, how, keep):
    """-> (h, last, carry); carry: the states that a backward pass starts from, if `keep`"""
    (B, T, D), xs, wide = _sizes(x)
    if x.device.type == "cpu":
        if wide:
            return (*_forward_torch(x, gate, h0, _lengths(lengths, B, T), *how), None)
        h, last = _forward_torch(_cube(x), _cube(gate), _cube(h0), _lengths(lengths, B, T), *how)
        return h.squeeze(2), last.squeeze(1), None
    entry = native("pda_scan_fwd")
    kw = {"dtype": torch.float32, "device": x.device}
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    last = torch.empty((B, D) if wide else B, **kw)
    carries, chunks = _plan(B, T, D, TYPE_CODES[x.dtype])
    carry = torch.empty(B, carries, D, **kw) if keep else None
    sums = torch.empty(B, chunks, 2, D, **kw) if chunks > 1 else None
    run_on(x, entry, "linear_scan",
           _Args(x.data_ptr(), gate.data_ptr(), None, *xs, *(gate.stride() if wide else (*gate.stride(), 1)), 0, 0, 0, ptr(h0),
                 None, ptr(lengths), lengths is not None and lengths.dtype == torch.int64, h.data_ptr(), last.data_ptr(),
                 ptr(carry), ptr(sums), None, None, None, B, T, D, *how, chunks))
    return h, last, carry


class _LinearScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, lengths, logit, mix, reverse):
        ctx.how = (logit, mix, reverse)
        h, last, carry = _forward(x, gate, h0, lengths, ctx.how, True)
        ctx.save_for_backward(x, gate, h0, lengths, carry)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @differentiable_once
    def backward(ctx, dh, dlast):
        x, gate, h0, lengths, carry = ctx.saved_tensors
        if dh is None and dlast is None:
            return (None,) * 7
        (B, T, D), xs, wide = _sizes(x)
        if x.device.type == "cpu":
            n = _lengths(lengths, B, T)
            if wide:
                dx, dg, dh0 = _backward_torch(x, gate, h0, n, *ctx.how, dh, dlast)
            else:
                dx, dg, dh0 = (t.squeeze(-1) for t in _backward_torch(_cube(x), _cube(gate), _cube(h0), n, *ctx.how,
                                                                      _cube(dh), _cube(dlast)))
        else:
            entry = native("pda_scan_bwd")
            dlast = dlast.contiguous() if dlast is not None else None
            kw = {"dtype": torch.float32, "device": x.device}
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            dg, dh0 = torch.empty_like(dx), torch.empty((B, D) if wide else B, **kw)
            chunks = _plan(B, T, D, TYPE_CODES[x.dtype])[1]
            sums = torch.empty(B, chunks, 2, D, **kw) if chunks > 1 else None
            ds = (0, 0, 0) if dh is None else dh.stride() if wide else (*dh.stride(), 1)
            run_on(x, entry, "linear_scan backward",
                   _Args(x.data_ptr(), gate.data_ptr(), ptr(dh), *xs, *(gate.stride() if wide else (*gate.stride(), 1)), *ds,
                         ptr(h0), ptr(dlast), ptr(lengths), lengths is not None and lengths.dtype == torch.int64, None, None,
                         ptr(carry), ptr(sums), dx.data_ptr(), dg.data_ptr(), dh0.data_ptr(), B, T, D, *ctx.how, chunks))
        return dx, dg, (dh0 if h0 is not None else None), None, None, None, None


def _check_gates(gates):
    if gates not in GATES:
        raise ValueError("gates must be one of %s, not %r" % ("|".join(GATES), gates))
    return int(gates == "logit")


def _same(t, what, like, dtype=None):
    dtype = like.dtype if dtype is None else dtype
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != like.device:
        raise ValueError("%s must be a %s tensor on %s" % (what, dtype, like.device))


def linear_scan(x, gate, h0=None, gates="decay", mix=False, reverse=False, lengths=None):
    """-> (h, last): h_t = a_t h_{t-1} + u_t along dimension 1.

    x, gate    [B, T, D] (or [B, T]: one channel), float32, bfloat16 or float16, of one type; any strides, so a gate
               shared by steps or channels may be passed as an expanded view (its gradient is summed by autograd);
               on a GPU up to 8 million sequences times groups of 32 channels
    gates      "decay": a = gate  |  "logit": a = sigmoid(gate)
    mix        False: u = x  |  True: u = (1 - a) x (a leaky average)
    h0         [B, D] (or [B]) float32 state in front of the first step, None = 0
    reverse    run from the last step to the first (discounted returns: gate = gamma, 0 behind an episode's end)
    lengths    [B] int32 / int64: sequence b is its first lengths[b] steps (clamped to 0 .. T; reverse starts at the last
               of them); the other steps are not read, their h and gradients are 0

    h has x's shape and type and is contiguous; last is the float32 state behind the last step (h0 where a length is 0).
    The state is 32 bits wide throughout.  Gradients flow from h and last to x, gate and h0 (not twice).  Decay gates are
    meant to be within [-1, 1]; with larger ones, products of gates over a few hundred steps can overflow 32 bits and the
    result is then inf or NaN even where the exact one is finite.  A state that became infinite or NaN stays one of the two,
    not always the one that the formula gives, in its own channel and from its own step on (of a sequence whose state is
    infinite, last too)."""
    check_floating(x, "x")
    logit = _check_gates(gates)
    if x.dim() not in (2, 3):
        raise ValueError("x must be [B, T, D] or [B, T], not shape %s" % (tuple(x.shape),))
    _same(gate, "gate", x)
    if gate.shape != x.shape:
        raise ValueError("gate has shape %s, x %s (expand a shared gate)" % (tuple(gate.shape), tuple(x.shape)))
    state = (x.shape[0],) + tuple(x.shape[2:])
    if h0 is not None:
        _same(h0, "h0", x, torch.float32)
        if tuple(h0.shape) != state:
            raise ValueError("h0 has shape %s, expected %s" % (tuple(h0.shape), state))
    if lengths is not None:
        check_int(lengths, "lengths", x.shape[:1], x.device)
        lengths = lengths.contiguous()
    if x.shape[0] * (x.shape[2] if x.dim() == 3 else 1) >= 1 << 31 or x.shape[1] >= 1 << 30:
        raise ValueError("x of shape %s is too large" % (tuple(x.shape),))
    h0 = h0.contiguous() if h0 is not None else None
    how = (logit, int(bool(mix)), int(bool(reverse)))
    if wants_graph(x, gate, h0):
        return _LinearScan.apply(x, gate, h0, lengths, *how)
    return _forward(x, gate, h0, lengths, how, False)[:2]


def _span(t):
    """The addresses [first, behind the last) of a 2-d tensor."""
    first = t.data_ptr()
    if t.is_contiguous():
        return first, first + t.element_size() * t.numel()
    (n0, n1), (s0, s1) = t.shape, t.stride()
    return first, first + t.element_size() * ((n0 - 1) * s0 + (n1 - 1) * s1 + 1 if n0 and n1 else 0)


def linear_scan_step(x, gate, state, gates="decay", mix=False, state_out=None):
    """One step of `linear_scan` for every request of a batch: h = a state + u, returned in x's type and written in 32 bits
    to `state` itself, or to state_out, a second buffer.  Memory that overlaps state, x or gate otherwise than as the same view
    is refused, and so are views that interleave, such as pool[:, 0] and pool[:, 1].

    x, gate [B, D] of one type, state float32 [B, D]; any strides, but no element of the written buffer may be shared
    (an expanded view is refused).  No gradient: h and the written state are no part of a graph, whatever x, gate and state
    are; tangents carried forward are refused."""
    check_floating(x, "x")
    logit = _check_gates(gates)
    if x.dim() != 2:
        raise ValueError("x must be [B, D], not shape %s" % (tuple(x.shape),))
    _same(gate, "gate", x)
    out = state if state_out is None else state_out
    for t, what in ((state, "state"), (out, "state_out")):
        _same(t, what, x, torch.float32)
    for t, what in ((gate, "gate"), (state, "state"), (out, "state_out")):
        if t.shape != x.shape:
            raise ValueError("%s has shape %s, x %s" % (what, tuple(t.shape), tuple(x.shape)))
    refuse_tangents("linear_scan_step", x, gate, state, state_out)
    B, D = x.shape
    if not out.is_contiguous():
        (s0, n0), (s1, n1) = sorted(zip(out.stride(), out.shape))
        if (n0 > 1 and s0 == 0) or (n1 > 1 and s1 < s0 * (n0 - 1) + 1):
            raise ValueError("the written state shares elements between requests or channels (strides %s)" % (out.stride(),))
    first, behind = _span(out)
    for t, what in ((state, "state"), (x, "x"), (gate, "gate")):
        if t is out or (t.data_ptr() == first and t.stride() == out.stride() and t.dtype == out.dtype):
            continue
        a, b = _span(t)
        if a < behind and first < b:
            raise ValueError("the written state overlaps %s in memory without being the same view" % what)
    if x.device.type == "cpu":
        with torch.no_grad():
            h = _advance(state, x, gate, logit, mix)
            out.copy_(h)
            return h.to(x.dtype)
    entry = native("pda_scan_step")
    h = torch.empty(B, D, dtype=x.dtype, device=x.device)
    run_on(x, entry, "linear_scan_step",
           _StepArgs(x.data_ptr(), gate.data_ptr(), state.data_ptr(), out.data_ptr(), h.data_ptr(), *x.stride(),
                     *gate.stride(), *state.stride(), *out.stride(), B, D, logit, bool(mix)))
    _written((out,))            # (behind torch's back: a graph that saved it has to notice)
    return h
