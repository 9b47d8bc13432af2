"""Log-probabilities of given tokens (actions), with entropy and the best alternatives, and their gradient
(csrc/logprob.hip).  It stands beside the fused DQN head and the action head (csrc/rl_kernels.hip: arg-max, Q of the
taken action, loss with its gradient), which cover up to 32 actions; this one reads logits of any vocabulary once.
The torch learner core's conservative loss (agent_params.cql_alpha) runs on it.

On CPU tensors the same function computes the same formulas in torch.
"""
import ctypes
import math
from collections import namedtuple

import torch

from ._seq import check_floating, check_int, differentiable_once, native, ptr, run_on, wants_graph

MAX_TOP = 32        # csrc/logprob.hip LP_MAX_TOP
TokenLogprobs = namedtuple("TokenLogprobs", "logprob, entropy, logsumexp, top_logprobs, top_tokens")

_LOG2E = 1.4426950408889634
_vp, _i64 = ctypes.c_void_p, ctypes.c_longlong


class _Args(ctypes.Structure):      # mirrors LogprobArgs in csrc/logprob.hip
    _fields_ = [("logits", _vp), ("ld", _i64), ("rows", _i64), ("vocab", ctypes.c_int), ("tokens", _vp),
                ("tok64", ctypes.c_int), ("ignore", _i64), ("inv_t", ctypes.c_float), ("c", ctypes.c_float), ("top_k", ctypes.c_int),
                ("logprob", _vp), ("entropy", _vp), ("lse", _vp), ("stat_m", _vp), ("stat_l2", _vp), ("top_lp", _vp),
                ("top_id", _vp), ("d_lp", _vp), ("d_ent", _vp), ("d_lse", _vp), ("d_logits", _vp),
                ("splits", ctypes.c_int), ("part_stat", _vp), ("part_top", _vp)]


def _forward_torch(x, tokens, inv_t, top_k, ignore):
    z = x.float()
    v = z.shape[1]
    live = tokens != ignore
    known = (tokens >= 0) & (tokens < v)
    m = z.amax(1)
    empty = m == -math.inf
    d = (z - torch.where(empty, torch.zeros_like(m), m)[:, None]) * inv_t
    e = torch.exp(d)
    s = e.sum(1)
    ls = torch.where(empty, torch.zeros_like(s), torch.log(s))
    u = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1)
    zero, inf = torch.zeros_like(m), torch.full_like(m, -math.inf)
    tok = torch.where(known, tokens, torch.zeros_like(tokens)).long()
    lp = torch.where(empty, inf, d.gather(1, tok[:, None])[:, 0] - ls)
    lp = torch.where(known, lp, torch.full_like(lp, math.nan))
    ent = torch.where(empty, zero, ls - u / s)
    lse = torch.where(empty, inf, m * inv_t + ls)
    ids = torch.sort(z, dim=1, descending=True, stable=True)[1][:, :top_k]
    top = torch.where(empty[:, None], torch.full_like(ids, -math.inf, dtype=torch.float32), d.gather(1, ids) - ls[:, None])
    dead = ~live[:, None]
    return (torch.where(live, lp, zero), torch.where(live, ent, zero), torch.where(live, lse, zero), m, ls,
            top.masked_fill(dead, 0.0), ids.masked_fill(dead, -1))


def _backward_torch(x, tokens, m, ls, ent, d_lp, d_ent, d_lse, inv_t, ignore):
    zero = torch.zeros_like(m)
    d_lp, d_ent, d_lse = (zero if t is None else t for t in (d_lp, d_ent, d_lse))
    known = (tokens >= 0) & (tokens < x.shape[1])
    off = (tokens == ignore) | (m == -math.inf)
    lp = (x.float() - torch.where(off, zero, m)[:, None]) * inv_t - ls[:, None]
    p = torch.exp(lp)
    k0 = d_lse - d_lp - d_ent * ent
    g = torch.where(p == 0, torch.zeros_like(p), p * (k0[:, None] - d_ent[:, None] * lp))
    tok = torch.where(known, tokens, torch.zeros_like(tokens)).long()[:, None]
    g = g.scatter_add(1, tok, d_lp[:, None]) * inv_t
    g = torch.where(known[:, None], g, torch.full_like(g, math.nan))
    return torch.where(off[:, None], torch.zeros_like(g), g).to(x.dtype)


def _forward(x, tokens, inv_t, top_k, ignore, keep):
    """-> (logprob, entropy, logsumexp, top_logprobs, top_tokens, stat); stat: what a backward pass needs, if `keep`"""
    n, v = x.shape
    if x.device.type == "cpu":
        lp, ent, lse, m, ls, top, ids = _forward_torch(x, tokens, inv_t, top_k, ignore)
        return lp, ent, lse, top, ids, torch.stack([m, ls])
    entry = native("pda_logprob")
    kw = {"dtype": torch.float32, "device": x.device}
    lp, ent, lse = torch.empty(n, **kw), torch.empty(n, **kw), torch.empty(n, **kw)
    stat = torch.empty(2, n, **kw) if keep else None
    top = torch.empty(n, top_k, **kw) if top_k else None
    ids = torch.empty(n, top_k, dtype=torch.int64, device=x.device) if top_k else None
    splits, part, m = 1, 0, stat.data_ptr() if keep else 0
    if v > 1024:
        splits = native("pda_logprob_splits")(_i64(n), v, top_k)
    if splits > 1:      # long rows in parts, joined by a second launch: four floats and top_k keys for each part
        work = torch.empty(n * splits * (2 + top_k), dtype=torch.int64, device=x.device)
        part = work.data_ptr()
    run_on(x, entry, "token_logprobs",
           _Args(x.data_ptr(), x.stride(0), n, v, tokens.data_ptr(), tokens.dtype == torch.int64, ignore, inv_t,
                 inv_t * _LOG2E, top_k, lp.data_ptr(), ent.data_ptr(), lse.data_ptr(), m, m + 4 * n if keep else 0, ptr(top),
                 ptr(ids), None, None, None, None, splits, part, part + 16 * n * splits))
    return lp, ent, lse, top, ids, stat


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tokens, inv_t, top_k, ignore):
        lp, ent, lse, top, ids, stat = _forward(x, tokens, inv_t, top_k, ignore, True)
        ctx.save_for_backward(x, tokens, stat, ent)
        ctx.how = (inv_t, ignore)
        ctx.set_materialize_grads(False)
        if top_k:
            ctx.mark_non_differentiable(top, ids)
            return lp, ent, lse, top, ids
        return lp, ent, lse

    @staticmethod
    @differentiable_once
    def backward(ctx, d_lp, d_ent, d_lse, *_):
        x, tokens, stat, ent = ctx.saved_tensors
        inv_t, ignore = ctx.how
        if not ctx.needs_input_grad[0] or (d_lp is None and d_ent is None and d_lse is None):
            return None, None, None, None, None
        if x.device.type == "cpu":
            return _backward_torch(x, tokens, *stat, ent, d_lp, d_ent, d_lse, inv_t, ignore), None, None, None, None
        entry = native("pda_logprob_bwd")
        d_lp, d_ent, d_lse = (None if t is None else t.contiguous() for t in (d_lp, d_ent, d_lse))
        n, v = x.shape
        dx = torch.empty(n, v, dtype=x.dtype, device=x.device)
        m = stat.data_ptr()
        run_on(x, entry, "token_logprobs backward",
               _Args(x.data_ptr(), x.stride(0), n, v, tokens.data_ptr(), tokens.dtype == torch.int64, ignore, inv_t,
                     inv_t * _LOG2E, 0, None, ent.data_ptr(), None, m, m + 4 * n, None, None, ptr(d_lp), ptr(d_ent),
                     ptr(d_lse), dx.data_ptr(), 1, None, None))
        return dx, None, None, None, None


def token_logprobs(logits, tokens, temperature=1.0, top_k=0, ignore_index=-100):
    """-> TokenLogprobs(logprob, entropy, logsumexp, top_logprobs, top_tokens) of softmax(logits / temperature).

    logits        [..., V] float32, bfloat16 or float16; rows may be strided, a last dimension that is not contiguous is
                  copied.  -inf marks a masked token (probability 0, gradient 0).
    tokens        [...] int32 or int64: the tokens (actions) whose log-probabilities are wanted.  `ignore_index` marks a
                  padded row: its logits are not read, its outputs and gradient are 0, its alternatives' tokens -1.  Any
                  other value outside [0, V) gives NaN, in the log-probability and in the row's gradient.
    temperature   2^-126 .. 2^126;  top_k: 0 .. min(32, V) alternatives, best first, the lower token of equals first

    logprob, entropy and logsumexp (float32, shaped as tokens) are differentiable with respect to logits;
    top_logprobs (float32) and top_tokens (int64), [..., top_k], are not, and are None for top_k = 0.
    A row whose every logit is -inf has logprob and logsumexp -inf, entropy 0 and gradient 0; a row that holds NaN or
    +inf gives NaN.  Everything is computed in 32 bits; the gradient is rounded once to the logits' type."""
    check_floating(logits, "logits")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must have a last dimension of at least one token, not shape %s" % (tuple(logits.shape),))
    check_int(tokens, "tokens", logits.shape[:-1], logits.device)
    temperature = float(temperature)
    if not 2.0 ** -126 <= temperature <= 2.0 ** 126:        # (1 / T is a 32-bit factor)
        raise ValueError("temperature must be in [2^-126, 2^126], not %r" % temperature)
    v = logits.shape[-1]
    if isinstance(top_k, bool) or not isinstance(top_k, int) or not 0 <= top_k <= min(MAX_TOP, v):
        raise ValueError("top_k must be an int in [0, %d], not %r" % (min(MAX_TOP, v), top_k))
    if isinstance(ignore_index, bool) or not isinstance(ignore_index, int) or not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError("ignore_index must be a 64-bit int, not %r" % (ignore_index,))
    lead = tokens.shape
    x = logits.reshape(-1, v) if logits.dim() != 2 else logits
    if x.stride(1) != 1 and v > 1:
        x = x.contiguous()
    tokens = tokens.reshape(-1).contiguous()
    if wants_graph(x):
        out = _TokenLogprobs.apply(x, tokens, 1.0 / temperature, top_k, ignore_index)
    else:
        out = _forward(x, tokens, 1.0 / temperature, top_k, ignore_index, False)[:5 if top_k else 3]
    if len(lead) != 1:
        out = [t.reshape(lead) for t in out[:3]] + [t.reshape(lead + (top_k,)) for t in out[3:]]
    return TokenLogprobs(*out) if top_k else TokenLogprobs(*out, None, None)
