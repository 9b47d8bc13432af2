"""Rows, lengths and layouts of the sequence-policy operators that lie off the ordinary paths of their kernels (ops/logprob.py,
ops/scan.py, ops/dropout.py), and calls that have to be refused."""
import os
import sys
import weakref

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import sequence_oracle as oracle  # noqa: E402
from test_sequence_ops import FORMS, INF, check_logprob, check_scan, close, np64, on_devices, on_types, rand, rounding, \
    scan_inputs  # noqa: E402

from pytorch_distributed_amd.ops import build, scan  # noqa: E402
from pytorch_distributed_amd.ops._seq import native  # noqa: E402
from pytorch_distributed_amd.ops.dropout import CounterDropout, dropout  # noqa: E402
from pytorch_distributed_amd.ops.logprob import token_logprobs  # noqa: E402
from pytorch_distributed_amd.ops.scan import linear_scan, linear_scan_step  # noqa: E402


# ---- token log-probabilities ---------------------------------------------------------------------------------------
def masked_rows(v, dt, dev, top, fill):
    """Five rows of which a part is left, the rest `fill`; -> (logits, the tokens asked for)"""
    x = torch.full((5, v), fill, dtype=dt)
    live = rand((5, v), torch.float32, "cpu", v, 3.0, top).to(dt)
    where = torch.zeros(5, v, dtype=torch.bool)
    where[0, :200] = True
    where[1, v // 2:v // 2 + 300] = True
    where[2, ::2] = True
    where[3, 7::500] = True
    where[4, v // 3:] = True
    return torch.where(where, live, x).to(dev), torch.tensor([5, v // 2 + 3, 8, 507, v - 1], device=dev)


@on_devices
@on_types
@pytest.mark.parametrize("v", [2500, 20000])
@pytest.mark.parametrize("top", [1e4, 6e4, 1e6])
def test_logprob_rows_masked_with_the_lowest_value(dev, dt, v, top):
    """Large logits among masks: forward and backward pass measure a row's exponents from the same rounded reference."""
    x, tokens = masked_rows(v, dt, dev, min(top, 6e4) if dt == torch.float16 else top, torch.finfo(dt).min)
    check_logprob(x, tokens, k=5)


@on_devices
@on_types
@pytest.mark.parametrize("v", [700, 2500, 20000])
def test_logprob_masks_by_a_low_value_are_masks(dev, dt, v):
    """A mask of a low finite value is a mask of -inf, bit for bit: such rows take the one pass that others take, whose sums run
    in another order than those of a row that is walked again."""
    def run(fill):
        x, tokens = masked_rows(v, dt, dev, 1.0, fill)
        x.requires_grad_()
        o = token_logprobs(x, tokens, top_k=2)          # (every row has two tokens left)
        d, = torch.autograd.grad(o.logprob.sum() + o.entropy.sum() + o.logsumexp.sum(), x)
        return [o.logprob, o.entropy, o.logsumexp, o.top_logprobs, o.top_tokens, d]
    want = run(-INF)
    for fill in (torch.finfo(dt).min, -3e4) + (() if dt == torch.float16 else (-5e8, -1e9, -1e20)):
        for a, b in zip(run(fill), want):
            assert torch.equal(a, b), fill


@on_devices
@pytest.mark.parametrize("v", [2500, 20000])
@pytest.mark.parametrize("around", [-6931471.5, 6931472.0, -6.931472e8, -7.0e5])
def test_logprob_rows_of_large_logits(dev, v, around):
    """Logits whose exponents' references lie on either side of the bounds at which a part or a row changes its form."""
    x = rand((5, v), torch.float32, "cpu", v, 1.0) * torch.tensor([[2.0], [20.0], [200.0], [2000.0], [0.0]]) + around
    x[4, :v // 2] -= 0.5                # whole parts on one side, the row's maximum on the other
    x = x.to(dev)
    tokens = torch.tensor([0, 7, v // 2, v - 1, 0], device=dev)
    leaf = x.clone().requires_grad_()
    out = token_logprobs(leaf, tokens, top_k=3)
    up = [rand((5,), torch.float32, dev, i) for i in range(3)]
    d, = torch.autograd.grad(out[:3], leaf, up)
    want, tol, dx, dtol = oracle.logprob(np64(x), tokens.cpu().numpy(), 1.0, -100, *[np64(t) for t in up])
    for name, got in (("lp", out.logprob), ("ent", out.entropy), ("lse", out.logsumexp)):
        close(got, want[name], tol[name])
    assert torch.equal(out.top_tokens.cpu(), torch.sort(x.cpu(), dim=1, descending=True, stable=True)[1][:, :3])
    # a probability below 2^-126 may be taken as 0: p k with |k| <= |dlse| + |dlp| + |dent| (|logp| + entropy), and at that
    # border |logp| is 88, while p falls faster than |logp| rises behind it
    a, b, c = (np.abs(np64(t)) for t in up)
    flushed = 2.0 ** -126 * (a + c + b * (88 + want["ent"]))
    close(d, dx, dtol + flushed[:, None] + rounding(torch.float32, dx))


@pytest.mark.gpu
@on_types
@pytest.mark.parametrize("v", [1500, 9001])
def test_logprob_gradient_rows_off_the_store_grid(dt, v):
    """Logits and gradient rows of which most are not on the 16-byte grid together."""
    big = rand((4, v + 9), dt, "cuda", 3, 2.0)
    tokens = torch.tensor([0, 2, v // 2, v - 1], device="cuda")
    for off in (1, 3):
        check_logprob(big[:, off:off + v], tokens, T=0.9)


# ---- linear recurrence ---------------------------------------------------------------------------------------------
@on_devices
@pytest.mark.parametrize("second_buffer", [False, True])
def test_a_state_that_a_graph_saved_is_not_overwritten_unseen(dev, second_buffer):
    x, g, state = rand((3, 8), torch.float32, dev, 1), torch.full((3, 8), 0.5, device=dev), rand((3, 8), torch.float32, dev, 2)
    w = torch.ones(3, 8, device=dev, requires_grad=True)
    out = torch.zeros(3, 8, device=dev) if second_buffer else state
    y = (out * w).sum()                 # saves the buffer that the step writes
    before = out._version
    linear_scan_step(x, g, state, state_out=out if second_buffer else None)
    assert out._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():        # tensors without a version counter
        a = state.clone()
        b = linear_scan_step(x, g, a)
        assert torch.equal(a, b)


@on_devices
def test_the_step_refuses_tangents(dev):
    from torch.autograd import forward_ad
    x, g, state = (rand((3, 8), torch.float32, dev, i) for i in range(3))
    want = linear_scan_step(x, g, state.clone())
    with forward_ad.dual_level():
        for i in range(4):
            args = [x, g, state.clone(), torch.zeros_like(state)]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(x))
            with pytest.raises(NotImplementedError):
                linear_scan_step(*args[:3], state_out=args[3])
        assert torch.equal(linear_scan_step(x, g, state), want)


def test_the_recurrence_is_built_with_signed_zeros():
    """A gate that is saturated at 1, or whose step does not exist, is -0 in the kernels; without the sign the state is lost."""
    flags = build.FLAGS + build.SOURCE_FLAGS["scan.hip"]
    assert "-fsigned-zeros" in flags[flags.index("-ffast-math"):]


@on_devices
@on_types
@pytest.mark.parametrize("d", [1, 40])
def test_saturated_gates_keep_the_state(dev, dt, d):
    x = torch.zeros(2, 70, d, dtype=dt, device=dev)
    h0 = rand((2, d), torch.float32, dev, 1)
    n = torch.tensor([70, 3], device=dev)
    for logit in (200.0, INF):
        gate = torch.full_like(x, logit).requires_grad_()
        for mix in (False, True):
            h, last = linear_scan(x, gate, h0, gates="logit", mix=mix, lengths=n)
            assert torch.equal(last, h0) and torch.equal(h[0], h0[0].to(dt).expand(70, d)) and (h[1, 3:] == 0).all()
            grad, = torch.autograd.grad(h.sum() + last.sum(), gate)
            assert torch.equal(grad, torch.zeros_like(grad))
            state = h0.clone()
            assert torch.equal(linear_scan_step(x[:, 0], gate[:, 0].detach(), state, gates="logit", mix=mix), h0.to(dt))
            assert torch.equal(state, h0)


@on_devices
@pytest.mark.parametrize("gates,mix,reverse", FORMS)
@pytest.mark.parametrize("t,d", [(60, 3), (700, 1), (900, 40)])
def test_an_infinite_state_stays_in_its_channel(dev, gates, mix, reverse, t, d):
    x, g = scan_inputs((2, t, d), torch.float32, dev, gates, seed=t)
    n = torch.tensor([t, t - 20], device=dev)
    clean, last = linear_scan(x, g, gates=gates, mix=mix, reverse=reverse, lengths=n)
    y, at, c = x.clone(), t // 2, d - 1
    y[1, at, c] = INF
    h, fin = linear_scan(y, g, gates=gates, mix=mix, reverse=reverse, lengths=n)
    behind = slice(0, at + 1) if reverse else slice(at, t - 20)
    assert not torch.isfinite(h[1, behind, c]).any() and not torch.isfinite(fin[1, c])
    h[1, behind, c], fin[1, c] = clean[1, behind, c], last[1, c]
    assert torch.equal(h, clean) and torch.equal(fin, last)


def returns_like(shape, dev, seed):
    x = rand(shape, torch.float32, "cpu", seed)
    g = torch.full(shape, 0.995)
    g[torch.rand(shape, generator=torch.Generator().manual_seed(seed + 1)) < 1e-3] = 0.0
    return x.to(dev), g.to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("b,t,d", [(1, 57345, 1), (2, 70001, 1), (1, 57400, 3)])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("layout", ["contiguous", "strided"])
def test_scan_one_channel_in_chunks(b, t, d, reverse, layout):
    """Concatenated episodes: fewer than 8 channels and enough steps to be cut; lengths inside a chunk and at its end."""
    x, g = returns_like((b, t, d), "cuda", t + d)
    n = torch.tensor([t - 100, 16384][:b], device="cuda")
    if layout == "strided":
        x, g = (torch.stack([q, q, q], 3)[..., 1] for q in (x, g))
    h0 = rand((b, d), torch.float32, "cuda", 7)
    check_scan(x, g, h0, None if b == 1 else n, reverse=reverse)
    if b == 1:
        check_scan(x, g, None, n, reverse=reverse)


@pytest.mark.gpu
@on_types
def test_scan_one_channel_in_chunks_types(dt):
    x, g = scan_inputs((1, 57345, 1), dt, "cuda", "logit", seed=3)
    check_scan(x, g, rand((1, 1), torch.float32, "cuda", 7), None, "logit", True, True)


@pytest.mark.gpu
@on_types
@pytest.mark.parametrize("gates,mix,reverse", FORMS[1:3])
def test_scan_many_chunks(dt, gates, mix, reverse):
    """More chunks than a workgroup folds at a time, in either direction."""
    t = 40001 if dt == torch.float32 else 20001
    x, g = scan_inputs((1, t, 24), dt, "cuda", gates, seed=t)
    h0 = rand((1, 24), torch.float32, "cuda", 7)
    check_scan(x, g, h0, None, gates, mix, reverse)
    check_scan(x, g, h0, torch.tensor([t - 1111], device="cuda"), gates, mix, reverse)


def test_the_cpu_path_keeps_no_states_that_nothing_reads(monkeypatch):
    states, alive = [], []
    advance = scan._advance

    def watched(h, *args):
        states.append(weakref.ref(h))
        alive.append(sum(r() is not None for r in states))
        return advance(h, *args)
    monkeypatch.setattr(scan, "_advance", watched)
    x = rand((2, 50, 8), torch.float32, "cpu", 1)
    linear_scan(x, torch.full_like(x, 0.5))
    linear_scan(x[..., 0].clone().requires_grad_(), torch.full_like(x[..., 0], 0.5))
    assert len(alive) == 100 and max(alive) <= 2


# ---- dropout -------------------------------------------------------------------------------------------------------
@on_devices
@pytest.mark.parametrize("use_reentrant", [False, True])
def test_dropout_under_activation_checkpointing(dev, use_reentrant):
    from torch.utils.checkpoint import checkpoint
    x = rand((40, 25), torch.float32, dev, 1)
    ctr = torch.full((1,), 6, dtype=torch.int64, device=dev)
    drop = CounterDropout(0.5, seed=3).to(dev)

    def gradient(f, again):
        leaf = x.clone().requires_grad_()
        y = checkpoint(f, leaf, use_reentrant=use_reentrant) if again else f(leaf)
        y.sum().backward()
        return y.detach(), leaf.grad
    for a, b in zip(*(gradient(lambda t: dropout(t * 2, 0.5, 3, ctr).square(), again) for again in (False, True))):
        assert torch.equal(a, b)
    gradient(drop, False)
    with pytest.raises(RuntimeError, match="checkpointing"):
        gradient(lambda t: drop(t * 2).square(), True)
    drop.eval()                         # nothing is dropped, nothing to disagree
    for a, b in zip(*(gradient(lambda t: drop(t * 2).square(), again) for again in (False, True))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_the_dropout_layer_in_a_compiled_function(backend):
    from torch.utils.checkpoint import checkpoint
    torch._dynamo.reset()
    one, two = CounterDropout(0.5, seed=3), CounterDropout(0.5, seed=3)
    x = rand((40, 25), torch.float32, "cpu", 1).requires_grad_()
    f = torch.compile(lambda t: one(t * 2).square(), backend=backend)
    for _ in range(2):
        y, z = f(x), two(x * 2).square()
        assert torch.equal(y, z) and int(one.counter) == int(two.counter)
        for a, b in zip(torch.autograd.grad(y.sum(), x), torch.autograd.grad(z.sum(), x)):
            assert torch.equal(a, b)
    again = torch.compile(lambda t: checkpoint(lambda q: one(q * 2).square(), t, use_reentrant=False), backend=backend)
    with pytest.raises(RuntimeError, match="checkpointing"):
        torch.autograd.grad(again(x).sum(), x)


# ---- together ------------------------------------------------------------------------------------------------------
def calls(dev):
    """-> {name: function of a [4, 60] tensor}"""
    tok, ctr = torch.zeros(4, dtype=torch.int64, device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    gate, state = torch.full((4, 60), 0.5, device=dev), rand((4, 60), torch.float32, dev, 2)
    return {"logprob": lambda t: token_logprobs(t, tok).logprob, "scan": lambda t: linear_scan(t, gate)[0],
            "step": lambda t: linear_scan_step(t, gate, state.clone()), "dropout": lambda t: dropout(t, 0.5, 1, ctr)}


@on_devices
@pytest.mark.parametrize("name", ["logprob", "scan", "step", "dropout"])
@pytest.mark.parametrize("pre_dispatch", [False, True])
def test_recorded_programs(dev, name, pre_dispatch):
    """make_fx: on the CPU the formulas are recorded; a launch cannot be, and is refused."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x, y = calls(dev)[name], rand((4, 60), torch.float32, dev, 0), rand((4, 60), torch.float32, dev, 1)
    if dev == "cuda":
        with pytest.raises(RuntimeError, match="traced program"):
            make_fx(f, pre_dispatch=pre_dispatch)(x)
        f(x)
    else:
        assert torch.equal(make_fx(f, pre_dispatch=pre_dispatch)(x)(y), f(y))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["logprob", "scan", "step", "dropout"])
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_traces(name):
    f, x = calls("cuda")[name], rand((4, 60), torch.float32, "cuda", 0)
    with pytest.raises(RuntimeError, match="traced program"):
        torch.jit.trace(f, (x,), check_trace=False)
    if name == "dropout":       # with a gradient the call is one recorded operation
        traced = torch.jit.trace(f, (x.clone().requires_grad_(),), check_trace=False)
        y = rand((4, 60), torch.float32, "cuda", 1)
        assert torch.equal(traced(y), f(y))


def test_the_library_is_not_handed_to_a_tracer():
    from torch.fx.experimental.proxy_tensor import make_fx

    def f(t):
        native("pda_scan_step")
        return t
    for how in (lambda: torch.jit.trace(f, (torch.zeros(2),), check_trace=False), lambda: make_fx(f)(torch.zeros(2)),
                lambda: make_fx(f, pre_dispatch=True)(torch.zeros(2))):
        with pytest.raises(RuntimeError, match="traced program"):
            how()


# ---- the evaluator's returns ---------------------------------------------------------------------------------------
def test_returns_take_the_steps_of_the_longest_episode(monkeypatch):
    from pytorch_distributed_amd.agents import evaluators
    seen = []

    def seen_scan(x, *args, **kw):
        seen.append(x.shape[1])
        return linear_scan(x, *args, **kw)
    monkeypatch.setattr(evaluators, "linear_scan", seen_scan)
    lengths = [3, 1, 40, 7, 12]
    trace = [(float(i % 5) - 1.0, i + 1 == n, 0.25 * i) for n in lengths for i in range(n)]
    for cut in (0, 2):                  # the last episode ended, or cut short
        steps = trace[:len(trace) - cut]
        want, bias, at = [], [], 0
        for n in lengths[:-1] + [lengths[-1] - cut]:
            g = 0.0
            for r, _, v in reversed(steps[at:at + n]):
                g = r + 0.9 * g
                bias.append(v - g)
            want.append(g)
            at += n
        ret, off = evaluators.returns_report(steps, 0.9)
        # returns below 30, a memory of 10 steps, means of 61 values: 64 half steps of 30
        assert abs(ret - sum(want) / len(want)) < 64 * 30 * 2.0 ** -24
        assert abs(off - sum(bias) / len(bias)) < 64 * 30 * 2.0 ** -24
    assert seen == [40, 40]
