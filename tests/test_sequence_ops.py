"""Token log-probabilities, linear recurrence and counter-based dropout (ops/logprob.py, ops/scan.py, ops/dropout.py)
against their 64-bit definitions (sequence_oracle.py), on the CPU path and on the HIP kernels."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import sequence_oracle as oracle  # noqa: E402

from pytorch_distributed_amd.ops.dropout import CounterDropout, dropout, keep_mask  # noqa: E402
from pytorch_distributed_amd.ops.logprob import token_logprobs  # noqa: E402
from pytorch_distributed_amd.ops.scan import linear_scan, linear_scan_step  # noqa: E402

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = math.inf
on_devices = pytest.mark.parametrize("dev", DEVICES)
on_types = pytest.mark.parametrize("dt", TYPES, ids=["fp32", "bf16", "fp16"])


def np64(t):
    return t.detach().cpu().double().numpy()


def rounding(dt, x):
    return oracle.half_step(torch.finfo(dt).eps, x, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps)


def close(got, want, tol):
    got = np64(got) if isinstance(got, torch.Tensor) else got
    assert got.shape == want.shape, (got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), "NaN in different places"
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)]), "infinities differ"
    bad = fin & ~(np.abs(got - np.where(fin, want, 0)) <= tol)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError("%d of %d off; first at %s: %r, exact %r, tolerance %r"
                             % (bad.sum(), bad.size, i, got[i], want[i], np.broadcast_to(tol, want.shape)[i]))


def rand(shape, dt, dev, seed, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dt).to(dev)


# ---- token log-probabilities ---------------------------------------------------------------------------------------
def check_logprob(logits, tokens, T=1.0, k=0, ignore=-100, grads=True, seed=0):
    leaf = logits.detach().requires_grad_(grads)
    out = token_logprobs(leaf, tokens, temperature=T, top_k=k, ignore_index=ignore)
    x, n = np64(logits), logits.shape[0]
    g = np.random.RandomState(seed)
    up = [g.randn(n).astype(np.float32) for _ in range(3)]
    want, tol, dx, dtol = oracle.logprob(x, tokens.cpu().numpy(), T, ignore, *[u.astype(np.float64) for u in up])
    for name, got in (("lp", out.logprob), ("ent", out.entropy), ("lse", out.logsumexp)):
        assert got.dtype == torch.float32
        close(got, want[name], tol[name])
    if grads:
        d, = torch.autograd.grad((out.logprob, out.entropy, out.logsumexp), leaf,
                                 [torch.from_numpy(u).to(logits.device) for u in up])
        assert d.dtype == logits.dtype
        close(d, dx, dtol + rounding(logits.dtype, np.nan_to_num(dx)))
    if k:
        live = tokens.cpu().numpy() != ignore
        ids = oracle.top(x[live], k)
        assert out.top_tokens.dtype == torch.int64
        assert np.array_equal(out.top_tokens.cpu().numpy()[live], ids)
        assert (out.top_tokens.cpu().numpy()[~live] == -1).all()
        lp = np64(out.top_logprobs)[live]
        for j in range(k):
            w, t, _, _ = oracle.logprob(x[live], ids[:, j], T, ignore)
            close(lp[:, j], w["lp"], t["lp"])
    else:
        assert out.top_tokens is None and out.top_logprobs is None


@on_devices
@on_types
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (3, 2, 2), (128, 6, 0), (5, 18, 3), (7, 63, 5), (2, 64, 32), (9, 65, 8),
                                   (4, 255, 20), (3, 513, 1), (66, 1024, 0), (5, 1025, 7), (2, 4099, 20), (3, 9001, 32)])
def test_logprob_sizes(dev, dt, n, v, k):
    g = torch.Generator().manual_seed(n * 1000 + v)
    tokens = torch.randint(0, v, (n,), generator=g).to(dev)
    check_logprob(rand((n, v), dt, dev, v, 2.5), tokens, T=0.7, k=k)
    check_logprob(rand((n, v), dt, dev, v + 1, 0.1), tokens.int(), T=1.0, k=k)


@pytest.mark.gpu
def test_logprob_large_tensors_equal_their_parts():
    x = torch.empty(2048, 32000, dtype=torch.bfloat16, device="cuda").normal_() * 2       # 131 MB: stores past the caches
    tok = torch.randint(0, 32000, (2048,), device="cuda")

    def run(sl):
        leaf = x[sl].detach().requires_grad_()
        o = token_logprobs(leaf, tok[sl])
        d, = torch.autograd.grad(o.logprob.sum() + o.entropy.sum(), leaf)
        return o.logprob.detach(), o.entropy.detach(), d
    whole = run(slice(None))
    for a, b in zip(whole, run(slice(512, 1536))):      # (no split of the rows in either)
        assert torch.equal(a[512:1536], b)


@pytest.mark.gpu
def test_dropout_large_tensors():
    n = 50 * (1 << 20) + 16         # 100 MB: stores past the caches
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = dropout(x, 0.5, 9, counter_at(2, "cuda"), residual=x)
    for at in (0, 1 << 20, n - 4096):
        want = 1 + 2 * oracle.keep_mask(range(at, at + 4096), 0.5, 9, 2, 0).astype(np.float64)
        assert np.array_equal(np64(y[at:at + 4096]), want)


@pytest.mark.gpu
@on_types
@pytest.mark.parametrize("n,v,k", [(1, 131072, 20), (61, 50257, 5), (2, 200003, 32), (300, 3001, 0), (1030, 2048, 4)])
def test_logprob_large(dt, n, v, k):
    g = torch.Generator().manual_seed(v)
    tokens = torch.randint(0, v, (n,), generator=g).cuda()
    check_logprob(rand((n, v), dt, "cuda", v, 3.0), tokens, T=1.3, k=min(k, 8) if n > 100 else k)


@on_devices
@on_types
@pytest.mark.parametrize("v", [6, 130, 2500, 20000])
def test_logprob_special_rows(dev, dt, v):
    low = torch.finfo(dt).min
    x = rand((12, v), dt, dev, 5, 2.0)
    x[0, :] = -INF                       # nothing is left
    x[1, :] = -INF
    x[1, v // 2] = 1.5                   # one token is left
    x[2, 1:] = -INF                      # ... the taken one
    x[3, :] = low                        # masks of the type's lowest value: all equal
    x[4, 1:] = low
    x[5, 3] = INF
    x[6, 4] = float("nan")
    x[7, :] = float("nan")               # ignored: not read
    x[8, ::2] = -INF
    x[9, :] = 0.0
    x[9, ::3] = -0.0                     # equal to +0: the lower index first
    x[10, :] = -INF
    x[10, 0] = float("nan")
    tokens = torch.tensor([0, 1, 0, 2, 0, 0, 1, -100, 1, 5, 2, 3], device=dev)
    check_logprob(x, tokens, T=1.0, k=min(v, 5))
    check_logprob(x, tokens, T=2.0, k=0)


@on_devices
def test_logprob_token_outside_the_vocabulary(dev):
    x = rand((4, 9), torch.float32, dev, 1)
    for dt in (torch.int32, torch.int64):
        check_logprob(x, torch.tensor([9, -1, 3, -7], device=dev, dtype=dt), ignore=-7)
    check_logprob(x, torch.tensor([1 << 40, -(1 << 40), 3, 8], device=dev))     # (no low 32 bits of either are used)


@on_devices
@on_types
@pytest.mark.parametrize("order", ["up", "down", "equal", "ties"])
@pytest.mark.parametrize("v,k", [(300, 8), (5000, 32)])
def test_logprob_alternatives_in_hard_orders(dev, dt, order, v, k):
    ramp = torch.linspace(-4, 4, v)
    row = {"up": ramp, "down": ramp.flip(0), "equal": torch.ones(v), "ties": (torch.arange(v) * 7919 % 11).float()}[order]
    x = row.to(dt).expand(3, v).contiguous().to(dev)
    check_logprob(x, torch.zeros(3, dtype=torch.int64, device=dev), k=k, grads=False)


@on_devices
@on_types
@pytest.mark.parametrize("order", ["up", "down", "equal", "ties", "steps", "masked", "nearly empty"])
@pytest.mark.parametrize("v,k", [(20003, 32), (8192, 5)])
def test_logprob_alternatives_in_hard_orders_of_split_rows(dev, dt, order, v, k):
    """Rows cut into parts: more equal values, or values above a part's limit, than a wave can order at once; parts with fewer
    tokens left than alternatives are asked for."""
    i = torch.arange(v)
    row = {"up": torch.linspace(-4, 4, v), "down": torch.linspace(4, -4, v), "equal": torch.ones(v), "ties": (i * 7919 % 11).float(),
           "steps": (i // 700).float(), "masked": torch.where(i % 300 == 7, i / v, torch.full((v,), -INF)),
           "nearly empty": torch.where((i == 3) | (i == v - 1), torch.ones(v), torch.full((v,), -INF))}[order]
    x = row.to(dt).expand(3, v).contiguous().to(dev)
    check_logprob(x, torch.tensor([3, 7, v - 1], device=dev), k=k, grads=False)


@on_devices
@on_types
def test_logprob_strides_and_shapes(dev, dt):
    big = rand((10, 1000), dt, dev, 3, 2.0)
    tokens = torch.arange(5, device=dev)
    check_logprob(big[:5, 3:700], tokens, k=4)                  # rows start off the 16-byte grid
    check_logprob(big[::2, 1:130], tokens, k=4)
    check_logprob(big[:1, :600].expand(5, 600), tokens, k=4, grads=False)       # one row, read five times
    check_logprob(big[:, :5].t(), tokens, k=4, grads=False)     # not contiguous: copied
    x = rand((2, 3, 40), dt, dev, 4)
    tok = torch.randint(0, 40, (2, 3), generator=torch.Generator().manual_seed(1)).to(dev)
    a, b = token_logprobs(x, tok, top_k=2), token_logprobs(x.reshape(6, 40), tok.reshape(6), top_k=2)
    assert a.logprob.shape == (2, 3) and a.top_tokens.shape == (2, 3, 2)
    for p, q in zip(a, b):
        assert torch.equal(p.reshape(q.shape), q)
    one = token_logprobs(x[0, 0], tok[0, 0])
    assert one.logprob.shape == () and torch.equal(one.entropy, a.entropy[0, 0])
    empty = token_logprobs(x[:0, 0], tok[:0, 0], top_k=2)
    assert empty.logprob.shape == (0,) and empty.top_tokens.shape == (0, 2)


@on_devices
def test_logprob_partial_and_broadcast_gradients(dev):
    x = rand((6, 50), torch.float32, dev, 9).requires_grad_()
    tok = torch.arange(6, device=dev)
    for pick in ("logprob", "entropy", "logsumexp"):
        d, = torch.autograd.grad(getattr(token_logprobs(x, tok), pick).sum(), x)      # a stride-0 gradient
        ref = torch.log_softmax(x.double(), 1)
        val = {"logprob": ref.gather(1, tok[:, None]).sum(), "entropy": -(ref.exp() * ref).sum(),
               "logsumexp": torch.logsumexp(x.double(), 1).sum()}[pick]
        want, = torch.autograd.grad(val, x)
        close(d, np64(want), 1e-6)      # values below 1, 50 terms: under 16 half steps
    # expanded rows: autograd adds the rows' gradients
    row = x.detach()[:1].clone().requires_grad_()
    d, = torch.autograd.grad(token_logprobs(row.expand(6, 50), tok).logprob.sum(), row)
    p = torch.softmax(row.detach().double(), 1)
    want = torch.zeros(1, 50, dtype=torch.float64, device=dev)
    want[0, :6] = 1
    close(d, np64(want - 6 * p), 6e-6)


@on_devices
def test_logprob_gradient_against_differences(dev):
    x = rand((3, 11), torch.float32, dev, 12)
    tok = torch.tensor([0, 4, 10], device=dev)
    leaf = x.clone().requires_grad_()

    def f(z):
        o = token_logprobs(z, tok, temperature=0.8)
        return o.logprob.sum() + 0.3 * o.entropy.sum() + 0.1 * o.logsumexp.sum()

    d, = torch.autograd.grad(f(leaf), leaf)
    h = 2.0 ** -6       # central: h^2 f''' / 6 < 2^-12 (1 / 0.8)^3 and the sums' rounding 2^-20 / h
    for i in range(3):
        for j in range(11):
            e = torch.zeros_like(x)
            e[i, j] = h
            assert abs(float(f(x + e) - f(x - e)) / (2 * h) - float(d[i, j])) < 1e-3


@on_devices
def test_logprob_refusals(dev):
    x, t = rand((4, 8), torch.float32, dev, 0), torch.zeros(4, dtype=torch.int64, device=dev)
    for args, kw in (((x.double(), t), {}), ((x.int(), t), {}), ((x, t.float()), {}), ((x, t[:3]), {}), ((x, t[:, None]), {}),
                     ((x, t), {"temperature": 0.0}), ((x, t), {"temperature": -1.0}), ((x, t), {"temperature": INF}),
                     ((x, t), {"temperature": math.nan}), ((x, t), {"top_k": 9}), ((x, t), {"top_k": -1}),
                     ((x, t), {"top_k": 1.0}), ((x[:, :0], t), {}), ((x, t), {"ignore_index": 1 << 63}),
                     ((x, t), {"ignore_index": 0.5}), ((rand((4, 40), torch.float32, dev, 0), t), {"top_k": 33}),
                     ((x, t.to("meta")), {}), ((x.to("meta"), t.to("meta")), {})):
        with pytest.raises(ValueError):
            token_logprobs(*args, **kw)


@on_devices
@pytest.mark.parametrize("v", (8, 2000))
def test_logprob_temperatures_at_the_borders(dev, v):
    """1 / T is a 32-bit factor: temperatures whose 1 / T or log2(e) / T leaves the normal numbers are refused."""
    x, t = torch.zeros(2, v, device=dev), torch.tensor([3, 4], device=dev)
    x[:, 3] = 1.0
    for T in (2.0 ** -127, 1e-39, 2.0 ** 127, 1e300):
        with pytest.raises(ValueError):
            token_logprobs(x, t, temperature=T)
    hot = token_logprobs(x, t, temperature=2.0 ** 126).logprob
    assert (hot + math.log(v)).abs().max() < 4 * 2.0 ** -24 * math.log(v)       # a log and one product, each within an ulp
    cold = token_logprobs(x, t, temperature=2.0 ** -126)
    assert cold.logprob[0] == 0 and cold.logsumexp[0] == 2.0 ** 126 and cold.entropy.tolist() == [0.0, 0.0]
    assert abs(float(cold.logprob[1]) / 2.0 ** 126 + 1) < 4 * 2.0 ** -24        # (two roundings, c's and that of c ln 2)


# ---- linear recurrence ---------------------------------------------------------------------------------------------
def check_scan(x, gate, h0=None, lengths=None, gates="decay", mix=False, reverse=False, seed=0, grads=True):
    dt = x.dtype
    lx, lg = x.detach().requires_grad_(grads), gate.detach().requires_grad_(grads)
    lh = h0.detach().requires_grad_(grads) if h0 is not None else None
    h, last = linear_scan(lx, lg, lh, gates=gates, mix=mix, reverse=reverse, lengths=lengths)
    assert h.dtype == dt and last.dtype == torch.float32 and h.is_contiguous()
    dh = rand(x.shape, dt, x.device, seed + 100)
    dl = rand(last.shape, torch.float32, x.device, seed + 101)
    flat = x.dim() == 2

    def cube(t):
        return None if t is None else (np64(t)[..., None] if flat else np64(t))

    want = oracle.scan(cube(x), cube(gate), cube(h0), lengths.cpu().numpy() if lengths is not None else None,
                       gates == "logit", mix, reverse, cube(dh), cube(dl))
    got = {"h": h, "last": last}
    if grads:
        leaves = [lx, lg] + ([lh] if lh is not None else [])
        res = torch.autograd.grad((h, last), leaves, (dh, dl))
        got.update(dx=res[0], dg=res[1])
        if lh is not None:
            got["dh0"] = res[2]
    for name, t in got.items():
        w, tol = want[name]
        if flat:
            w, tol = w[..., 0], tol[..., 0]
        try:
            close(t, w, tol + rounding(t.dtype, w))
        except AssertionError as exc:
            raise AssertionError("%s: %s" % (name, exc))
    return h, last


def scan_inputs(shape, dt, dev, gates, seed=0, spread=1.5, shift=2.0):
    gate = rand(shape, torch.float32, "cpu", seed + 1, spread, shift)
    if gates == "decay":
        gate = torch.sigmoid(gate)
    return rand(shape, dt, dev, seed), gate.to(dt).to(dev)


FORMS = [("decay", False, False), ("decay", True, True), ("logit", False, True), ("logit", True, False)]


@on_devices
@on_types
@pytest.mark.parametrize("gates,mix,reverse", FORMS)
@pytest.mark.parametrize("b,t,d", [(1, 1, 1), (2, 3, 5), (3, 17, 8), (1, 65, 33), (2, 130, 64), (1, 513, 12), (2, 259, 40)])
def test_scan_sizes(dev, dt, gates, mix, reverse, b, t, d):
    x, g = scan_inputs((b, t, d), dt, dev, gates, seed=t)
    check_scan(x, g, rand((b, d), torch.float32, dev, 7), None, gates, mix, reverse)
    check_scan(x, g, None, None, gates, mix, reverse)


@on_devices
@on_types
@pytest.mark.parametrize("b,t", [(1, 1), (3, 7), (2, 64), (5, 257), (2, 1000), (70, 33)])
def test_scan_one_channel(dev, dt, b, t):
    for gates, mix, reverse in FORMS:
        x, g = scan_inputs((b, t), dt, dev, gates, seed=t)
        check_scan(x, g, rand((b,), torch.float32, dev, 7), None, gates, mix, reverse)


@pytest.mark.gpu
@on_types
@pytest.mark.parametrize("gates,mix,reverse", FORMS)
@pytest.mark.parametrize("b,t,d", [(1, 5003, 24), (2, 2049, 64), (1, 3000, 200), (3, 1031, 7), (1, 4097, 3), (2, 12500, 1)])
def test_scan_long(dt, gates, mix, reverse, b, t, d):
    x, g = scan_inputs((b, t, d), dt, "cuda", gates, seed=t)
    check_scan(x, g, rand((b, d), torch.float32, "cuda", 7), None, gates, mix, reverse)
    n = torch.tensor([t - 1, 0, t // 3][:b], device="cuda")
    check_scan(x, g, rand((b, d), torch.float32, "cuda", 7), n, gates, mix, reverse)


@on_devices
@on_types
@pytest.mark.parametrize("d", [5, 33, 64])
def test_scan_every_form(dev, dt, d):
    """Each combination of gates, mixing and direction, whole tiles and parts, with and without 16-byte accesses."""
    for gates in ("decay", "logit"):
        for mix in (False, True):
            for reverse in (False, True):
                x, g = scan_inputs((2, 70, d), dt, dev, gates, seed=d)
                check_scan(x, g, rand((2, d), torch.float32, dev, 7), torch.tensor([70, 64], device=dev), gates, mix, reverse)


@pytest.mark.gpu
@pytest.mark.parametrize("gates,mix,reverse", FORMS)
def test_scan_large_tensors_equal_their_parts(gates, mix, reverse):
    """Above 96 MB stores go past the caches; 48 sequences at once and 8 at a time are the same arithmetic."""
    shape = (48, 520, 2048)
    x = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_()
    g = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_() * 1.5 + 2
    if gates == "decay":
        g = torch.sigmoid(g)
    n = torch.arange(48, device="cuda") * 11 + 3
    dh = torch.empty_like(x).normal_()

    def run(sl):
        leaves = [t[sl].detach().requires_grad_() for t in (x, g)]
        h, last = linear_scan(*leaves, gates=gates, mix=mix, reverse=reverse, lengths=n[sl])
        return (h.detach(), last.detach()) + torch.autograd.grad((h, last), leaves, (dh[sl], torch.ones_like(last)))
    whole = run(slice(None))
    for i in range(0, 48, 8):
        for a, b in zip(whole, run(slice(i, i + 8))):
            assert torch.equal(a[i:i + 8], b)


@on_devices
@on_types
@pytest.mark.parametrize("gates,mix,reverse", FORMS)
@pytest.mark.parametrize("d", [1, 3, 40])
def test_scan_lengths(dev, dt, gates, mix, reverse, d):
    x, g = scan_inputs((6, 45, d), dt, dev, gates, seed=2)
    h0 = rand((6, d), torch.float32, dev, 8)
    for kind in (torch.int32, torch.int64):
        n = torch.tensor([45, 0, 1, 44, 13, 2], device=dev, dtype=kind)
        for i, v in enumerate(n.tolist()):      # behind a sequence's end nothing is read
            x[i, v:] = float("nan")
            g[i, v:] = float("nan")
        h, last = linear_scan(x, g, h0, gates=gates, mix=mix, reverse=reverse, lengths=n)
        assert torch.isfinite(h.float()).all() and torch.equal(last[1], h0[1])
        lx, lg = x.clone().requires_grad_(), g.clone().requires_grad_()
        y, fin = linear_scan(lx, lg, h0, gates=gates, mix=mix, reverse=reverse, lengths=n)
        dh = torch.full_like(y, 1.0)
        for i, v in enumerate(n.tolist()):
            dh[i, v:] = float("nan")
        for grad in torch.autograd.grad((y, fin), (lx, lg), (dh, torch.ones_like(fin))):
            assert torch.isfinite(grad.float()).all()
            for i, v in enumerate(n.tolist()):
                assert (grad[i, v:] == 0).all() and (h[i, v:] == 0).all()
        clean = [torch.nan_to_num(t.float()).to(dt) for t in (x, g)]
        check_scan(*clean, h0, n, gates, mix, reverse)
    out_of_range = torch.tensor([99, -5, 1, 44, 13, 2], device=dev)     # clamped to 0 .. T
    a = linear_scan(*clean, h0, gates=gates, mix=mix, reverse=reverse, lengths=out_of_range)
    b = linear_scan(*clean, h0, gates=gates, mix=mix, reverse=reverse, lengths=out_of_range.clamp(0, 45))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@on_devices
def test_scan_gates_at_the_borders(dev):
    T = 200
    x = rand((1, T, 16), torch.float32, dev, 3)
    one, zero = torch.ones_like(x), torch.zeros_like(x)
    check_scan(x, one)                                  # a plain sum
    h, _ = linear_scan(x, zero)
    assert torch.equal(h, x)                            # nothing is kept
    reset = one.clone()
    reset[:, ::50] = 0
    check_scan(x, reset)
    check_scan(x, -0.9 * one)
    # saturated logits: exactly 0 and 1, also at infinity
    for mix in (False, True):
        h, _ = linear_scan(x, zero - INF, gates="logit", mix=mix)
        assert torch.equal(h, x)
    h, _ = linear_scan(x, zero + INF, gates="logit", mix=True)
    assert torch.equal(h, zero)                         # 1 - a = 0: the state never moves
    g = (zero + INF).requires_grad_()
    grad, = torch.autograd.grad(linear_scan(x, g, gates="logit", mix=True)[0].sum(), g)
    assert torch.equal(grad, zero)
    check_scan(x, 40 * torch.sign(rand(x.shape, torch.float32, dev, 4)), gates="logit")
    # a memory of 1e5 steps: the error of 1 - a stays relative to 1 - a
    check_scan(x, zero + 11.5, rand((1, 16), torch.float32, dev, 5), gates="logit", mix=True)
    # an infinite input stays where the recurrence carries it, and does not reach other channels
    y = x.clone()
    y[0, 100, 3] = INF
    h, _ = linear_scan(y, 0.5 * one)
    assert torch.isinf(h[0, 100:, 3]).all() and torch.isfinite(h[0, :100]).all()
    assert torch.isfinite(h[0, :, torch.arange(16) != 3]).all()


@on_devices
@on_types
def test_scan_strides(dev, dt):
    x, g = scan_inputs((4, 60, 48), dt, dev, "decay", seed=5)
    check_scan(x[:, ::2], g[:, ::2])
    check_scan(x[:, :, 3:40], g[:, :, 3:40])            # channels start off the 16-byte grid
    check_scan(x[:, :, ::3], g[:, :, ::3])
    check_scan(x.transpose(0, 1), g.transpose(0, 1))    # time-major data
    check_scan(x.transpose(1, 2), g.transpose(1, 2))    # channel-major data
    check_scan(x, g[:, :, :1].expand_as(x))             # one gate for all channels
    check_scan(x, g[:, :1].expand_as(x))                # one gate for all steps
    check_scan(x[:1].expand(4, 60, 48), g)
    check_scan(x[:, :, 0], g[:, :, 0])
    check_scan(x[:, 0], g[:, 0])


@on_devices
def test_scan_shared_and_partial_gradients(dev):
    x, g = scan_inputs((2, 40, 24), torch.float32, dev, "logit", seed=6)
    lg = g[:, :, :1].clone().requires_grad_()
    h, last = linear_scan(x, lg.expand_as(x), gates="logit", mix=True)
    d, = torch.autograd.grad(h.sum(), lg)               # h's gradient is a stride-0 view, last has none
    full = g[:, :, :1].expand_as(x).clone().requires_grad_()
    want, = torch.autograd.grad(linear_scan(x, full, gates="logit", mix=True)[0].sum(), full)
    close(d, np64(want.double().sum(2, keepdim=True)), 24 * 2.0 ** -23 * np64(want.abs().sum(2, keepdim=True)))
    lx = x.clone().requires_grad_()
    only_last, = torch.autograd.grad(linear_scan(lx, g, gates="logit")[1].sum(), lx)
    a = 1 / (1 + np.exp(-np64(g)))
    tail = np.ones_like(a)
    for t in range(38, -1, -1):
        tail[:, t] = tail[:, t + 1] * a[:, t + 1]
    close(only_last, tail, 40 * 20 * 2.0 ** -24)


@on_devices
def test_scan_gradient_against_differences(dev):
    x, g = scan_inputs((1, 9, 3), torch.float32, dev, "logit", seed=7)
    h0 = rand((1, 3), torch.float32, dev, 9)
    w = rand(x.shape, torch.float32, dev, 10)
    for mix, reverse in ((True, False), (False, True)):
        def f(*a):
            h, last = linear_scan(*a, gates="logit", mix=mix, reverse=reverse)
            return (h.double() * w).sum() + last.double().sum()
        leaves = [t.clone().requires_grad_() for t in (x, g, h0)]
        grads = torch.autograd.grad(f(*leaves), leaves)
        step = 2.0 ** -6
        for i, grad in enumerate(grads):
            for j in range(grad.numel()):
                lo, hi = [t.clone() for t in (x, g, h0)], [t.clone() for t in (x, g, h0)]
                lo[i].view(-1)[j] -= step
                hi[i].view(-1)[j] += step
                # central: step^2 f''' / 6 < 2^-12 * 8 (nine steps, weights of size 2) and rounding 2^-19 / step
                assert abs(float(f(*hi) - f(*lo)) / (2 * step) - float(grad.view(-1)[j])) < 4e-3


@on_devices
def test_scan_empty(dev):
    z = torch.zeros(2, 0, 5, device=dev)
    h0 = rand((2, 5), torch.float32, dev, 1).requires_grad_()
    h, last = linear_scan(z, z, h0)
    assert h.shape == (2, 0, 5) and torch.equal(last, h0)
    d, = torch.autograd.grad(last.sum(), h0)
    assert torch.equal(d, torch.ones_like(d))
    assert torch.equal(linear_scan(z, z)[1], torch.zeros(2, 5, device=dev))
    for shape in ((0, 4, 5), (2, 4, 0)):
        z = torch.zeros(shape, device=dev, requires_grad=True)
        h, last = linear_scan(z, z)
        assert h.shape == shape and last.shape == (shape[0], shape[2])
        torch.autograd.grad(h.sum(), z)


@on_devices
@on_types
@pytest.mark.parametrize("gates,mix,reverse", FORMS)
@pytest.mark.parametrize("b,d", [(1, 1), (3, 7), (64, 96), (2, 1030)])
def test_scan_step_is_the_sequence(dev, dt, gates, mix, reverse, b, d):
    x, g = scan_inputs((b, 5, d), dt, dev, gates, seed=d)
    h0 = rand((b, d), torch.float32, dev, 2)
    want = oracle.scan(np64(x), np64(g), np64(h0), None, gates == "logit", mix, False)
    state, other = h0.clone(), torch.full_like(h0, float("nan"))
    for t in range(5):
        if t % 2:
            h = linear_scan_step(x[:, t], g[:, t], state, gates=gates, mix=mix)
        else:
            h = linear_scan_step(x[:, t], g[:, t], state, gates=gates, mix=mix, state_out=other)
            state, other = other, state
        w, tol = want["h"][0][:, t], want["h"][1][:, t]
        close(h, w, tol + rounding(dt, w))
        close(state, w, tol + rounding(torch.float32, w))
    pool = rand((2 * b, d + 3), torch.float32, dev, 3)
    before = pool.clone()
    view = pool[::2, 1:d + 1]
    linear_scan_step(x[:, 0], g[:, 0], view, gates=gates, mix=mix)
    a = linear_scan_step(x[:, 0], g[:, 0], before[::2, 1:d + 1].clone(), gates=gates, mix=mix)
    assert torch.equal(view.to(dt), a)
    assert torch.equal(pool[1::2], before[1::2]) and torch.equal(pool[:, 0], before[:, 0])


@on_devices
def test_scan_refusals(dev):
    x, g = scan_inputs((2, 4, 3), torch.float32, dev, "decay")
    h0, n = torch.zeros(2, 3, device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
    for args, kw in (((x.double(), g.double()), {}), ((x, g.half()), {}), ((x, g[:, :3]), {}), ((x, g, h0.half()), {}),
                     ((x, g, h0[:1]), {}), ((x, g, h0[:, 0]), {}), ((x, g), {"gates": "log"}), ((x[0, 0], g[0, 0]), {}),
                     ((x, g), {"lengths": n.float()}), ((x, g), {"lengths": n[:1]}), ((x, g), {"lengths": n.to("meta")}),
                     ((x, g.to("meta")), {}), ((x, None), {}), ((x[:, :, 0], g[:, :, 0], h0), {})):
        with pytest.raises(ValueError):
            linear_scan(*args, **kw)
    y, k = x[:, 0], g[:, 0]
    big = torch.zeros(40, device=dev)
    for args, kw in (((y.double(), k, h0), {}), ((y, k.half(), h0), {}), ((y, k, h0.half()), {}), ((y, k, h0[:1]), {}),
                     ((x, g, h0), {}), ((y, k, h0), {"state_out": h0.double()}), ((y, k, h0), {"state_out": h0[:1]}),
                     ((y, k, h0[:1].expand(2, 3)), {}), ((y, k, h0), {"state_out": h0[:, :1].expand(2, 3)}),
                     ((y, k, h0), {"gates": "none"}), ((y, k, big[:6].view(2, 3)), {"state_out": big[3:9].view(2, 3)}),
                     ((big[1:7].view(2, 3), k, big[:6].view(2, 3)), {})):
        with pytest.raises(ValueError):
            linear_scan_step(*args, **kw)


# ---- dropout -------------------------------------------------------------------------------------------------------
def counter_at(v, dev):
    return torch.full((1,), v, dtype=torch.int64, device=dev)


@on_devices
@on_types
@pytest.mark.parametrize("shape", [(1,), (3,), (5, 7), (64, 96), (3, 1031), (2, 3, 5, 16)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout_values_and_gradients(dev, dt, shape, p):
    x, r, dy = (rand(shape, dt, dev, i) for i in range(3))
    lx, lr = x.clone().requires_grad_(), r.clone().requires_grad_()
    ctr = counter_at(5, dev)
    y = dropout(lx, p, 1234, ctr, site=2)
    z = dropout(lx, p, 1234, ctr, site=2, residual=lr)
    ctr.add_(1)         # the backward passes use what their forward passes read
    n = x.numel()
    keep = oracle.keep_mask(range(n), p, 1234, 5, 2).reshape(shape)
    s = 1 / (1 - p) if p < 1 else 0.0
    want = np.where(keep, np64(x) * s, 0.0)
    close(y, want, rounding(dt, want) + 2 * oracle.U * np.abs(want))
    both = want + np64(r)
    close(z, both, rounding(dt, both) + 3 * oracle.U * (np.abs(want) + np.abs(np64(r))))
    dwant = np.where(keep, np64(dy) * s, 0.0)
    dx, = torch.autograd.grad(y, lx, dy)
    close(dx, dwant, rounding(dt, dwant) + 2 * oracle.U * np.abs(dwant))
    dx2, dr = torch.autograd.grad(z, (lx, lr), dy)
    assert torch.equal(dx2, dx) and torch.equal(dr, dy)
    only, = torch.autograd.grad(dropout(x, p, 1234, ctr, residual=lr).sum(), lr)
    assert torch.equal(only, torch.ones_like(lr))


@on_devices
@on_types
def test_dropout_special_values_and_strides(dev, dt):
    x = rand((40, 50), dt, dev, 1)
    x[::3] = INF
    x[1::3] = float("nan")
    y = dropout(x, 0.5, 3, counter_at(0, dev))
    keep = torch.from_numpy(oracle.keep_mask(range(2000), 0.5, 3, 0, 0).reshape(40, 50)).to(dev)
    assert (y[~keep] == 0).all() and torch.equal(torch.isnan(y), torch.isnan(x) & keep)
    big = rand((40, 60), dt, dev, 2)
    ctr = counter_at(9, dev)
    for view in (big[:, 5:33], big.t(), big[::2], big[:1].expand(40, 60)):
        assert torch.equal(dropout(view, 0.3, 8, ctr), dropout(view.contiguous(), 0.3, 8, ctr))
        assert torch.equal(dropout(view, 0.3, 8, ctr, residual=view), dropout(view.contiguous(), 0.3, 8, ctr,
                                                                             residual=view.contiguous()))
    flat = big.reshape(-1)
    for off in (1, 2, 3, 5):    # off the 16-byte grid: the element's index counts from the tensor's start
        assert torch.equal(dropout(flat[off:off + 801], 0.3, 8, ctr), dropout(flat[off:off + 801].clone(), 0.3, 8, ctr))
    assert dropout(big[:0], 0.3, 8, ctr).shape == (0, 60)
    lx = big[:, ::2].clone().requires_grad_()
    d, = torch.autograd.grad(dropout(lx, 0.25, 8, ctr).sum(), lx)       # a stride-0 gradient
    m = torch.from_numpy(oracle.keep_mask(range(1200), 0.25, 8, 9, 0).reshape(40, 30)).to(dev)
    assert torch.equal(d, torch.where(m, torch.full_like(lx, 1 / 0.75), torch.zeros_like(lx)))


@on_devices
@pytest.mark.parametrize("seed,counter,site", [(0, 0, 0), (-1, 3, 1), ((1 << 64) + 5, (1 << 62) + 1, (1 << 32) - 1),
                                               (1 << 63, -7, 12345)])
def test_dropout_mask_is_its_definition(dev, seed, counter, site):
    x = torch.ones(3000, device=dev)
    for p in (0.3, 2.0 ** -20, 1 - 2.0 ** -20, 0.5 + 2.0 ** -30):
        want = oracle.keep_mask(range(3000), p, seed, counter, site)
        y = dropout(x, p, seed, counter_at(counter, dev), site=site)
        assert np.array_equal(y.cpu().numpy() != 0, want)
        assert np.array_equal(keep_mask(3000, p, seed, counter_at(counter, "cpu"), site).numpy(), want)


@pytest.mark.gpu
def test_dropout_large_masks_agree_with_the_cpu():
    n = 3 * (1 << 20) + 7
    x = torch.ones(n, device="cuda")
    for p in (0.1, 1.5 * 2.0 ** -17, 1 - 2.0 ** -17):       # thresholds inside one step of the first 16 bits
        y = dropout(x, p, 77, counter_at(4, "cuda"), site=6)
        assert torch.equal(y.cpu() != 0, keep_mask(n, p, 77, counter_at(4, "cpu"), 6))


@on_devices
def test_dropout_rate_and_independence(dev):
    n = 1 << 16
    x = torch.ones(n, device=dev)
    masks = {}
    for seed, ctr, site in ((1, 0, 0), (1, 1, 0), (1, 0, 1), (2, 0, 0), (3, 0, 0)):
        m = dropout(x, 0.25, seed, counter_at(ctr, dev), site=site) != 0
        assert abs(float(m.float().mean()) - 0.75) < 6 * (0.25 * 0.75 / n) ** 0.5
        masks[(seed, ctr, site)] = m.float() - 0.75
    ms = list(masks.values())
    for i in range(len(ms)):
        for j in range(i):
            assert abs(float((ms[i] * ms[j]).mean())) < 6 * 0.25 * 0.75 / n ** 0.5
        for lag in (1, 2, 3, 4, 64):
            assert abs(float((ms[i][lag:] * ms[i][:-lag]).mean())) < 6 * 0.25 * 0.75 / (n - lag) ** 0.5


@on_devices
def test_dropout_module(dev):
    m = CounterDropout(0.5, seed=3, site=1).to(dev)
    x = rand((20, 30), torch.float32, dev, 1)
    assert not m.state_dict() and not list(m.parameters())
    a, b = m(x), m(x)
    assert not torch.equal(a, b) and int(m.counter) == 2
    assert torch.equal(a, dropout(x, 0.5, 3, counter_at(0, dev), site=1))
    with torch.no_grad():
        assert m(x) is x
    m.eval()
    assert m(x) is x and torch.equal(m(x, residual=x), x + x) and int(m.counter) == 2
    with pytest.raises(ValueError):
        CounterDropout(1.5)


@on_devices
def test_dropout_refusals(dev):
    x, c = rand((4, 6), torch.float32, dev, 0), counter_at(0, dev)
    for args, kw in (((x, -0.1, 0, c), {}), ((x, 1.1, 0, c), {}), ((x, math.nan, 0, c), {}), ((x.double(), 0.5, 0, c), {}),
                     ((x, 0.5, 0.0, c), {}), ((x, 0.5, 0, c.int()), {}), ((x, 0.5, 0, torch.zeros(2, dtype=torch.int64, device=dev)), {}),
                     ((x, 0.5, 0, 3), {}), ((x, 0.5, 0, c), {"site": -1}), ((x, 0.5, 0, c), {"site": 1 << 32}),
                     ((x, 0.5, 0, c.to("meta")), {}), ((x, 0.5, 0, c), {"residual": x[:2]}),
                     ((x, 0.5, 0, c), {"residual": x.half()}), ((x, 0.5, 0, c), {"residual": x.to("meta")})):
        with pytest.raises(ValueError):
            dropout(*args, **kw)


# ---- together ------------------------------------------------------------------------------------------------------
def policy_loss(x, wg, wo, tokens, adv, ctr, lengths):
    """dropout -> gated memory -> logits -> policy gradient with an entropy bonus"""
    y = dropout(x, 0.2, 11, ctr, site=0)
    h, last = linear_scan(y, y.matmul(wg), gates="logit", mix=True, lengths=lengths)
    h = dropout(h, 0.2, 11, ctr, site=1, residual=x)
    out = token_logprobs(h.matmul(wo), tokens)
    return -(adv * out.logprob).sum() - 0.01 * out.entropy.sum() + last.square().sum(), out


def plain_loss(x, wg, wo, tokens, adv, lengths):
    keep = [torch.from_numpy(oracle.keep_mask(range(x.numel()), 0.2, 11, 5, s).reshape(x.shape)) for s in (0, 1)]
    y = torch.where(keep[0], x / 0.8, torch.zeros_like(x))
    a = torch.sigmoid(y.matmul(wg))
    h = torch.zeros_like(x[:, 0])
    hs = []
    for t in range(x.shape[1]):
        on = (t < lengths)[:, None]
        h = torch.where(on, a[:, t] * h + (1 - a[:, t]) * y[:, t], h)
        hs.append(torch.where(on, h, torch.zeros_like(h)))
    z = torch.where(keep[1], torch.stack(hs, 1) / 0.8, torch.zeros_like(x)) + x
    lp = torch.log_softmax(z.matmul(wo), -1)
    live = tokens != -100
    taken = torch.where(live, lp.gather(-1, tokens.clamp_min(0)[..., None])[..., 0], torch.zeros_like(adv))
    ent = torch.where(live, -(lp.exp() * lp).sum(-1), torch.zeros_like(adv))
    return -(adv * taken).sum() - 0.01 * ent.sum() + h.square().sum()


def policy_data(dev, b=3, t=21, d=24, v=37):
    n = torch.tensor([t, t // 2, 3])
    tokens = torch.randint(0, v, (b, t), generator=torch.Generator().manual_seed(5))
    tokens[torch.arange(t)[None] >= n[:, None]] = -100
    data = [rand((b, t, d), torch.float32, "cpu", 1), rand((d, d), torch.float32, "cpu", 2, 0.2),
            rand((d, v), torch.float32, "cpu", 3, 0.3), tokens, rand((b, t), torch.float32, "cpu", 4), n]
    return [q.to(dev) for q in data]


@on_devices
def test_tangents_are_refused(dev):
    """Forward-mode differentiation is not offered: an error, not a result without its tangent."""
    from torch.autograd import forward_ad
    x, tok = rand((3, 8), torch.float32, dev, 0), torch.zeros(3, dtype=torch.int64, device=dev)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for f in (lambda: token_logprobs(d, tok), lambda: linear_scan(d, x), lambda: dropout(d, 0.5, 1, counter_at(0, dev))):
            with pytest.raises(RuntimeError):       # (NotImplementedError is one)
                f()


@on_devices
def test_calls_without_gradients(dev):
    """Calls that need no gradient take a shorter way to the same kernels: same results, and outputs free to be written."""
    x, g = rand((3, 700, 12), torch.float32, dev, 0), torch.sigmoid(rand((3, 700, 12), torch.float32, dev, 1))
    tok, ctr, n = torch.arange(3, device=dev)[:, None].expand(3, 700), counter_at(4, dev), torch.tensor([700, 0, 33], device=dev)
    for f in (lambda t: token_logprobs(t, tok, temperature=0.5, top_k=4), lambda t: token_logprobs(t, tok)[:3],
              lambda t: linear_scan(t, g, lengths=n), lambda t: linear_scan(t[:, :, 0], g[:, :, 0], reverse=True, lengths=n),
              lambda t: (dropout(t, 0.25, 1, ctr),), lambda t: (dropout(t, 0.25, 1, ctr, residual=t),)):
        want = f(x.clone().requires_grad_())
        with torch.no_grad():
            inside = f(x.clone().requires_grad_())
        outside = f(x)
        for w, a, b in zip(want, inside, outside):
            assert torch.equal(w, a) and torch.equal(w, b) and not a.requires_grad and not b.requires_grad
            assert w.shape == b.shape and w.stride() == b.stride()
            b.zero_()


@pytest.mark.gpu
@pytest.mark.parametrize("op", ("logprob", "scan", "dropout"))
def test_offsets_past_32_bits(op):
    """More than 2^31 elements: the last part of the tensor equals the same part taken alone."""
    def noise(*shape):
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_()

    if op == "logprob":
        x, tok = noise(33000, 65540), torch.arange(33000, device="cuda")
        part = slice(32000, 33000)      # (more than 512 rows: not split in either call)

        def run(sl):
            leaf = x[sl].detach().requires_grad_()
            o = token_logprobs(leaf, tok[sl], top_k=3)
            return o.logprob, o.top_tokens, torch.autograd.grad(o.logprob.sum() + o.entropy.sum(), leaf)[0]
    elif op == "scan":
        x, g = noise(3, 45000, 16384), torch.rand((1, 45000, 16384), dtype=torch.float32, device="cuda").to(torch.bfloat16)
        part = slice(2, 3)

        def run(sl):
            leaf = x[sl].detach().requires_grad_()
            h, last = linear_scan(leaf, g.expand(leaf.shape))
            return h, last, torch.autograd.grad(h.sum(), leaf)[0]
    else:
        n = (1 << 31) + (1 << 22)
        y = dropout(torch.ones(n, dtype=torch.bfloat16, device="cuda"), 0.5, 3, counter_at(1, "cuda"))
        for at in (0, (1 << 31) - 2048, n - 4096):
            want = 2 * oracle.keep_mask(range(at, at + 4096), 0.5, 3, 1, 0).astype(np.float64)
            assert np.array_equal(np64(y[at:at + 4096]), want)
        return
    assert x.numel() > 1 << 31
    whole = run(slice(None))
    for a, b in zip(whole, run(part)):
        assert torch.equal(a[part], b)


@on_devices
@pytest.mark.parametrize("op", ("logprob", "scan", "dropout"))
def test_gradients_are_not_differentiated_again(dev, op):
    """A graph of the gradient may be asked for (as a larger graph does); going through it is refused, not wrong."""
    x = rand((3, 4, 8), torch.float32, dev, 0).requires_grad_()
    y = {"logprob": lambda: token_logprobs(x, torch.zeros(3, 4, dtype=torch.int64, device=dev)).logprob,
         "scan": lambda: linear_scan(x, torch.full_like(x, 0.5))[0],
         "dropout": lambda: dropout(x, 0.25, 1, counter_at(0, dev))}[op]()
    plain, = torch.autograd.grad(y.square().sum(), x, retain_graph=True)
    d, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    assert torch.equal(d, plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), x)


@on_devices
def test_recurrent_policy_step(dev):
    x, wg, wo, tokens, adv, n = policy_data(dev)
    leaves = [q.clone().requires_grad_() for q in (x, wg, wo)]
    loss, _ = policy_loss(*leaves, tokens, adv, counter_at(5, dev), n)
    got = torch.autograd.grad(loss, leaves)
    ref = [q.cpu().double().requires_grad_() for q in (x, wg, wo)]
    want_loss = plain_loss(*ref, tokens.cpu(), adv.cpu().double(), n.cpu())
    want = torch.autograd.grad(want_loss, ref)
    # every value passes two products of up to 63 terms, 21 recurrent steps and a softmax in 32 bits: a few hundred
    # roundings of sums whose terms are below 4; 512 half steps of the largest entry bound them
    loss, want_loss = loss.detach(), want_loss.detach()
    assert abs(float(loss) - float(want_loss)) < 512 * 2.0 ** -24 * (1 + abs(float(want_loss)))
    for g, w in zip(got, want):
        close(g, np64(w), 512 * 2.0 ** -24 * max(1.0, float(w.abs().max())))


@on_devices
def test_serving_steps_are_the_sequence(dev):
    x, wg, wo, tokens, _, _ = policy_data(dev)
    h, _ = linear_scan(x, x.matmul(wg), gates="logit", mix=True)
    state = torch.zeros(3, 24, device=dev)
    for t in range(x.shape[1]):
        y = linear_scan_step(x[:, t], x[:, t].matmul(wg), state, gates="logit", mix=True)
        # the products' rounding differs with their shape: 24 terms below 4, then 21 steps
        assert float((y - h[:, t]).abs().max()) < 256 * 2.0 ** -24 * 4
        out = token_logprobs(h[:, t].matmul(wo), tokens[:, 0], top_k=3)
        assert torch.equal(out.top_tokens[:, 0], h[:, t].matmul(wo).argmax(1))
