"""The sequence-policy operators inside hipGraphs, on side streams and side by side (ops/logprob.py, scan.py, dropout.py)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def native():
    from pytorch_distributed_amd import ops
    ops.require_native()


def rand(shape, dt, seed, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dt).cuda()


def make(kind, dt, seed):
    """-> (inputs that change from replay to replay, function of them that returns every output and gradient)"""
    from pytorch_distributed_amd.ops.dropout import dropout
    from pytorch_distributed_amd.ops.logprob import token_logprobs
    from pytorch_distributed_amd.ops.scan import linear_scan, linear_scan_step
    if kind == "logprob":
        n, v = 5, 9000
        x = rand((n, v), dt, seed, 2.0)
        tok = torch.arange(n, device="cuda") + seed
        w = rand((n,), torch.float32, seed + 1)

        def f():
            leaf = x.detach().requires_grad_()
            o = token_logprobs(leaf, tok, temperature=0.9, top_k=6)
            d, = torch.autograd.grad((o.logprob, o.entropy), leaf, (w, w))
            return o.logprob.detach(), o.entropy.detach(), o.top_logprobs, o.top_tokens, d
        return (x, tok, w), f
    if kind in ("scan", "scan_long", "returns"):
        shape = {"scan": (3, 300, 72), "scan_long": (1, 6000, 40), "returns": (4, 5000, 1)}[kind]
        x, g = rand(shape, dt, seed), rand(shape, dt, seed + 1, 1.5, 2.0)
        h0, dh, dl = rand((shape[0], shape[2]), torch.float32, seed + 2), rand(shape, dt, seed + 3), \
            rand((shape[0], shape[2]), torch.float32, seed + 4)

        def f():
            leaves = [t.detach().requires_grad_() for t in (x, g, h0)]
            h, last = linear_scan(*leaves, gates="logit", mix=kind == "scan", reverse=kind == "returns")
            return (h.detach(), last.detach()) + torch.autograd.grad((h, last), leaves, (dh, dl))
        return (x, g, h0, dh, dl), f
    if kind == "step":
        x, g, s = rand((9, 130), dt, seed), rand((9, 130), dt, seed + 1), rand((9, 130), torch.float32, seed + 2)
        out = torch.empty_like(s)

        def f():
            return linear_scan_step(x, g, s, gates="logit", state_out=out), out.clone()
        return (x, g, s), f
    x, r, dy = (rand((33, 515), dt, seed + i) for i in range(3))
    ctr = torch.full((1,), 10 + seed, dtype=torch.int64, device="cuda")

    def f():
        lx, lr = x.detach().requires_grad_(), r.detach().requires_grad_()
        y = dropout(lx, 0.3, 5, ctr, residual=lr)
        return (y.detach(),) + torch.autograd.grad(y, (lx, lr), dy)
    return (x, r, dy, ctr), f


KINDS = ["logprob", "scan", "scan_long", "returns", "step", "dropout"]


def same(a, b):
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def capture(f):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    return graph, out


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
def test_replays_equal_eager_runs(kind, dt):
    ins, f = make(kind, dt, 0)
    graph, out = capture(f)
    for seed in range(1, 6):
        fresh, g = make(kind, dt, seed)
        for a, b in zip(ins, fresh):
            a.copy_(b)
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        same(got, g())                  # the program's own eager work between replays
        same(got, g())
        torch.cuda.synchronize()


def test_a_replayed_counter_draws_new_masks():
    from pytorch_distributed_amd.ops.dropout import dropout
    x = torch.ones(1000, device="cuda")
    ctr = torch.zeros(1, dtype=torch.int64, device="cuda")

    def f():
        leaf = x.detach().requires_grad_()
        y = dropout(leaf, 0.5, 1, ctr)
        ctr.add_(1)
        return y.detach(), torch.autograd.grad(y.sum(), leaf)[0]
    graph, (y, d) = capture(f)
    ctr.zero_()
    for step in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = dropout(x, 0.5, 1, torch.full((1,), step, dtype=torch.int64, device="cuda"))
        assert torch.equal(y, want) and torch.equal(d, want)


@pytest.mark.parametrize("kind", ["logprob", "scan_long", "returns", "dropout"])
def test_calls_without_gradients_replay_what_calls_with_them_give(kind):
    from pytorch_distributed_amd.ops.dropout import dropout
    from pytorch_distributed_amd.ops.logprob import token_logprobs
    from pytorch_distributed_amd.ops.scan import linear_scan
    ctr, tok = torch.full((1,), 7, dtype=torch.int64, device="cuda"), torch.arange(5, device="cuda")
    gate = rand((3, 9000), torch.float32, 5, 1.5, 2.0)
    x, f = {"logprob": (rand((5, 9000), torch.bfloat16, 0), lambda t: token_logprobs(t, tok, top_k=6)),
            "scan_long": (rand((1, 6000, 40), torch.bfloat16, 1),
                          lambda t: linear_scan(t, torch.full_like(t, 0.75), mix=True)),
            "returns": (rand((3, 9000), torch.float32, 2), lambda t: linear_scan(t, gate, gates="logit", reverse=True)),
            "dropout": (rand((33, 515), torch.bfloat16, 3), lambda t: (dropout(t, 0.3, 5, ctr, residual=t),))}[kind]
    with torch.no_grad():
        graph, out = capture(lambda: f(x))
    for seed in range(4):
        x.copy_(rand(x.shape, x.dtype, 20 + seed))
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        want = f(x.clone().requires_grad_())
        assert any(t.requires_grad for t in want)
        same(got, [t.detach() for t in want])
        torch.cuda.synchronize()


@pytest.mark.parametrize("kind", ["logprob", "scan", "scan_long", "returns"])
def test_two_graphs_at_once(kind):
    """Two captured calls share no scratch: replayed side by side on two streams they keep their results."""
    pairs = [make(kind, torch.bfloat16, s) for s in (3, 4)]
    graphs = [capture(f) for _, f in pairs]
    want = [[t.clone() for t in f()] for _, f in pairs]
    streams = [torch.cuda.Stream() for _ in pairs]
    torch.cuda.synchronize()
    for _ in range(20):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        same(out, w)


@pytest.mark.parametrize("kind", KINDS)
def test_on_a_side_stream(kind):
    ins, f = make(kind, torch.float32, 2)
    want = [t.clone() for t in f()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = f()
    torch.cuda.current_stream().wait_stream(s)
    same(got, want)
