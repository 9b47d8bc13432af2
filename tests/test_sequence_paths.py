"""The paths that run on the sequence-policy operators: conservative loss and dropout of the torch learner core, the
evaluator's returns (agents/learners.py, models/, agents/evaluators.py)."""
import copy

import numpy as np
import pytest
import torch

from pytorch_distributed_amd.agents.evaluators import returns_report, run_episodes
from pytorch_distributed_amd.agents.learners import DdpgTorchCore, DqnTorchCore, make_core
from pytorch_distributed_amd.launcher import prepare_options, run
from pytorch_distributed_amd.ops.dropout import CounterDropout
from pytorch_distributed_amd.parallel.comm import FakeComm, SingleComm
from pytorch_distributed_amd.parallel.inference_server import native_learner_expected
from pytorch_distributed_amd.utils.board import read_scalars
from pytorch_distributed_amd.utils.factory import EnvsDict, ModelsDict
from pytorch_distributed_amd.utils.options import Options, torch_core_options

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
on_devices = pytest.mark.parametrize("dev", DEVICES)


class OneBatch(object):
    def __init__(self, batch, weights=None):
        self.batch, self.weights, self.enable_per = batch, weights, weights is not None
        self.seen = None

    def sample_with_priorities(self, n):
        w = self.weights if self.weights is not None else torch.ones(n, 1)
        return self.batch, torch.arange(n), w

    def update_priorities(self, inds, td):
        self.seen = td


def options(config, **ov):
    return prepare_options(Options(config=config, overrides=dict({"device": "cpu", "agent_params.batch_size": 24}, **ov)))


def batch_for(opt, n=24, seed=0):
    g = torch.Generator().manual_seed(seed)
    d = int(np.prod(opt.state_shape))
    s = [torch.randn((n,) + tuple(opt.state_shape), generator=g) for _ in range(2)]
    if opt.agent_type == "dqn":
        a = torch.randint(0, opt.action_space, (n, 1), generator=g).float()
    else:
        a = torch.rand(n, opt.action_space, generator=g) * 2 - 1
    assert d > 0
    return (s[0], a, torch.randn(n, 1, generator=g), torch.full((n, 1), 0.9), s[1], torch.zeros(n, 1))


def model_for(opt, seed=0):
    torch.manual_seed(seed)
    return ModelsDict[opt.model_type](opt.model_params, opt.norm_val, opt.state_shape, opt.action_space, opt.action_shape)


@on_devices
@pytest.mark.parametrize("per", [False, True])
def test_conservative_loss_and_its_gradient(dev, per):
    opt = options(6, **{"agent_params.cql_alpha": 0.7})
    batch = batch_for(opt)
    w = torch.rand(24, 1, generator=torch.Generator().manual_seed(4)) if per else None
    proto = model_for(opt)
    core = DqnTorchCore(opt, copy.deepcopy(proto).to(dev), copy.deepcopy(proto).to(dev), OneBatch(batch, w))
    core.step()
    ref = copy.deepcopy(proto).double()
    s0, a, r, g, s1, t = (x.double() for x in batch)
    with torch.no_grad():
        y = r + g * ref.critic(s1.flatten(1)).max(1, keepdim=True)[0]
    q = ref.critic(s0.flatten(1))
    pick = q.gather(1, a.long())
    ww = w.double() if per else torch.ones(24, 1, dtype=torch.float64)
    loss = (ww * (pick - y) ** 2).mean() + 0.7 * (ww * (torch.logsumexp(q, 1, keepdim=True) - pick)).mean()
    loss.backward()
    # four layers of 256-term products in 32 bits: 2048 roundings of values near 1 bound them
    tol = 2048 * 2.0 ** -24
    assert abs(core.loss_values()["critic_loss"] - float(loss.detach())) < tol
    for p, want in zip(core.model.parameters(), ref.parameters()):
        assert float((p.grad.cpu().double() - want.grad).abs().max()) < tol
    if per:
        assert core.memory.seen is not None


@on_devices
@pytest.mark.parametrize("config", [6, 3])
def test_learner_with_dropout(dev, config):
    opt = options(config, **{"model_params.dropout": 0.25})
    plain = options(config)
    proto = model_for(opt)
    assert list(proto.state_dict()) == list(model_for(plain).state_dict())          # checkpoints are unchanged
    for a, b in zip(proto.parameters(), model_for(plain).parameters()):
        assert torch.equal(a, b)
    kind = DqnTorchCore if opt.agent_type == "dqn" else DdpgTorchCore
    make = lambda: kind(opt, copy.deepcopy(proto).to(dev), copy.deepcopy(proto).to(dev), OneBatch(batch_for(opt)))
    one, two = make(), make()
    for _ in range(3):
        one.step()
        two.step()
    assert torch.equal(one.flat_params(), two.flat_params())            # masks are a function of seed, counter and site
    per_step = 1 if opt.agent_type == "dqn" else 2                      # (DDPG: actor loss and critic loss)
    assert [int(m.counter) for m in one.drops] == [3 * per_step] * len(one.drops)
    # a resumed learner goes on with the next masks
    three = make()
    three.load_resume_state(one.resume_state())
    assert [int(m.counter) for m in three.drops] == [3 * per_step] * len(one.drops)
    one.step()
    three.step()
    assert torch.equal(one.flat_params(), three.flat_params())
    # acting and targets do not drop
    x = batch_for(opt)[0].to(dev)
    with torch.no_grad():
        f = one.model.forward if opt.agent_type == "dqn" else one.model.forward_actor
        assert torch.equal(f(x), f(x))


@on_devices
def test_dropout_gradient_of_the_whole_model(dev):
    """The backward pass drops what the forward pass dropped: the critic's gradient against a model whose masks are fixed."""
    opt = options(6, **{"model_params.dropout": 0.5})
    m = model_for(opt).to(dev)
    x = batch_for(opt)[0].to(dev)
    q = m(x)
    grads = torch.autograd.grad(q.square().sum(), list(m.parameters()))
    ref = model_for(options(6)).double()
    from pytorch_distributed_amd.ops.dropout import keep_mask
    h = x.cpu().double().flatten(1)
    for i, drop in enumerate(m.drops):
        h = torch.relu(ref.critic[2 * i](h))
        keep = keep_mask(h.numel(), 0.5, drop.seed, torch.zeros(1, dtype=torch.int64), drop.site).reshape(h.shape)
        h = torch.where(keep, h * 2, torch.zeros_like(h))
    want = torch.autograd.grad(ref.critic[6](h).square().sum(), list(ref.parameters()))
    for g, w in zip(grads, want):
        assert float((g.cpu().double() - w).abs().max()) < 4096 * 2.0 ** -24 * max(1.0, float(w.abs().max()))


def test_ranks_draw_different_masks():
    opt = options(6, **{"model_params.dropout": 0.25})
    proto = model_for(opt)
    cores = [DqnTorchCore(opt, copy.deepcopy(proto), copy.deepcopy(proto), OneBatch(batch_for(opt)), comm)
             for comm in [SingleComm()] + FakeComm.create(2)[1:]]
    assert cores[0].drops[0].seed == opt.seed and cores[1].drops[0].seed != cores[0].drops[0].seed


def test_cnn_dropout_and_defaults():
    opt = options(1, **{"model_params.dropout": 0.3})
    m = model_for(opt)
    x = torch.randint(0, 256, (2, 4, 84, 84), dtype=torch.uint8)
    assert not torch.equal(m(x), m(x)) and [type(d) for d in m.drops] == [CounterDropout]
    assert set(m.state_dict()) == set(model_for(options(1)).state_dict())
    assert model_for(options(1)).drops is None
    for config in range(10):
        o = Options(config=config)
        assert torch_core_options(o) == [] and o.agent_params.evaluate_returns is False
    with pytest.raises(ValueError):
        model_for(options(6, **{"model_params.dropout": 1.5}))


def test_native_core_is_not_taken_for_these_options(monkeypatch):
    from pytorch_distributed_amd.agents import learners
    monkeypatch.setattr(learners, "_pick_compute", lambda args, device: "native")       # as on a GPU
    for ov in ({"agent_params.cql_alpha": 0.1}, {"model_params.dropout": 0.1}):
        opt = options(6, **ov)
        proto = model_for(opt)
        core = make_core("dqn", opt, proto, copy.deepcopy(proto), OneBatch(batch_for(opt)), SingleComm(), torch.device("cpu"))
        assert isinstance(core, DqnTorchCore)
        opt.compute = "native"
        with pytest.raises(ValueError, match=list(ov)[0]):
            make_core("dqn", opt, proto, copy.deepcopy(proto), OneBatch(batch_for(opt)), SingleComm(), torch.device("cpu"))
        opt = options(2, **ov)
        opt.device, opt.compute = "cuda", "auto"
        assert native_learner_expected(opt) is False        # inference is not hosted by a core without shadow weights


@pytest.mark.gpu
def test_torch_core_on_device_replay():
    from pytorch_distributed_amd.memories.device_memory import DeviceMemory
    dev = torch.device("cuda")
    opt = prepare_options(Options(config=4, overrides={"memory_params.memory_size": 512, "agent_params.batch_size": 32,
                                                       "agent_params.cql_alpha": 0.5, "model_params.dropout": 0.1}))
    mem = DeviceMemory(opt.memory_params).attach(dev)
    s = torch.randint(0, 256, (256, 4, 84, 84), dtype=torch.uint8, device=dev)
    mem.feed_batch(s, torch.randint(0, 6, (256, 1), device=dev), torch.randn(256, 1, device=dev),
                   torch.full((256, 1), 0.95, device=dev), s.flip(0), torch.zeros(256, 1, device=dev))
    core = make_core("dqn", opt, model_for(opt).to(dev), model_for(opt).to(dev), mem, SingleComm(), dev)
    assert isinstance(core, DqnTorchCore)
    before = core.flat_params().clone()
    for _ in range(3):
        core.step()
    assert torch.isfinite(core.flat_params()).all() and not torch.equal(core.flat_params(), before)
    assert int(core.drops[0].counter) == 3


@on_devices
def test_returns_report(dev):
    rng = np.random.RandomState(0)
    trace = [(float(rng.randn()), bool(rng.rand() < 0.03) or i == 499, float(rng.randn())) for i in range(500)]
    ret, bias = returns_report(trace, 0.97, torch.device(dev))
    G, g = [0.0] * 500, 0.0
    for i in range(499, -1, -1):
        r, end, _ = trace[i]
        g = r + 0.97 * (0.0 if end else g)
        G[i] = g
    starts = [0] + [i + 1 for i in range(499) if trace[i][1]]
    # returns below 40, memory of 33 steps, means of at most 500 of them: 64 half steps of 40
    assert abs(ret - np.mean([G[i] for i in starts])) < 64 * 40 * 2.0 ** -24
    assert abs(bias - np.mean([trace[i][2] - G[i] for i in range(500)])) < 64 * 40 * 2.0 ** -24
    assert returns_report([], 0.97) == (0.0, 0.0)


def test_run_episodes_traces_what_it_counts():
    opt = options(6)
    env = EnvsDict[opt.env_type](opt.env_params, 0)
    model = model_for(opt)
    trace = []
    steps, reward, n, _ = run_episodes(env, model, 3, 20, trace=trace)
    assert len(trace) == steps and sum(e for _, e, _ in trace) == n == 3
    assert abs(sum(r for r, _, _ in trace) - reward) < 1e-9


def test_job_with_these_options(tmp_root):
    opt = Options(config=6, overrides={
        "root_dir": tmp_root, "timestamp": "seq", "device": "cpu", "num_actors": 1, "agent_params.steps": 60,
        "agent_params.learn_start": 40, "agent_params.poll_interval": 0.2, "agent_params.logger_freq": 0.3,
        "agent_params.evaluator_freq": 0.5, "agent_params.evaluator_nepisodes": 1, "agent_params.learner_freq": 5,
        "param_sync_freq": 5, "agent_params.cql_alpha": 0.1, "model_params.dropout": 0.1,
        "agent_params.evaluate_returns": True})
    sup = run(opt)
    assert all(c == 0 for c in sup.exitcodes), sup.exitcodes
    tags = {s["tag"] for s in read_scalars(opt.log_dir)}
    assert {"evaluator/avg_discounted_return", "evaluator/avg_value_bias", "learner/critic_loss"} <= tags
    opt.mode = 2
    opt.apply({})
    assert run(opt).procs[0][3].exitcode == 0
