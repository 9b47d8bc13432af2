"""The sequence-policy operators of `pytorch_distributed_amd.ops` as measurable cases: what each is in plain torch
operations, what a user's program calls, the work it cannot do without, and its definition in 64 bits.

`logprob`   ops.logprob.token_logprobs      log-probabilities of given tokens / actions, entropy, top alternatives
`scan`      ops.scan.linear_scan            gated linear recurrence over sequences
`step`      ops.scan.linear_scan_step       the same recurrence for one token per request
`dropout`   ops.dropout.dropout             counter-based dropout (+ residual), mask regenerated in the backward pass
"""
import math

import numpy as np
import torch

own = False     # True: `run` calls the framework's operators instead of the plain forms

IGNORE = -100
GOLDEN = 0x9E3779B97F4A7C15
MIX1, MIX2 = 0xFF51AFD7ED558CCD, 0xC4CEB9FE1A85EC53
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---- cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the conservative loss of a DQN learner step: batch 128, six actions, forward and gradient (latency)
        {"name": "logprob_actions_128x6", "op": "logprob", "rows": 128, "vocab": 6, "type": "fp32", "top": 0,
         "train": True, "temperature": 1.0, "masked": 0.0, "ignored": 0.0},
        # large-batch learner, illegal actions masked with -inf
        {"name": "logprob_actions_4096x18", "op": "logprob", "rows": 4096, "vocab": 18, "type": "fp32", "top": 0,
         "train": True, "temperature": 0.5, "masked": 0.3, "ignored": 0.0},
        # one sequence being served: its next token's log-probability and the 20 best alternatives
        {"name": "logprob_serve_1x131072", "op": "logprob", "rows": 1, "vocab": 131072, "type": "bf16", "top": 20,
         "train": False, "temperature": 0.7, "masked": 0.0, "ignored": 0.0},
        # a batch of requests over an odd vocabulary
        {"name": "logprob_serve_61x50257", "op": "logprob", "rows": 61, "vocab": 50257, "type": "fp16", "top": 5,
         "train": False, "temperature": 1.0, "masked": 0.0, "ignored": 0.0},
        # a policy-gradient step over 4096 tokens, some of them padding
        {"name": "logprob_train_4096x32000", "op": "logprob", "rows": 4096, "vocab": 32000, "type": "bf16", "top": 0,
         "train": True, "temperature": 1.0, "masked": 0.0, "ignored": 0.1},
        # scoring prompts: large vocabulary, 8 alternatives each
        {"name": "logprob_score_4096x131072", "op": "logprob", "rows": 4096, "vocab": 131072, "type": "bf16", "top": 8,
         "train": False, "temperature": 1.0, "masked": 0.0, "ignored": 0.0},
        # discounted returns of 16 evaluation episodes of up to 12500 steps (gate = gamma, 0 at episode ends)
        {"name": "scan_returns_16x12500", "op": "scan", "batch": 16, "steps": 12500, "dim": 1, "type": "fp32",
         "gates": "decay", "mix": False, "reverse": True, "ragged": True, "train": False},
        # a recurrent layer's training pass over padded sequences
        {"name": "scan_train_8x2048x2048", "op": "scan", "batch": 8, "steps": 2048, "dim": 2048, "type": "bf16",
         "gates": "logit", "mix": True, "reverse": False, "ragged": True, "train": True},
        # one long sequence of odd length in 32 bits: too few channels to fill the card without splitting the time axis
        {"name": "scan_long_1x65521x512", "op": "scan", "batch": 1, "steps": 65521, "dim": 512, "type": "fp32",
         "gates": "decay", "mix": False, "reverse": False, "ragged": False, "train": True},
        # one token for each of 64 requests
        {"name": "step_64x2048", "op": "step", "batch": 64, "dim": 2048, "type": "bf16", "gates": "logit", "mix": True},
        # the hidden layer of the 512-wide heads at batch 128 (latency)
        {"name": "dropout_128x512", "op": "dropout", "rows": 128, "cols": 512, "type": "fp32", "p": 0.1,
         "residual": False, "train": True},
        # dropout and residual sum of a wide layer over 16384 tokens, forward and gradient
        {"name": "dropout_16384x4096", "op": "dropout", "rows": 16384, "cols": 4096, "type": "bf16", "p": 0.1,
         "residual": True, "train": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprob", "logprob", "logprob", "scan", "scan", "scan", "step", "dropout", "dropout"])
    if op == "logprob":
        vocab = _log_int(rng, 2, 131072)
        train = rng.random() < 0.5
        rows = _log_int(rng, 1, max(1, min(16384, (4096 * (32000 if train else 131072)) // vocab)))
        return {"op": op, "rows": rows, "vocab": vocab, "type": rng.choice(["fp32", "bf16", "fp16"]) if rows * vocab < 1 << 26
                else rng.choice(["bf16", "fp16"]), "top": 0 if train else rng.choice([0, 1, min(5, vocab), min(20, vocab)]),
                "train": train, "temperature": rng.choice([0.5, 0.7, 1.0, 1.3]),
                "masked": rng.choice([0.0, 0.3]) if train and vocab < 256 else 0.0,
                "ignored": rng.choice([0.0, 0.1])}
    if op == "scan":
        dim = rng.choice([1, _log_int(rng, 1, 4096), _log_int(rng, 16, 4096), 8 * _log_int(rng, 2, 512)])
        batch = _log_int(rng, 1, 64)
        steps = _log_int(rng, 1, max(1, min(65521, (1 << 25) // (dim * batch))))
        return {"op": op, "batch": batch, "steps": steps, "dim": dim,
                "type": rng.choice(["fp32", "bf16", "fp16"]) if batch * steps * dim < 1 << 24 else "bf16",
                "gates": rng.choice(["decay", "logit"]), "mix": rng.choice([True, False]),
                "reverse": rng.choice([True, False]), "ragged": rng.choice([True, False]),
                "train": rng.choice([True, False])}
    if op == "step":
        return {"op": op, "batch": _log_int(rng, 1, 512), "dim": _log_int(rng, 8, 8192),
                "type": rng.choice(["fp32", "bf16", "fp16"]), "gates": rng.choice(["decay", "logit"]),
                "mix": rng.choice([True, False])}
    cols = _log_int(rng, 3, 8192)
    rows = _log_int(rng, 1, (1 << 26) // cols)
    return {"op": "dropout", "rows": rows, "cols": cols,
            "type": rng.choice(["fp32", "bf16", "fp16"]) if rows * cols < 1 << 25 else rng.choice(["bf16", "fp16"]),
            "p": rng.choice([0.05, 0.1, 0.25, 0.5]), "residual": rng.choice([True, False]), "train": rng.choice([True, False])}


# ---- inputs --------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dt = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=dev, dtype=torch.float32)

    st = {"case": dict(case)}
    if case["op"] == "logprob":
        n, v = case["rows"], case["vocab"]
        tokens = torch.randint(0, v, (n,), generator=gen, device=dev)
        logits = torch.empty(n, v, device=dev, dtype=dt)
        block = max(1, (1 << 26) // v)
        for i in range(0, n, block):        # blocks: a whole fp32 image of the largest case is not needed
            k = min(block, n - i)
            z = normal(k, v) * 2.5
            if case["masked"] > 0:
                z = torch.where(uniform(k, v) < case["masked"], torch.full_like(z, -math.inf), z)
                r = torch.arange(k, device=dev)     # the taken action is a legal one
                z[r, tokens[i:i + k]] = normal(k)
            logits[i:i + k] = z
        if case["ignored"] > 0:
            tokens = torch.where(uniform(n) < case["ignored"], torch.full_like(tokens, IGNORE), tokens)
        st.update(logits=logits.requires_grad_(case["train"]), tokens=tokens)
        if case["train"]:       # a policy gradient's weights: advantages and the entropy bonus
            st.update(d_logprob=normal(n) / n, d_entropy=torch.full((n,), -0.01 / n, device=dev))
    elif case["op"] in ("scan", "step"):
        step = case["op"] == "step"
        shape = (case["batch"], case["dim"]) if step else (case["batch"], case["steps"], case["dim"])
        if not step and case["dim"] == 1:
            # rewards of an episode: mostly nothing, now and then a point; gamma, and 0 where an episode ends
            x = torch.sign(normal(*shape)) * (uniform(*shape) < 0.05).float()
            gate = torch.where(uniform(*shape) < 1e-3, torch.zeros(shape, device=dev), torch.full(shape, 0.99, device=dev))
            if case["gates"] == "logit":
                gate = normal(*shape) + 2.0
        else:
            x = normal(*shape)
            gate = normal(*shape) * 1.5 + 2.0
            if case["gates"] == "decay":
                gate = torch.sigmoid(gate)
        train = not step and case["train"]
        st.update(x=x.to(dt).requires_grad_(train), gate=gate.to(dt).requires_grad_(train))
        state = normal(case["batch"], case["dim"])
        if step:
            st.update(state=state, next=torch.empty_like(state))    # two state buffers, swapped from token to token
        else:
            st.update(h0=state.requires_grad_(train), lengths=None)
            if case["ragged"]:
                t = case["steps"]
                low = max(0, t // 2)
                st["lengths"] = torch.randint(low, t + 1, (case["batch"],), generator=gen, device=dev)
            if train:
                st.update(d_h=normal(*shape).to(dt), d_last=normal(case["batch"], case["dim"]))
    else:
        shape = (case["rows"], case["cols"])
        st.update(x=normal(*shape).to(dt).requires_grad_(case["train"]), residual=None, seed=int(seed) * 7919 + 17,
                  site=3, counter=torch.full((1,), 1000 + int(seed) % 1000, dtype=torch.int64, device=dev))
        if case["residual"]:
            st["residual"] = normal(*shape).to(dt).requires_grad_(case["train"])
        if case["train"]:
            st["d_y"] = normal(*shape).to(dt)
    return st


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    c = st["case"]
    if c["op"] == "logprob":
        from pytorch_distributed_amd.ops.logprob import token_logprobs
        out = token_logprobs(st["logits"], st["tokens"], temperature=c["temperature"], top_k=c["top"], ignore_index=IGNORE)
        res = {"logprob": out.logprob, "entropy": out.entropy, "logsumexp": out.logsumexp}
        if c["top"]:
            res.update(top_logprobs=out.top_logprobs, top_tokens=out.top_tokens)
        if c["train"]:
            res["d_logits"], = torch.autograd.grad((out.logprob, out.entropy), (st["logits"],),
                                                   (st["d_logprob"], st["d_entropy"]))
            for k in ("logprob", "entropy", "logsumexp"):
                res[k] = res[k].detach()
        return res
    if c["op"] == "step":
        from pytorch_distributed_amd.ops.scan import linear_scan_step
        h = linear_scan_step(st["x"], st["gate"], st["state"], gates=c["gates"], mix=c["mix"], state_out=st["next"])
        return {"h": h, "state": st["next"]}
    if c["op"] == "scan":
        from pytorch_distributed_amd.ops.scan import linear_scan
        h, last = linear_scan(st["x"], st["gate"], st["h0"], gates=c["gates"], mix=c["mix"], reverse=c["reverse"],
                              lengths=st["lengths"])
        if not c["train"]:
            return {"h": h, "last": last}
        dx, dg, dh0 = torch.autograd.grad((h, last), (st["x"], st["gate"], st["h0"]), (st["d_h"], st["d_last"]))
        return {"h": h.detach(), "last": last.detach(), "d_x": dx, "d_gate": dg, "d_h0": dh0}
    from pytorch_distributed_amd.ops.dropout import dropout
    y = dropout(st["x"], c["p"], st["seed"], st["counter"], site=st["site"], residual=st["residual"])
    if not c["train"]:
        return {"y": y}
    leaves = [st["x"]] + ([st["residual"]] if c["residual"] else [])
    grads = torch.autograd.grad(y, leaves, st["d_y"])
    res = {"y": y.detach(), "d_x": grads[0]}
    if c["residual"]:
        res["d_residual"] = grads[1]
    return res


def _run_plain(st):
    with torch.no_grad():
        return {"logprob": _plain_logprob, "step": _plain_step, "scan": _plain_scan, "dropout": _plain_dropout}[
            st["case"]["op"]](st)


def _plain_logprob(st):
    c = st["case"]
    logits, tokens = st["logits"].detach(), st["tokens"]
    live = tokens != IGNORE
    tok = torch.where(live, tokens, torch.zeros_like(tokens))[:, None]
    z = logits.float()
    if c["temperature"] != 1.0:
        z = z / c["temperature"]
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    s = e.sum(1, keepdim=True)
    lse = m + torch.log(s)
    logp = z - lse
    p = e / s
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    entropy = -plogp.sum(1)
    zero = torch.zeros_like(entropy)
    res = {"logprob": torch.where(live, logp.gather(1, tok)[:, 0], zero), "entropy": torch.where(live, entropy, zero),
           "logsumexp": torch.where(live, lse[:, 0], zero)}
    if c["top"]:
        rest = logits.float()
        idx = torch.arange(c["vocab"], device=rest.device)[None, :]
        ids = []
        for _ in range(c["top"]):       # the largest that is left, the first of equals
            best = rest.amax(1, keepdim=True)
            first = torch.where(rest == best, idx, torch.full_like(idx, c["vocab"])).amin(1, keepdim=True)
            ids.append(first)
            rest = torch.where(idx == first, torch.full_like(rest, -math.inf), rest)
        ids = torch.cat(ids, 1)
        lp = logp.gather(1, ids)
        res["top_logprobs"] = torch.where(live[:, None], lp, torch.zeros_like(lp))
        res["top_tokens"] = torch.where(live[:, None], ids, torch.full_like(ids, -1))
    if c["train"]:
        dlp = torch.where(live, st["d_logprob"], zero)[:, None]
        dent = torch.where(live, st["d_entropy"], zero)[:, None]
        g = -dlp * p - dent * (plogp + p * entropy[:, None])
        g.scatter_add_(1, tok, dlp)
        res["d_logits"] = (g / c["temperature"]).to(logits.dtype)
    return res


def _gates(gate, x, c):
    """-> (a, u, 1 - a): h_t = a_t h_{t-1} + u_t"""
    if c["gates"] == "logit":
        a, keep = torch.sigmoid(gate), torch.sigmoid(-gate)
    else:
        a, keep = gate, 1 - gate
    return a, (keep * x if c["mix"] else x), keep


def _doubling(a, u):
    """h_t = a_t h_{t-1} + u_t over dim 1 from h = 0, in log2(T) sweeps over the whole sequence."""
    a, h = a.clone(), u.clone()
    k, t = 1, a.shape[1]
    while k < t:
        h[:, k:] += a[:, k:] * h[:, :-k].clone()
        a[:, k:] *= a[:, :-k].clone()
        k *= 2
    return h


def _order(st, t, dev):
    """For every step of the recurrence the position it reads, and whether that step exists."""
    c = st["case"]
    n = st["lengths"] if st["lengths"] is not None else torch.full((c["batch"],), t, device=dev)
    steps = torch.arange(t, device=dev)[None, :].expand(c["batch"], t)
    live = steps < n[:, None]
    pos = torch.where(live, n[:, None] - 1 - steps, steps) if c["reverse"] else steps
    return n, pos, live


def _plain_scan(st):
    c = st["case"]
    x0 = st["x"].detach()
    # 64 bits for 32-bit data: rounding a gate next to 1 is repeated over the whole memory of the recurrence
    wide = torch.float64 if x0.dtype == torch.float32 else torch.float32
    t = c["steps"]
    n, pos, live = _order(st, t, x0.device)
    idx = pos[:, :, None].expand_as(x0)
    lv = live[:, :, None]

    def along(v):       # into the recurrence's own order
        return torch.where(lv, v.to(wide).gather(1, idx) if c["reverse"] else v.to(wide), torch.zeros((), device=v.device, dtype=wide))

    def back(v):
        return v.gather(1, idx) if c["reverse"] else v

    x, g = along(x0), along(st["gate"].detach())
    a, u, keep = _gates(g, x, c)
    a, u = torch.where(lv, a, torch.zeros_like(a)), torch.where(lv, u, torch.zeros_like(u))
    h0 = st["h0"].detach().to(wide)
    u = u.clone()
    u[:, 0] += a[:, 0] * h0
    h = _doubling(a, u)
    at = (n - 1).clamp_min(0)[:, None, None].expand(-1, 1, c["dim"])
    last = torch.where((n > 0)[:, None], h.gather(1, at)[:, 0], h0)
    res = {"h": back(h).to(x0.dtype), "last": last.float()}
    if c["train"]:
        dh = along(st["d_h"])
        dlast = st["d_last"].to(wide)
        some = (n > 0)[:, None]
        dh = dh.scatter_add(1, at, torch.where(some, dlast, torch.zeros_like(dlast))[:, None])
        nxt = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
        gr = _doubling(nxt.flip(1), dh.flip(1)).flip(1)      # G_t = dh_t + a_{t+1} G_{t+1}
        gr = torch.where(lv, gr, torch.zeros_like(gr))
        prev = torch.cat([h0[:, None], h[:, :-1]], 1)
        da = gr * (prev - x if c["mix"] else prev)
        if c["gates"] == "logit":
            da = da * a * keep
        res["d_x"] = back(gr * keep if c["mix"] else gr).to(x0.dtype)
        res["d_gate"] = back(torch.where(lv, da, torch.zeros_like(da))).to(x0.dtype)
        res["d_h0"] = torch.where(some, a[:, 0] * gr[:, 0], dlast).float()
    return res


def _plain_step(st):
    c = st["case"]
    a, u, _ = _gates(st["gate"].float(), st["x"].float(), c)
    h = a * st["state"] + u
    return {"h": h.to(st["x"].dtype), "state": h}


def _signed(v):
    v &= (1 << 64) - 1
    return v - (1 << 64) if v >> 63 else v


def _mix_int(z):
    z &= (1 << 64) - 1
    z ^= z >> 33
    z = (z * MIX1) & ((1 << 64) - 1)
    z ^= z >> 33
    z = (z * MIX2) & ((1 << 64) - 1)
    return z ^ (z >> 33)


def _mix(z):
    """The 64-bit finaliser on a tensor of counters (int64 arithmetic wraps)."""
    def down(v):
        return (v >> 33) & 0x7FFFFFFF
    z = (z ^ down(z)) * _signed(MIX1)
    z = (z ^ down(z)) * _signed(MIX2)
    return z ^ down(z)


def _plain_dropout(st):
    c = st["case"]
    x = st["x"].detach()
    n = x.numel()
    dev = x.device
    # key of this call: seed, step counter (on the device) and site
    key = _mix(_signed(st["seed"]) + _signed(GOLDEN) * (1 + st["counter"]))
    key = _mix(key + _signed(GOLDEN * (1 + st["site"])))
    key2 = _mix(key)
    thr = min(int(round(c["p"] * 2.0 ** 48)), 1 << 48)
    hi, lo = thr >> 32, thr & 0xFFFFFFFF
    words = _mix(key + _signed(GOLDEN) * (1 + torch.arange((n + 3) // 4, device=dev)))
    u = torch.stack([(words >> (16 * j)) & 0xFFFF for j in range(4)], 1).reshape(-1)[:n]
    tie = (_mix(key2 + _signed(GOLDEN) * (1 + torch.arange(n, device=dev))) >> 32) & 0xFFFFFFFF
    keep = ((u > hi) | ((u == hi) & (tie >= lo))).reshape(x.shape)
    scale = 1.0 / (1.0 - c["p"])
    zero = torch.zeros((), device=dev)
    y = torch.where(keep, x.float() * scale, zero)
    if c["residual"]:
        y = y + st["residual"].detach().float()
    res = {"y": y.to(x.dtype)}
    if c["train"]:
        res["d_x"] = torch.where(keep, st["d_y"].float() * scale, zero).to(x.dtype)
        if c["residual"]:
            res["d_residual"] = st["d_y"].clone()
    return res


# ---- the work ------------------------------------------------------------------------------------------------------
def work(case):
    b = SIZES[case["type"]]
    if case["op"] == "logprob":
        n, v, k = case["rows"], case["vocab"], case["top"]
        nbytes = n * v * b + n * (8 + 12) + n * k * 12
        flops = 6 * n * v
        if case["train"]:
            nbytes += n * v * b + n * 8
            flops += 6 * n * v
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "scan":
        n, state = case["batch"] * case["steps"] * case["dim"], case["batch"] * case["dim"]
        per = 4 if case["gates"] == "logit" else 0
        nbytes, flops = 3 * n * b + 8 * state, (2 + per + (2 if case["mix"] else 0)) * n
        if case["train"]:       # + d_h read, d_x and d_gate written
            nbytes += 3 * n * b + 8 * state
            flops += (4 + per) * n
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "step":
        n = case["batch"] * case["dim"]
        return {"bytes": n * (3 * b + 8), "flops": 8 * n}
    n = case["rows"] * case["cols"]
    passes = 2 + (1 if case["residual"] else 0)
    if case["train"]:
        passes += 2             # d_y read, d_x written (the residual's gradient is d_y itself)
    return {"bytes": passes * n * b, "flops": 8 * n}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"logprob": _exact_logprob, "step": _exact_step, "scan": _exact_scan, "dropout": _exact_dropout}[
            case["op"]](st)


def _exact_logprob(st):
    c = st["case"]
    n, v, k = c["rows"], c["vocab"], c["top"]
    logits, tokens = st["logits"].detach(), st["tokens"]
    dev = logits.device
    out = {name: torch.zeros(n, dtype=torch.float64, device=dev) for name in ("logprob", "entropy", "logsumexp")}
    if k:
        out["top_logprobs"] = torch.zeros(n, k, dtype=torch.float64, device=dev)
        out["top_tokens"] = torch.full((n, k), -1, dtype=torch.int64, device=dev)
    if c["train"]:
        out["d_logits"] = torch.zeros(n, v, dtype=torch.float64, device=dev)
    block = max(1, (1 << 25) // v)
    for i in range(0, n, block):
        rows = torch.nonzero(tokens[i:i + block] != IGNORE)[:, 0] + i
        if rows.numel() == 0:
            continue
        raw = logits[rows]
        t = tokens[rows]
        r = torch.arange(rows.numel(), device=dev)
        q = torch.log_softmax(raw.double() / c["temperature"], 1)
        pr = q.exp()
        h = -torch.special.xlogy(pr, pr).sum(1)
        out["logprob"][rows] = q[r, t]
        out["entropy"][rows] = h
        out["logsumexp"][rows] = torch.logsumexp(raw.double() / c["temperature"], 1)
        if k:
            ids = torch.sort(raw.float(), dim=1, descending=True, stable=True)[1][:, :k]
            out["top_tokens"][rows] = ids
            out["top_logprobs"][rows] = q.gather(1, ids)
        if c["train"]:
            w, e = st["d_logprob"][rows].double(), st["d_entropy"][rows].double()
            g = -pr * w[:, None] - e[:, None] * (torch.special.xlogy(pr, pr) + pr * h[:, None])
            g[r, t] += w
            out["d_logits"][rows] = g / c["temperature"]
    return out


def _exact_scan(st):
    c = st["case"]
    x, g = st["x"].detach().double(), st["gate"].detach().double()
    bsz, t, d = x.shape
    n = (st["lengths"] if st["lengths"] is not None else torch.full((bsz,), t, device=x.device))[:, None]
    row = torch.arange(bsz, device=x.device)
    a = 1 / (1 + torch.exp(-g)) if c["gates"] == "logit" else g
    b = 1 / (1 + torch.exp(g)) if c["gates"] == "logit" else 1 - g
    h = torch.zeros_like(x)
    state = st["h0"].detach().double()
    hist = torch.empty(t, bsz, d, dtype=torch.float64, device=x.device)
    full = bool((n == t).all())

    def where(i):       # position of the i-th step of every sequence
        return (n[:, 0] - 1 - i).clamp_min(0) if c["reverse"] else torch.full_like(n[:, 0], i)

    for i in range(t):
        hist[i] = state
        if full:
            j = t - 1 - i if c["reverse"] else i
            state = a[:, j] * state + (b[:, j] * x[:, j] if c["mix"] else x[:, j])
            h[:, j] = state
            continue
        j = where(i)
        on = i < n
        nxt = a[row, j] * state + (b[row, j] * x[row, j] if c["mix"] else x[row, j])
        state = torch.where(on, nxt, state)
        h[row, j] = torch.where(on, state, h[row, j])
    res = {"h": h, "last": state}
    if c["train"]:
        dh = st["d_h"].double()
        dx, dg = torch.zeros_like(x), torch.zeros_like(x)
        carry = st["d_last"].double()
        for i in range(t - 1, -1, -1):
            j = where(i)
            on = i < n
            aj, xj = a[row, j], x[row, j]
            gr = carry + dh[row, j]
            da = gr * (hist[i] - xj if c["mix"] else hist[i])
            if c["gates"] == "logit":
                da = da * aj * b[row, j]
            dxj = gr * b[row, j] if c["mix"] else gr
            dx[row, j] = torch.where(on, dxj, dx[row, j])
            dg[row, j] = torch.where(on, da, dg[row, j])
            carry = torch.where(on, aj * gr, carry)
        res.update(d_x=dx, d_gate=dg, d_h0=carry)
    return res


def _exact_step(st):
    c = st["case"]
    x, g = st["x"].double(), st["gate"].double()
    a = 1 / (1 + torch.exp(-g)) if c["gates"] == "logit" else g
    b = 1 / (1 + torch.exp(g)) if c["gates"] == "logit" else 1 - g
    h = a * st["state"].double() + (b * x if c["mix"] else x)
    return {"h": h, "state": h}


def _exact_dropout(st):
    c = st["case"]
    x = st["x"].detach()
    n = x.numel()
    key = _mix_int(st["seed"] + GOLDEN * (1 + int(st["counter"].item())))
    key = _mix_int(key + GOLDEN * (1 + st["site"]))
    key2 = _mix_int(key)
    thr = min(int(round(c["p"] * 2.0 ** 48)), 1 << 48)

    def mixed(start, counters):
        z = np.uint64(start) + np.uint64(GOLDEN) * (counters.astype(np.uint64) + np.uint64(1))
        for m in (MIX1, MIX2):
            z ^= z >> np.uint64(33)
            z *= np.uint64(m)
        return z ^ (z >> np.uint64(33))

    with np.errstate(over="ignore"):
        u = mixed(key, np.arange((n + 3) // 4, dtype=np.uint64)).view(np.uint16)[:n]     # little-endian: bits 16 j first
        keep = u > (thr >> 32)
        even = np.nonzero(u == (thr >> 32))[0]
        keep[even] = (mixed(key2, even) >> np.uint64(32)) >= np.uint64(thr & 0xFFFFFFFF)
    keep = torch.from_numpy(keep).to(x.device).reshape(x.shape)
    y = x.double() * keep / (1.0 - c["p"])
    if c["residual"]:
        y = y + st["residual"].detach().double()
    res = {"y": y}
    if c["train"]:
        res["d_x"] = st["d_y"].double() * keep / (1.0 - c["p"])
        if c["residual"]:
            res["d_residual"] = st["d_y"].double()
    return res
