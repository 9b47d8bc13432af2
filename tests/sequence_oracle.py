"""64-bit definitions of the sequence-policy operators, with bounds on what 32-bit arithmetic may leave (shared by
test_sequence_ops.py's cases; numpy, written from the formulas)."""
import numpy as np

U = 2.0 ** -24      # half a step of fp32, relative


def half_step(dtype_eps, x, tiny):
    """One rounding to the output type: half a step relative to the value, or of the smallest subnormal."""
    return dtype_eps / 2 * np.abs(x) + tiny / 2


# ---- token log-probabilities ---------------------------------------------------------------------------------------
def logprob(x, tokens, T, ignore, d_lp=None, d_ent=None, d_lse=None):
    """x (N, V) float64 -> dict of values and of bounds (key + '_tol') for finite rows; special rows as defined."""
    n, v = x.shape
    out = {k: np.zeros(n) for k in ("lp", "ent", "lse")}
    tol = {k: np.zeros(n) for k in out}
    g, gtol = np.zeros((n, v)), np.zeros((n, v))
    for r in range(n):
        t = int(tokens[r])
        if t == ignore:
            continue
        row = x[r]
        known = 0 <= t < v
        if np.isnan(row).any() or (row == np.inf).any():
            out["lp"][r] = out["ent"][r] = out["lse"][r] = np.nan
            g[r] = np.nan
            continue
        m = row.max()
        if m == -np.inf:
            out["lp"][r], out["lse"][r] = (-np.inf if known else np.nan), -np.inf
            continue
        with np.errstate(over="ignore", invalid="ignore"):
            d = (row - m) / T
            e = np.exp(d)
        s = e.sum()
        p = e / s
        dd = np.where(p > 0, d, 0.0)
        ls = np.log(s)
        h = ls - (p * dd).sum()
        lpi = d - ls
        e1, e2 = (p * -dd).sum(), (p * dd * dd).sum()
        # 32 bits: x - m, 1 / T and the product leave 3 U |d| in an exponent, the exponential 2 U |d| + 2 steps; a sum of
        # v terms leaves at most v U (any order), the logarithm 2 steps of |log s| + 2 U
        rel_s = U * (5 * e1 + 4 + v)
        ls_tol = rel_s + U * (4 * abs(ls) + 4)
        h_tol = ls_tol + U * (8 * e2 + (v + 12) * e1) + rel_s * e1 + 2 * U * abs(h)
        out["lp"][r] = lpi[t] if known else np.nan
        tol["lp"][r] = ls_tol + 4 * U * abs(d[t]) + U * abs(lpi[t]) if known and np.isfinite(d[t]) else 0.0
        out["ent"][r], tol["ent"][r] = h, h_tol
        out["lse"][r] = m / T + ls
        tol["lse"][r] = ls_tol + U * (2 * abs(m / T) + abs(m / T + ls))
        a = d_lp[r] if d_lp is not None else 0.0
        b = d_ent[r] if d_ent is not None else 0.0
        c = d_lse[r] if d_lse is not None else 0.0
        lpf = np.where(p > 0, lpi, 0.0)
        k = c - a - b * (lpf + h)
        g[r] = p * k
        lp_tol = ls_tol + 4 * U * np.abs(dd) + U * np.abs(lpf)
        mag = abs(c) + abs(a) + abs(b) * (np.abs(lpf) + abs(h))
        gtol[r] = p * (mag * (lp_tol + U * (2 * np.abs(lpf) + 8)) + abs(b) * (lp_tol + h_tol))
        if known:
            g[r, t] += a
            gtol[r, t] += 2 * U * abs(a)
        else:
            g[r] = np.nan
        g[r] /= T
        gtol[r] = gtol[r] / T + 3 * U * np.abs(g[r])
    return out, tol, g, gtol


def top(x, k):
    """Indices of the k best per row: larger first, NaN above all, the lower index of equals first."""
    idx = np.arange(x.shape[1])
    return np.stack([sorted(idx, key=lambda i: (not np.isnan(row[i]), -row[i] if not np.isnan(row[i]) else 0.0, i))[:k]
                     for row in x]).reshape(x.shape[0], k)


# ---- linear recurrence ---------------------------------------------------------------------------------------------
def scan(x, gate, h0, lengths, logit, mix, reverse, dh=None, dlast=None):
    """x, gate (B, T, D) float64 -> values and bounds.  Bounds: every product of gates and every sum of the recurrence is
    rounded once per step it passes, so the error obeys the recurrence itself with K U (|a| bar h + |u|) added per step,
    bar h being the recurrence of the absolute values; joining partial scans adds at most 32 roundings of bar h."""
    B, T, D = x.shape
    n = np.full(B, T) if lengths is None else np.clip(lengths, 0, T)
    a = 1 / (1 + np.exp(-gate)) if logit else gate
    c = 1 / (1 + np.exp(gate)) if logit else 1 - gate
    # relative error of a gate: exp of |g| (2 |g| + 2 steps), a sum, a reciprocal
    K = 16 + (2 * np.nanmax(np.abs(gate), initial=0.0) if logit else 0)
    K = min(K, 200.0)
    h, h_tol = np.zeros_like(x), np.zeros_like(x)
    last, last_tol = np.zeros((B, D)), np.zeros((B, D))
    dx, dg, dx_tol, dg_tol = (np.zeros_like(x) for _ in range(4))
    dh0, dh0_tol = np.zeros((B, D)), np.zeros((B, D))
    for b in range(B):
        order = list(range(n[b]))
        if reverse:
            order.reverse()
        s = np.zeros(D) if h0 is None else h0[b].copy()
        bar, err = np.abs(s), np.zeros(D)
        prev, prev_bar, prev_err = {}, {}, {}
        for t in order:
            prev[t], prev_bar[t], prev_err[t] = s, bar, err
            u = c[b, t] * x[b, t] if mix else x[b, t]
            s = a[b, t] * s + u
            bar = np.abs(a[b, t]) * bar + np.abs(u)
            err = np.abs(a[b, t]) * err + K * U * (bar + np.abs(c[b, t]) * prev_bar[t])
            h[b, t], h_tol[b, t] = s, err + 32 * U * bar
        last[b], last_tol[b] = s, err + 32 * U * bar
        gr = np.zeros(D) if dlast is None else dlast[b].copy()
        bar, err = np.abs(gr), np.zeros(D)
        for t in reversed(order):
            if dh is not None:
                gr = gr + dh[b, t]
                bar = bar + np.abs(dh[b, t])
            err = err + K * U * bar
            e = err + 32 * U * bar
            f = c[b, t] if mix else 1.0
            dx[b, t], dx_tol[b, t] = gr * f, np.abs(f) * (e + K * U * bar)
            w = prev[t] - x[b, t] if mix else prev[t]
            wbar = prev_bar[t] + (np.abs(x[b, t]) if mix else 0)
            werr = prev_err[t] + 34 * U * wbar
            q = a[b, t] * c[b, t] if logit else 1.0
            dg[b, t] = gr * w * q
            dg_tol[b, t] = np.abs(q) * (e * wbar + bar * werr + 2 * K * U * bar * wbar)
            gr, bar, err = a[b, t] * gr, np.abs(a[b, t]) * bar, np.abs(a[b, t]) * err + K * U * bar
        dh0[b], dh0_tol[b] = gr, err + 32 * U * bar
    return {"h": (h, h_tol), "last": (last, last_tol), "dx": (dx, dx_tol), "dg": (dg, dg_tol), "dh0": (dh0, dh0_tol)}


# ---- counter-based dropout -----------------------------------------------------------------------------------------
_M64 = (1 << 64) - 1
_G = 0x9E3779B97F4A7C15


def _mix(z):
    z &= _M64
    for m in (0xFF51AFD7ED558CCD, 0xC4CEB9FE1A85EC53):
        z ^= z >> 33
        z = z * m & _M64
    return z ^ z >> 33


def keep_mask(indices, p, seed, counter, site):
    """The mask at the given element indices, in Python integers."""
    key = _mix(_mix(seed + _G * (1 + counter)) + _G * (1 + site))
    key2 = _mix(key)
    thr = min(int(round(p * 2.0 ** 48)), 1 << 48)
    out = []
    for i in indices:
        u = _mix(key + _G * (1 + i // 4)) >> 16 * (i % 4) & 0xFFFF
        tie = _mix(key2 + _G * (1 + i)) >> 32
        out.append((u << 32 | tie) >= thr)
    return np.array(out)
