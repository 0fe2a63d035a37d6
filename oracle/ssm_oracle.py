"""float64 restatement of the state-space block's operators (include/mdfri.h "Operators of a state-space language-model block"), one token after the
other, with first-order bounds of what float32 arithmetic may be off by: every function returns (value, slack), |float32 result - value| <= slack
before the result's own rounding.  U = 2^-24 is half a step of float32.  Test infrastructure."""
import numpy as np

U = 2.0**-24


def silu(v):
    return v / (1 + np.exp(-v))


def conv(x, weight, bias, act, lengths, row_off, state=None, slots=None, positions=None):
    """x (R, C) -> out (R, C) (NaN where no sequence is), slack; `state` (n, width, C) is updated in place."""
    w, c = weight.shape
    out, slack = np.full(x.shape, np.nan), np.zeros(x.shape)
    for b, n in enumerate(lengths):
        slot = b if slots is None else int(slots[b])
        if state is not None and not 0 <= slot < len(state):
            continue
        pos = 0 if positions is None or state is None else int(positions[b])
        seq = x[row_off[b]:row_off[b] + n]
        before = np.zeros((w - 1, c))
        for back in range(1, w):
            if state is not None and pos - back >= 0:
                before[w - 1 - back] = state[slot, (pos - back) % w]
        full = np.concatenate([before, seq])
        v, mag = np.zeros((n, c)), np.zeros((n, c))
        for k in range(w):
            v += weight[k] * full[k:k + n]
            mag += np.abs(weight[k] * full[k:k + n])
        if bias is not None:
            v, mag = v + bias, mag + np.abs(bias)
        # width + 1 rounded terms; the activation's slope is at most 1.1, its exponential is off by (|v| + 2) steps, its division by three
        s = (w + 1) * U * mag * 1.1
        if act:
            s = s + (2 * np.abs(v) + 8) * U * np.abs(silu(v)) + 1e-38
            v = silu(v)
        out[row_off[b]:row_off[b] + n], slack[row_off[b]:row_off[b] + n] = v, s
        if state is not None:
            for t in range(max(0, n - w), n):
                state[slot, (pos + t) % w] = seq[t]
    return out, slack


def scan(x, dt, a, b, c, lengths, row_off, d=None, dt_bias=None, state=None, slots=None, positions=None, split=0.0):
    """x (R, H, P), dt (R, H), b, c (R, G, N) -> y (R, H, P) (NaN where no sequence is), slack; `state` (n, H, P, N) is updated in place and its slack
    returned third (NaN: not written).  `split`: the relative size of what a product operand may be cut to (0: float32)."""
    R, H, P = x.shape
    G, N = b.shape[1:]
    rep = np.arange(H) // (H // G)
    y, slack = np.full(x.shape, np.nan), np.zeros(x.shape)
    hslack = None if state is None else np.full(state.shape, np.nan)
    with np.errstate(all="ignore"):
        for s, n in enumerate(lengths):
            slot = s if slots is None else int(slots[s])
            if (state is not None and not 0 <= slot < len(state)) or n == 0:
                continue
            pos = 0 if positions is None or state is None else int(positions[s])
            h = state[slot].copy() if state is not None and pos > 0 else np.zeros((H, P, N))
            ha, hg = np.abs(h), np.zeros((H, P, N))      # magnitudes, and magnitudes times the (relative) error of the decays behind them
            for t in range(n):
                r = row_off[s] + t
                v = dt[r] + (0 if dt_bias is None else dt_bias)
                delta = np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))
                rel = 12 + np.minimum(np.abs(v), 200)     # steps that softplus may be off by (it is 0, or v itself, far out)
                decay = np.exp(delta * a)[:, None, None]
                new = (delta[:, None] * x[r])[:, :, None] * b[r][rep][:, None, :]
                h = decay * h + new
                hg = decay * (hg + (np.abs(delta * a) * (rel + 4))[:, None, None] * ha) + rel[:, None, None] * np.abs(new)
                ha = decay * ha + np.abs(new)
                ct = c[r][rep][:, None, :]
                y[r] = (h * ct).sum(-1)
                slack[r] = (np.abs(ct) * (ha * ((24 + N + t) * U + split) + hg * U)).sum(-1)
                if d is not None:
                    y[r] += d[:, None] * x[r]
                    slack[r] += 2 * U * np.abs(d[:, None] * x[r])
            slack[row_off[s]:row_off[s] + n] += 1e-36
            if state is not None:
                state[slot] = h
                hslack[slot] = ha * (24 + n) * U + hg * U + 1e-36
    return y, slack, hslack


def block_norm(s, residual=None, gate=None, gate_act="silu", gate_first=False, post_weight=None, post_bias=None, groups=1, scale=1.0, scale_vec=None, pre_weight=None, pre_bias=None,
               eps=1e-6, center=False):
    """-> (r, slack) or None, (out, slack) or None"""
    act = {"none": lambda z: z, "silu": silu, "sigmoid": lambda z: 1 / (1 + np.exp(-z))}[gate_act]

    def norm(v, e, g, weight, bias):
        rows, dim = v.shape
        v, e = v.reshape(rows * g, -1), e.reshape(rows * g, -1)
        k = (v.shape[1] / 64 + 24) * U                    # a sum in 64 lanes and a tree
        if center:
            m = v.mean(1, keepdims=True)
            e = e + e.mean(1, keepdims=True) + k * np.abs(v).mean(1, keepdims=True)
            v = v - m
        ms = (v * v).mean(1, keepdims=True)
        q = 1 / np.sqrt(ms + eps)
        eq = q**3 * ((np.abs(v) * e).mean(1, keepdims=True) + k * ms) + 4 * U * q
        out, eo = v * q, e * q + np.abs(v) * eq + 2 * U * np.abs(v * q)
        out, eo = out.reshape(rows, dim) * weight, eo.reshape(rows, dim) * np.abs(weight)
        if bias is not None:
            out = out + bias
        return out, eo + 2 * U * (np.abs(out) + (0 if bias is None else np.abs(bias)))

    v, e = s, np.zeros(s.shape)

    def gated(v, e):
        a = act(gate)
        return v * a, e * np.abs(a) + np.abs(v * a) * (2 * np.abs(gate) + 10) * U

    if gate is not None and gate_first:
        v, e = gated(v, e)
    if post_weight is not None:
        v, e = norm(v, e, groups, post_weight, post_bias)
    if gate is not None and not gate_first:
        v, e = gated(v, e)
    r = None
    if residual is not None:
        k = scale * (1 if scale_vec is None else scale_vec)
        e = e * np.abs(k) + 4 * U * (np.abs(k * v) + np.abs(residual))
        v = residual + k * v
        r = (v, e)
    if pre_weight is not None:
        v, e = norm(v, e, 1, pre_weight, pre_bias)
    return r, (v, e) if pre_weight is not None or residual is None else None
