"""The operators around the tree step restated on the CPU in 64 bits: the causal
convolution and the gated delta rule row by row, the accepted path node by
node."""
from __future__ import annotations

import numpy as np

STATUS_SPAN, STATUS_SLOT, STATUS_WEIGHT = 1, 32, 64


def spans(cu, batch, limit, rows):
    """[(first row, rows, status)] of every request."""
    out = []
    for b in range(batch):
        r0 = int(cu[b]) if cu is not None else b * limit
        n = int(cu[b + 1]) - r0 if cu is not None else limit
        status = STATUS_SPAN if n < 0 or n > limit or r0 < 0 or r0 + n > rows else 0
        there = 0 if r0 < 0 else max(rows - r0, 0)
        out.append((r0, min(max(n, 0), limit, there), status))
    return out


def _slots(indices, initial, slots, batch):
    """[(slot or -1, goes on from it, status)]"""
    out = []
    for b in range(batch):
        at = b if indices is None else int(indices[b])
        status = STATUS_SLOT if at >= slots else 0
        at = at if 0 <= at < slots else -1
        out.append((at, at >= 0 and (initial is None or bool(initial[b])), status))
    return out


def prompt_conv(x, conv_state, weight, bias, cu, *, batch, limit, silu=True, indices=None, initial=None):
    """(y, conv_state, status, magnitude): rows of no request are NaN; magnitude is the sum of the terms' sizes."""
    x, state, w = np.asarray(x, np.float64), np.array(conv_state, np.float64), np.asarray(weight, np.float64)
    W = w.shape[1]
    y, size = np.full(x.shape, np.nan), np.zeros(x.shape)
    status = np.zeros(batch, np.int32)
    old = state.copy()
    at = _slots(indices, initial, len(state), batch)
    for b, (r0, n, st) in enumerate(spans(cu, batch, limit, len(x))):
        slot, goes_on, st2 = at[b]
        status[b] = st | st2
        if n == 0:
            continue
        window = old[slot, :, :W - 1].T if goes_on else np.zeros((W - 1, x.shape[1]))
        line = np.concatenate([window, x[r0:r0 + n]])
        for t in range(n):
            terms = line[t:t + W] * w.T
            z = terms.sum(0) + (0 if bias is None else bias)
            size[r0 + t] = np.abs(terms).sum(0) + (0 if bias is None else np.abs(bias))
            with np.errstate(over="ignore"):
                y[r0 + t] = z / (1 + np.exp(-z)) if silu else z
        if slot >= 0 and W > 1:
            state[slot, :, :W - 1] = line[len(line) - (W - 1):].T
    return y, state, status, size


def prompt_gdn(y, a, b, rate, dt_bias, state, cu, *, hk, hv, batch, limit, scale=None, indices=None, initial=None):
    """(o, state, status) by the recurrence; state [slots, hv, k, v], rate = -exp(A_log); rows of no request are NaN."""
    y, state = np.asarray(y, np.float64), np.array(state, np.float64)
    D = state.shape[-1]
    scale = D ** -0.5 if scale is None else scale
    T = len(y)
    q, k, v = (np.array(p).reshape(T, -1, D) for p in np.split(y[:, :(2 * hk + hv) * D], [hk * D, 2 * hk * D], 1))
    q = q / np.sqrt((q * q).sum(2, keepdims=True) + 1e-6) * scale
    k = k / np.sqrt((k * k).sum(2, keepdims=True) + 1e-6)
    q, k = np.repeat(q, hv // hk, 1), np.repeat(k, hv // hk, 1)
    g = np.asarray(rate, np.float64) * np.logaddexp(0, np.asarray(a, np.float64)[:T, :hv] + dt_bias)
    with np.errstate(over="ignore"):
        beta = 1 / (1 + np.exp(-np.asarray(b, np.float64)[:T, :hv]))
    o, status = np.full((T, hv, D), np.nan), np.zeros(batch, np.int32)
    old = state.copy()
    at = _slots(indices, initial, len(state), batch)
    for r, (r0, n, st) in enumerate(spans(cu, batch, limit, T)):
        slot, goes_on, st2 = at[r]
        status[r] = st | st2
        if n == 0:
            continue
        S = old[slot].copy() if goes_on else np.zeros(state.shape[1:])
        for t in range(r0, r0 + n):
            S *= np.exp(g[t])[:, None, None]
            u = beta[t][:, None] * (v[t] - np.einsum("hkv,hk->hv", S, k[t]))
            S += k[t][:, :, None] * u[:, None]
            o[t] = np.einsum("hkv,hk->hv", S, q[t])
        if slot >= 0:
            state[slot] = S
    return o, state, status


def _row(p):
    p = np.asarray(p, np.float64)
    with np.errstate(invalid="ignore"):
        return np.where(p > 0, p, 0.0)


def accept(tokens, parent, probs, uniform, last, draft_probs=None, path_cols=16):
    """One request: (path, next token), path a list of nodes, token -1 where there is no weight."""
    n, V = len(tokens), probs.shape[1]
    if n == 0:
        return [], -1
    path = [0]
    while len(path) < path_cols:
        node = path[-1]
        r = p = _row(probs[node])
        q0 = None if draft_probs is None else _row(draft_probs[node])
        gone, off, chosen = [], 0.0, None
        for c in range(1, n):
            if max(int(parent[c]), 0) != node or c <= node or not 0 <= tokens[c] < V:
                continue
            t, u = int(tokens[c]), float(uniform[c])
            if q0 is None:
                here = 0.0 if t in gone else p[t]
                if u * (1 - off) < here:
                    chosen = c
                    break
                off += here
            else:
                q = q0 / (1 - off) if off < 1 else np.zeros(V)
                q[gone] = 0
                if u * q[t] < r[t]:
                    chosen = c
                    break
                rest = np.maximum(r - q, 0)
                if rest.sum() > 0:
                    r = rest / rest.sum()
                off += 0.0 if t in gone else q0[t]
            gone.append(t)
        if chosen is None:
            break
        path.append(chosen)
    else:
        r, gone = _row(probs[path[-1]]), []
        draft_probs = None
    if draft_probs is None and gone:
        rest = r.copy()
        rest[gone] = 0
        r = rest if rest.sum() > 0 else r
    cum = np.cumsum(r)
    if V == 0 or not cum[-1] > 0:
        return path, -1
    over = np.flatnonzero(cum > float(last) * cum[-1])
    return path, int(over[0]) if len(over) else int(np.flatnonzero(r > 0)[-1])
