"""The operators between a GDN layer's projections and its residual
(include/kq_hip.h: causal convolution, linear attention, norms around a block)
from their definitions, row by row in binary64.

Sequences: spans [(begin, end)], slots, fresh (lists). Rows and slots that no
sequence has keep what the given outputs hold.
"""
import numpy as np

NO_SLOT = 0xFFFFFFFF


def sigmoid(x):
    x = np.asarray(x, np.float64)
    e = np.exp(-np.abs(x))
    return np.where(x >= 0, 1.0, e) / (1.0 + e)


def softplus(x):
    x = np.asarray(x, np.float64)
    return np.maximum(x, 0.0) + np.log1p(np.exp(-np.abs(x)))


def conv(x, w, bias, silu, state, spans, slots, fresh, y, state_out):
    x, w = x.astype(np.float64), w.astype(np.float64)
    y, state_out = y.astype(np.float64), state_out.astype(np.float64)
    taps = w.shape[1]
    for (a, b), slot, new in zip(spans, slots, fresh):
        if slot == NO_SLOT:
            continue
        st = state[slot].astype(np.float64)
        line = np.concatenate([np.zeros_like(st) if new else st, x[a:b]])
        for t in range(b - a):
            v = (line[t:t + taps] * w.T).sum(0) + (0 if bias is None else bias)
            y[a + t] = v * sigmoid(v) if silu else v
        state_out[slot] = line[b - a:]
    return y, state_out


def attention(q, k, v, alpha, beta, rate, bias, scale, eps, state, spans, slots, fresh, y,
              state_out):
    """q, k [rows][key heads][dk], v [rows][value heads][dv]; eps None: rows as
    they are; alpha, beta None as in the entry point."""
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    y, state_out = y.astype(np.float64), state_out.astype(np.float64)
    hv = v.shape[1]
    if eps is not None:
        q = q / np.sqrt((q * q).sum(-1, keepdims=True) + eps)
        k = k / np.sqrt((k * k).sum(-1, keepdims=True) + eps)
    q = q * scale
    head = np.arange(hv) // (hv // q.shape[1])
    rate = rate.astype(np.float64)
    for (a, b), slot, new in zip(spans, slots, fresh):
        if slot == NO_SLOT:
            continue
        S = np.zeros(state.shape[1:]) if new else state[slot].astype(np.float64)
        for t in range(a, b):
            g = rate
            if alpha is not None:
                g = rate * softplus(alpha[t].astype(np.float64) + (0 if bias is None else bias))
            S = S * np.exp(g)[:, None, None]
            kt, qt, d = k[t][head], q[t][head], v[t]
            if beta is not None:
                d = sigmoid(beta[t])[:, None] * (d - np.einsum("hij,hi->hj", S, kt))
            S = S + kt[:, :, None] * d[:, None, :]
            y[t] = np.einsum("hij,hi->hj", S, qt)
        state_out[slot] = S
    return y, state_out


def rms(x, eps):
    x = np.asarray(x, np.float64)
    # x / sqrt(mean + eps) without leaving the range of the squares
    m = np.maximum(np.abs(x).max(-1, keepdims=True), 1e-100)
    return x / (m * np.sqrt(((x / m) ** 2).mean(-1, keepdims=True) + eps / m / m))


def act(kind, g):
    return 1.0 if kind == "none" else sigmoid(g) * (g.astype(np.float64) if kind == "silu" else 1)


def gated_norm(x, w, offset, gate, kind, eps):
    y = rms(x, eps)
    if w is not None:
        y = y * (np.float64(np.float32(offset)) + w)
    return y * act(kind, gate)


def block_join(block, post, post_offset, gate, kind, scale, residual, branch_gate, pre,
               pre_offset, eps):
    y = block.astype(np.float64)
    if post is not None:
        y = rms(y, eps) * (post_offset + post.astype(np.float64))
    y = y * act(kind, gate)
    c = 1.0 if branch_gate is None else branch_gate.astype(np.float64)[:, :, None]
    r = residual.astype(np.float64) + scale * c * y[:, None, :]
    return r, None if pre is None else rms(r, eps) * (pre_offset + pre.astype(np.float64))
