"""Rotary positions, a paged cache and the attention over it (include/kq_hip.h)
from their definitions in binary64, one row and one head at a time.

A cache here: keys and values [pages][heads][page tokens][width] as values of
the cache's type in float32, a table of pages by slot and lengths by slot.
"""
import numpy as np

NO_SLOT = 0xFFFFFFFF


def bf16_bits(x):
    """float32 to bf16's bits, to nearest, ties to even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_values(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def to_bits(x, bf16):
    return bf16_bits(x) if bf16 else np.asarray(x, np.float32).astype(np.float16).view(np.uint16)


def to_values(bits, bf16):
    return bf16_values(bits) if bf16 else np.asarray(bits, np.uint16).view(np.float16).astype(
        np.float32)


def turn(x, positions, frequencies, magnitude=1.0, pairs=False):
    """x [rows][heads][width]; frequencies [dims / 2] float64. Also the magnitude
    of the terms that an output is the sum of."""
    x = np.asarray(x, np.float64)
    half = len(frequencies)
    # an angle of n radians is n mod 2 pi in extended precision
    angle = np.asarray(positions, np.longdouble)[:, None] * np.asarray(frequencies, np.longdouble)
    c = (np.cos(angle) * magnitude).astype(np.float64)[:, None, :]
    s = (np.sin(angle) * magnitude).astype(np.float64)[:, None, :]
    i = 2 * np.arange(half) if pairs else np.arange(half)
    j = i + 1 if pairs else i + half
    y, size = x.copy(), np.abs(x)
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., i] * s + x[..., j] * c
    size[..., i] = size[..., j] = abs(magnitude) * (np.abs(x[..., i]) + np.abs(x[..., j]))
    return y, size


def places(spans, slots, fresh, lengths):
    """(row, sequence, position) of every row of the call."""
    for s, ((a, b), slot) in enumerate(zip(spans, slots)):
        if slot == NO_SLOT:
            continue
        past = 0 if fresh is not None and fresh[s] else int(lengths[slot])
        for t in range(a, b):
            yield t, s, past + t - a


def attention(q, keys, values, table, lengths, spans, slots, fresh, scale, causal=True, window=0,
              sinks=None, gate=None, out=None):
    """q [rows][query heads][width] -> out [rows][query heads][width]; rows of
    nobody keep what `out` holds."""
    q = np.asarray(q, np.float64)
    page = keys.shape[2]
    group = q.shape[1] // keys.shape[1]
    out = np.array(out, np.float64)
    for s, ((a, b), slot) in enumerate(zip(spans, slots)):
        if slot == NO_SLOT or a == b:
            continue
        past = 0 if fresh is not None and fresh[s] else int(lengths[slot])
        n = past + b - a
        ids = np.asarray(table[slot][:-(-n // page)], np.int64)
        at = np.arange(n)[None, :]
        mine = past + np.arange(b - a)[:, None]
        seen = at <= mine if causal else at < n
        seen = np.broadcast_to(seen, (b - a, n))
        if window:
            seen = seen & (at > mine - window)
        for h in range(keys.shape[1]):
            k = keys[ids, h].reshape(-1, q.shape[2])[:n].astype(np.float64)
            v = values[ids, h].reshape(-1, q.shape[2])[:n].astype(np.float64)
            for x in range(h * group, (h + 1) * group):
                e = np.where(seen, scale * (q[a:b, x] @ k.T), -np.inf)
                top = e.max(1, keepdims=True)
                if sinks is not None:
                    top = np.maximum(top, float(sinks[x]))
                w = np.exp(e - top)
                total = w.sum(1, keepdims=True)
                if sinks is not None:
                    total = total + np.exp(float(sinks[x]) - top)
                out[a:b, x] = (w / total) @ v
        if gate is not None:
            g = np.asarray(gate[a:b], np.float64)
            out[a:b] *= np.where(g >= 0, 1.0, np.exp(-np.abs(g))) / (1 + np.exp(-np.abs(g)))
    return out
