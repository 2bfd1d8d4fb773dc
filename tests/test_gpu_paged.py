"""Rotary positions, appending to a paged cache and the attention over it, on
the device, against their definitions in binary64 (tests/paged64.py).

Bars, from the arithmetic (u = 2^-24, half a step of binary32):
- rotation: an angle's quarter turns are exact to far below u; their fraction is
  rounded once (|r| < 1: u / 2), the series of its sine and cosine are 2 u off,
  the magnitude, the product and the sum round once each: at most 6 u of
  |m| (|x_i| + |x_j|), 8 u allowed;
- a value in the cache: half a step of its type besides, eps / 2 of the value, or
  of the type's smallest normal number below it;
- attention: a score's terms are products of a query held to 2^-22 of itself (the
  factor, two fp16 numbers) and a key held exactly, so that the score, in units of
  log2, is off by at most a few 2^-22 of the 2-norm of its terms, below 2^-20
  where scores are of the order of 1; that is a weight's relative error, and
  weights are held to 2^-22 again. Errors of independent sign leave the 2-norm of
  the output's error within 2e-6 of the output's where |scores| stay below 8, in
  proportion to the largest score above it; a single element's error has the
  root-mean-square of the others' and stays within 15 of it among a few million:
  3e-5 of max(|y|, rms y).
"""
import ctypes as C

import numpy as np
import pytest

import kq_hip
import paged64
from test_gpu_gdn import Call, Gen, capture, ctx, near, put, say, table  # noqa: F401

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SENTINEL = np.float32(-1234.5)
NO = paged64.NO_SLOT
NAN = 0x7FFF  # of both types
TYPES = {"f16": (kq_hip.TYPE_F16, False), "bf16": (kq_hip.TYPE_BF16, True)}


def u32(c, a):
    return None if a is None else c.up(np.asarray(a, np.uint32))


# ------------------------------------------------------------------ rotary


def rotary_case(ctx, rows, heads, width, dims, pairs, positions, magnitude=1.0, pad=0, shift=0,
                in_place=False, base=1e4):
    g = Gen(rows + dims)
    xs = heads * width + pad
    x = g.normal(rows * xs + shift)
    freq, _ = kq_hip.rotary_frequencies(dims, base)
    at = np.arange(rows) if positions is None else positions
    view = x[shift:].reshape(rows, xs)[:, :heads * width].reshape(rows, heads, width)
    want, size = paged64.turn(view, at, freq, magnitude, pairs)
    with Call(ctx) as c:
        r = kq_hip.rotary(dims, c.up(freq), "pairs" if pairs else "halves", magnitude)
        px = c.up(x) + 4 * shift
        out = x.copy() if in_place else np.full(x.shape, SENTINEL)
        py = px if in_place else c.up(out) + 4 * shift
        ctx.rotary(r, heads, width, rows, u32(c, positions), px, xs, py, xs)
        got = c.down(py - 4 * shift, out)
    rest = got[shift:].reshape(rows, xs)[:, heads * width:]
    assert np.array_equal(rest, out[shift:].reshape(rows, xs)[:, heads * width:])
    assert np.array_equal(got[:shift], out[:shift])
    got = got[shift:].reshape(rows, xs)[:, :heads * width].reshape(rows, heads, width)
    assert (np.abs(got - want) <= 8 * U * size).all()
    assert np.array_equal(got[..., dims:], view[..., dims:])


@pytest.mark.parametrize("rows", [1, 3, 4, 5, 130])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("heads,width,dims", [(1, 2, 2), (3, 64, 64), (2, 80, 34), (16, 128, 64),
                                              (5, 96, 96), (1, 1024, 1024), (2, 7, 6), (40, 256, 8)])
def test_rotary(ctx, rows, pairs, heads, width, dims):  # noqa: F811
    say("rotary", rows, pairs, heads, width, dims)
    rotary_case(ctx, rows, heads, width, dims, pairs, None)
    rotary_case(ctx, rows, heads, width, dims, pairs, None, in_place=True, pad=4)
    rotary_case(ctx, rows, heads, width, dims, pairs, None, magnitude=1.25, pad=3, shift=1)


@pytest.mark.parametrize("pairs", [False, True])
def test_rotary_positions(ctx, pairs):  # noqa: F811
    # far ones, in any order, some twice; quarter turns and their neighbours
    say("positions", pairs)
    at = np.array([0, 1, 2, (1 << 24) - 1, 1 << 20, 7, 7, 131071, 1000003], np.uint32)
    rotary_case(ctx, len(at), 3, 128, 128, pairs, at)
    rotary_case(ctx, len(at), 3, 128, 128, pairs, at, base=1e6, magnitude=0.5)


def test_rotary_quarter_turns(ctx):  # noqa: F811
    say("quarter turns")
    freq = np.array([np.pi / 2, np.pi / 4, np.pi, 0.0, 2.0, 1e-12, 100.0, -0.3])
    at = np.arange(64, dtype=np.uint32)
    x = Gen(3).normal(64, 1, 16)
    want, size = paged64.turn(x, at, freq)
    with Call(ctx) as c:
        y = c.up(np.zeros_like(x))
        ctx.rotary(kq_hip.rotary(16, c.up(freq)), 1, 16, 64, u32(c, at), c.up(x), 16, y, 16)
        got = c.down(y, x)
    assert (np.abs(got - want) <= 8 * U * size).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("where", ["turned", "passed", "frequency"])
def test_rotary_non_finite(ctx, bad, where):  # noqa: F811
    say("non-finite", bad, where)
    x = Gen(4).normal(6, 2, 16)
    freq = np.ones(4)
    if where == "frequency":
        freq[2] = bad
    else:
        x[5, 1, 3 if where == "turned" else 15] = bad
    with Call(ctx) as c:
        out = np.full(x.shape, SENTINEL)
        y = c.up(out)
        with pytest.raises(kq_hip.KqError) as e:
            ctx.rotary(kq_hip.rotary(8, c.up(freq)), 2, 16, 6, None, c.up(x), 32, y, 32)
        assert e.value.name == "NUMERIC_DOMAIN"
        assert (c.down(y, out) == SENTINEL).all()


# ------------------------------------------------------------------- cache


class Cache:
    """A pool of pages for sequences of these lengths (with `rows` more to come),
    NaN wherever no token lies, and page numbers that do not exist where a line
    of the table has no page."""

    def __init__(self, seed, type_, heads, width, page, past, rows, slot_count=None, slots=None,
                 scale=1.0, line=None):
        self.type_id, self.bf16 = TYPES[type_]
        self.heads, self.width, self.page = heads, width, page
        n = len(past)
        self.slot_count = n if slot_count is None else slot_count
        self.slots = list(range(n)) if slots is None else slots
        g = Gen(seed)
        held = [-(-(a + b) // page) for a, b in zip(past, rows)]
        self.pages = sum(held) + 2
        self.line = (max(held) + 1) if line is None else line
        order = g.r.permutation(self.pages).tolist()
        self.table = np.full((self.slot_count, self.line), 0xFFFFFFFF, np.uint32)
        self.lengths = np.full(self.slot_count, 0xFFFFFFF0, np.uint32)
        self.keys = np.full((self.pages, heads, page, width), NAN, np.uint16)
        self.values = self.keys.copy()
        self.past, self.rows = list(past), list(rows)
        for s, (a, b) in enumerate(zip(past, rows)):
            slot = self.slots[s]
            if slot == NO:
                continue
            ids = [order.pop() for _ in range(held[s])]
            self.table[slot, :held[s]] = ids
            self.lengths[slot] = a
            for pool in (self.keys, self.values):
                self._fill(pool, ids, 0, a + b, g, scale)

    def _fill(self, pool, ids, first, end, g, scale):
        for i, p in enumerate(ids):
            a, b = max(first, i * self.page), min(end, (i + 1) * self.page)
            if a < b:
                v = g.normal(self.heads, b - a, self.width, scale=scale)
                pool[p, :, a - i * self.page:b - i * self.page] = paged64.to_bits(v, self.bf16)

    def describe(self, c, keys=None, values=None, table_=None, lengths=None):
        up = lambda a, b: c.up(b) if a is None else a  # noqa: E731
        return kq_hip.paged_cache(self.type_id, self.heads, self.width, self.page, self.pages,
                                  self.line, up(keys, self.keys), up(values, self.values),
                                  up(table_, self.table), up(lengths, self.lengths))

    def floats(self):
        return paged64.to_values(self.keys, self.bf16), paged64.to_values(self.values, self.bf16)


def append_case(ctx, type_, heads, width, page, past, rows, offsets=True, slots=None,  # noqa: F811
                slot_count=None, fresh=None, dims=None, pairs=False, hq=0, pad=0, in_place=False,
                lead=0, gap=0):
    g = Gen(width + page + len(past))
    if offsets:
        off, spans, total = table(rows, lead, gap)
    else:
        off, total = None, len(past)
        spans = [(i, i + 1) for i in range(total)]
    k = Cache(7, type_, heads, width, page, past, [0] * len(past), slot_count, slots,
              line=max(-(-(a + b) // page) for a, b in zip(past, rows)) + 1)
    # pages for the rows to come, whatever the cache held there before
    spare = iter(range(k.pages, 1 << 30))
    for s, (a, b) in enumerate(zip(past, rows)):
        slot = k.slots[s]
        if slot == NO:
            continue
        start = 0 if fresh is not None and fresh[s] else a
        for i in range(-(-(start + b) // page)):
            if k.table[slot, i] == 0xFFFFFFFF:
                k.table[slot, i] = next(spare)
    more = next(spare) - k.pages
    k.pages += more
    grow = lambda a: np.concatenate([a, np.full((more, *a.shape[1:]), NAN, np.uint16)])  # noqa: E731
    k.keys, k.values = grow(k.keys), grow(k.values)
    w, qw = heads * width, hq * width
    stride = 2 * w + qw + pad
    qkv = g.normal(total, stride)
    mine = np.zeros(total, bool)
    for (a, b), s in zip(spans, k.slots):
        mine[a:b] = s != NO
    qkv[~mine] = np.nan  # rows of nobody are not looked at
    freq = None
    if dims:
        freq, _ = kq_hip.rotary_frequencies(dims, 1e4)
    want_k, want_v = (a.astype(np.float64) for a in k.floats())
    bar_k, bar_v = np.zeros_like(want_k), np.zeros_like(want_v)
    half_step = 2.0 ** -8 if k.bf16 else 2.0 ** -11
    tiny = 2.0 ** -126 if k.bf16 else 2.0 ** -14
    turn = lambda x, p: (paged64.turn(x, [p], freq, 1.25, pairs) if dims  # noqa: E731
                         else (x.astype(np.float64), np.zeros_like(x)))
    want_q = np.full((total, hq, width), SENTINEL, np.float64)
    bar_q = np.zeros_like(want_q)
    touched = np.zeros(want_k.shape, bool)
    for t, s, pos in paged64.places(spans, k.slots, fresh, k.lengths):
        at = (k.table[k.slots[s], pos // page], slice(None), pos % page)
        y, size = turn(qkv[t, :w].reshape(1, heads, width), pos)
        want_k[at], touched[at] = y[0], True
        bar_k[at] = 8 * U * size[0] + half_step * np.maximum(np.abs(y[0]), tiny) * (1 + 2 ** -10)
        v = qkv[t, w:2 * w].reshape(heads, width)
        want_v[at] = v
        bar_v[at] = half_step * np.maximum(np.abs(v), tiny)
        if hq:
            y, size = turn(qkv[t, 2 * w:2 * w + qw].reshape(1, hq, width), pos)
            want_q[t], bar_q[t] = y[0], 8 * U * size[0]
    with Call(ctx) as c:
        pk, pv = c.up(k.keys), c.up(k.values)
        seqs = kq_hip.sequences(total, len(past), k.slot_count, u32(c, off),
                                u32(c, slots), u32(c, fresh))
        p = c.up(qkv)
        out = np.full((total, qw + 4), SENTINEL)
        q_in = p + 8 * w
        po, os = (q_in, stride) if in_place else (c.up(out), qw + 4)
        inp = kq_hip.cache_rows(p, stride, p + 4 * w, stride, hq, q_in if hq else None, stride,
                                po if hq else None, os)
        rot = kq_hip.rotary(dims, c.up(freq), "pairs" if pairs else "halves", 1.25) if dims else None
        ctx.cache_append(k.describe(c, pk, pv), seqs, inp, rot)
        gk, gv = c.down(pk, k.keys), c.down(pv, k.values)
        if in_place:
            back = c.down(p, qkv)
            assert np.array_equal(back[:, :2 * w], qkv[:, :2 * w], equal_nan=True)
            gq = back[:, 2 * w:2 * w + qw]
            gq[~mine] = SENTINEL
        else:
            gq = c.down(po, out)
            assert (gq[:, qw:] == SENTINEL).all()
            gq = gq[:, :qw]
    assert np.array_equal(gk[~touched], k.keys[~touched])
    assert np.array_equal(gv[~touched], k.values[~touched])
    fk, fv = paged64.to_values(gk, k.bf16), paged64.to_values(gv, k.bf16)
    assert (np.abs(fk[touched] - want_k[touched]) <= bar_k[touched]).all()
    assert (np.abs(fv[touched] - want_v[touched]) <= bar_v[touched]).all()
    # values, and keys without a rotation, are rounded to nearest, ties to even
    assert np.array_equal(gv[touched], paged64.to_bits(want_v[touched].astype(np.float32), k.bf16))
    if not dims:
        assert np.array_equal(gk[touched],
                              paged64.to_bits(want_k[touched].astype(np.float32), k.bf16))
    if hq:
        assert (np.abs(gq.reshape(want_q.shape) - want_q) <= bar_q).all()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("width,page", [(64, 16), (128, 64), (256, 32), (64, 256), (128, 128)])
@pytest.mark.parametrize("n", [1, 4, 7])
def test_append_single_rows(ctx, type_, width, page, n):  # noqa: F811
    say("append single rows", type_, width, page, n)
    past = [(i * 37 + page - 1) % 300 for i in range(n)]
    slots = np.random.default_rng(n).permutation(n + 2)[:n].tolist()
    append_case(ctx, type_, 2, width, page, past, [1] * n, False, slots, n + 2,
                [i % 3 == 1 for i in range(n)], dims=width, hq=6)
    append_case(ctx, type_, 3, width, page, past, [1] * n, False, dims=width // 2, pairs=True, pad=4)


@pytest.mark.parametrize("rows", [[1], [5], [0], [16, 1, 0, 33, 2], [3, 0, 0, 70, 1, 1, 9]],
                         ids=str)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dims,pairs", [(None, False), (64, False), (64, True), (6, True),
                                        (30, False)])
def test_append_sequences(ctx, rows, type_, dims, pairs):  # noqa: F811
    say("append sequences", rows, type_, dims, pairs)
    n = len(rows)
    past = [(i * 29) % 50 for i in range(n)]
    slots = np.random.default_rng(n).permutation(n + 1)[:n].tolist()
    if n > 4:
        slots[3] = NO
    append_case(ctx, type_, 2, 64, 16, past, rows, True, slots, n + 1, [i % 2 for i in range(n)],
                dims, pairs, hq=4, lead=3, gap=2)
    # (a call has a row at least)
    append_case(ctx, type_, 2, 64, 16, past, rows, True, None, None, None, dims, pairs, hq=4,
                in_place=True, gap=int(sum(rows) == 0))
    append_case(ctx, type_, 1, 64, 32, past, rows, True, None, None, None, dims, pairs,
                lead=int(sum(rows) == 0))


def test_append_many_sequences(ctx):  # noqa: F811
    say("append many sequences")
    rows = [1, 0, 2, 1] * 70 + [40, 0, 0, 1]
    n = len(rows)
    append_case(ctx, "f16", 1, 64, 16, [(i * 7) % 33 for i in range(n)], rows, dims=64, hq=1,
                slots=np.random.default_rng(5).permutation(n).tolist(), slot_count=n, lead=1, gap=2)


def appending(ctx, k, rows, off, slots, count, qkv, dims=0):  # noqa: F811
    """The status of an append of `rows` rows of one key and value head."""
    with Call(ctx) as c:
        pk = c.up(k.keys)
        seqs = kq_hip.sequences(rows, count, k.slot_count, u32(c, off), u32(c, slots))
        p = c.up(qkv)
        inp = kq_hip.cache_rows(p, qkv.shape[1], p + 4 * k.width, qkv.shape[1])
        rot = kq_hip.rotary(dims, c.up(np.ones(dims // 2))) if dims else None
        with pytest.raises(kq_hip.KqError) as e:
            ctx.cache_append(k.describe(c, keys=pk), seqs, inp, rot)
        return e.value.name, c.down(pk, k.keys)


@pytest.mark.parametrize("what", ["slot", "slot twice", "page", "line", "length", "offsets",
                                  "offsets back"])
def test_append_bad_indexes(ctx, what):  # noqa: F811
    say("append bad", what)
    k = Cache(1, "f16", 1, 64, 16, [10, 20, 30], [6, 6, 2])
    off, slots = [0, 6, 12, 14], [0, 1, 2]
    if what == "slot":
        slots[1] = 3
    elif what == "slot twice":
        slots[2] = 0
    elif what == "page":
        k.table[1, 1] = k.pages
    elif what == "line":
        k.lengths[1] = k.line * 16 - 5
    elif what == "length":
        k.lengths[1] = 0xFFFFFFFF
    elif what == "offsets":
        off[3] = 15
    else:
        off[1], off[2] = 12, 6
    before = k.keys.copy()
    name, after = appending(ctx, k, 14, off, slots, 3, Gen(2).normal(14, 128))
    assert name == "INVALID_ARGUMENT"
    # nothing but the places of the call's own rows was written
    for s, (a, b) in enumerate([(10, 6), (20, 6), (30, 2)]):
        for pos in range(a, a + b):
            p = k.table[s, pos // 16]
            if p < k.pages:
                before[p, :, pos % 16] = after[p, :, pos % 16] = 0
    if what not in ("offsets back", "slot twice"):
        assert np.array_equal(before, after)


@pytest.mark.parametrize("type_,value", [("f16", np.nan), ("f16", 65520.0), ("bf16", np.inf),
                                         ("bf16", 3.4e38), ("f16", -1e6)])
@pytest.mark.parametrize("part", ["key", "value"])
@pytest.mark.parametrize("dims", [0, 64])
def test_append_out_of_the_type(ctx, type_, value, part, dims):  # noqa: F811
    say("append out of the type", type_, value, part, dims)
    k = Cache(1, type_, 1, 64, 16, [3], [5])
    qkv = Gen(2).normal(5, 128)
    qkv[4, 7 if part == "key" else 64 + 9] = value
    if dims:  # a rotation by 0: position 0 of a frequency 1
        k.lengths[0] = 0
    assert appending(ctx, k, 5, [0, 5], None, 1, qkv, 0 if part == "key" else dims)[0] == \
        "NUMERIC_DOMAIN"


# --------------------------------------------------------------- attention


class Attention:
    def __init__(self, seed, type_, heads, group, width, page, past, rows, slots=None,
                 slot_count=None, lead=0, gap=0, offsets=True, causal=True, window=0, sinks=False,
                 gate=False, pad=0, scale=None, kscale=1.0, line=None):
        self.k = Cache(seed, type_, heads, width, page, past, rows, slot_count, slots, kscale, line)
        self.hq = heads * group
        if offsets:
            self.off, self.spans, self.total = table(rows, lead, gap)
        else:
            self.off, self.total = None, len(rows)
            self.spans = [(i, i + 1) for i in range(self.total)]
        g = Gen(seed + 1)
        self.w = self.hq * width
        self.q = g.normal(self.total, self.w + pad)
        self.gate = g.normal(self.total, self.w + 4, scale=2.0) if gate else None
        self.sinks = g.normal(self.hq) if sinks else None
        self.scale = np.float32(width ** -0.5 if scale is None else scale)
        self.causal, self.window = causal, window
        mine = np.zeros(self.total, bool)
        for (a, b), s in zip(self.spans, self.k.slots):
            mine[a:b] = s != NO
        self.mine = mine
        self.q[~mine] = np.nan  # rows of nobody are not looked at

    def want(self, fresh=None):
        k, v = self.k.floats()
        n, w = self.total, self.k.width
        out = np.full((n, self.hq, w), SENTINEL, np.float64)
        q = self.q[:, :self.w].reshape(n, self.hq, w)
        gate = None if self.gate is None else self.gate[:, :self.w].reshape(n, self.hq, w)
        return paged64.attention(q, k, v, self.k.table, self.k.lengths, self.spans, self.k.slots,
                                 fresh, float(self.scale), self.causal, self.window, self.sinks,
                                 gate, out).reshape(n, self.w)

    def describe(self, c, fresh=None, slots=True):
        seqs = kq_hip.sequences(self.total, len(self.spans), self.k.slot_count, u32(c, self.off),
                                u32(c, self.k.slots) if slots else None, u32(c, fresh))
        at = kq_hip.paged_attention(self.hq, float(self.scale), self.causal, self.window,
                                    None if self.sinks is None else c.up(self.sinks),
                                    "none" if self.gate is None else "sigmoid")
        return at, self.k.describe(c), seqs

    def got(self, ctx, fresh=None, slots=True, pad=0):
        with Call(ctx) as c:
            at, k, seqs = self.describe(c, fresh, slots)
            out = np.full((self.total, self.w + pad), SENTINEL)
            y = c.up(out)
            n = kq_hip.paged_attention_scratch_bytes(at, k, seqs)
            ctx.paged_attention(at, k, seqs, c.up(self.q), self.q.shape[1],
                                None if self.gate is None else c.up(self.gate), self.w + 4, y,
                                self.w + pad, c.scratch(n), n)
            got = c.down(y, out)
            assert (got[:, self.w:] == SENTINEL).all()
            return got[:, :self.w]

    def check(self, got, fresh=None, rel=2e-6, big=3e-5):
        want = self.want(fresh)
        assert (got[~self.mine] == SENTINEL).all()
        if self.mine.any():
            near(got[self.mine], want[self.mine], rel, big)


SHAPES = [(1, 1, 64, 16), (2, 8, 128, 64), (2, 4, 256, 32), (3, 5, 64, 256), (1, 16, 128, 16),
          (1, 17, 128, 128), (2, 3, 128, 32), (4, 1, 256, 64)]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("past", [[0], [1], [15, 16, 62, 63, 64], [127, 0, 1000, 31]], ids=str)
def test_single_rows(ctx, type_, shape, past):  # noqa: F811
    say("single rows", type_, shape, past)
    heads, group, width, page = shape
    n = len(past)
    slots = np.random.default_rng(n).permutation(n + 2)[:n].tolist()
    a = Attention(n, type_, heads, group, width, page, past, [1] * n, slots, n + 2, offsets=False)
    a.check(a.got(ctx))
    a = Attention(n + 9, type_, heads, group, width, page, past, [1] * n, offsets=False, pad=4,
                  gate=True, sinks=True)
    fresh = [i % 2 for i in range(n)]
    a.check(a.got(ctx, fresh, slots=False, pad=8), fresh)


ROWS = [([2], [0]), ([16], [16]), ([17], [5]), ([64], [0]), ([65], [100]), ([33, 1, 0, 130, 7],
        [0, 77, 40, 3, 200]), ([0], [0]), ([1], [300]), ([200], [61])]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("rows,past", ROWS, ids=str)
def test_sequences(ctx, type_, shape, rows, past):  # noqa: F811
    say("sequences", type_, shape, rows, past)
    heads, group, width, page = shape
    n = len(rows)
    slots = np.random.default_rng(n).permutation(n + 1)[:n].tolist()
    if n > 4:
        slots[0] = NO
    a = Attention(sum(rows), type_, heads, group, width, page, past, rows, slots, n + 1,
                  lead=2 if n > 1 else 0, gap=1, pad=4)
    a.check(a.got(ctx, pad=4))


@pytest.mark.parametrize("rows,past", [([1], [200]), ([40], [300]), ([3, 150, 1], [64, 100, 700])],
                         ids=str)
@pytest.mark.parametrize("mode", [dict(window=1), dict(window=17), dict(window=64),
                                  dict(window=100000), dict(causal=False),
                                  dict(causal=False, window=70), dict(sinks=True),
                                  dict(gate=True), dict(scale=-0.2), dict(scale=0.0)], ids=str)
@pytest.mark.parametrize("type_", TYPES)
def test_forms(ctx, rows, past, mode, type_):  # noqa: F811
    say("forms", rows, past, mode, type_)
    for heads, group, width, page in ((2, 3, 64, 16), (1, 8, 128, 64)):
        a = Attention(len(rows), type_, heads, group, width, page, past, rows, **mode)
        a.check(a.got(ctx))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("rows,past", [([1], [20000]), ([2], [9001]), ([40], [12345]),
                                       ([1, 60, 1, 1], [7000, 3000, 20, 5000])], ids=str)
def test_long_pasts(ctx, type_, width, rows, past):  # noqa: F811
    # an item's keys in many parts, and their join
    say("long", type_, width, rows, past)
    a = Attention(3, type_, 2, 4, width, 64, past, rows, gate=len(rows) == 1)
    a.check(a.got(ctx))
    if rows == [1]:
        a = Attention(5, type_, 1, 2, width, 128, past, rows, offsets=False, sinks=True)
        a.check(a.got(ctx))


@pytest.mark.parametrize("n", [64, 65, 300])
def test_many_sequences(ctx, n):  # noqa: F811
    say("many sequences", n)
    r = np.random.default_rng(n)
    past = r.integers(0, 90, n).tolist()
    slots = r.permutation(n).tolist()
    a = Attention(n, "f16", 1, 3, 64, 16, past, [1] * n, slots, offsets=False)
    a.check(a.got(ctx))
    rows = [[1, 0, 2, 1, 1, 33][i % 6] for i in range(n)]
    past[7] = 2500
    slots[5] = slots[n - 1] = NO
    a = Attention(n + 1, "bf16", 2, 3, 64, 32, past, rows, slots, lead=1, gap=1)
    a.check(a.got(ctx))


def test_more_sequences_than_a_round_of_the_plan(ctx):  # noqa: F811
    say("1500 sequences")
    n = 1500
    rows = [[1, 0, 3][i % 3] for i in range(n)]
    past = [(i * 13) % 40 for i in range(n)]
    past[1400] = 4000
    a = Attention(8, "f16", 1, 2, 64, 16, past, rows)
    a.check(a.got(ctx))


# calls large enough for items of many rows, which share out rows in place of keys
LARGE = [([130, 65, 257], [900, 33, 0]), ([300], [1700]), ([700, 1, 90, 0, 1], [0, 800, 64, 3, 40]),
         ([129], [3000])]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("shape", [(8, 4, 64, 16), (8, 4, 128, 64), (7, 5, 128, 128),
                                   (4, 17, 64, 32), (6, 3, 256, 64)], ids=str)
@pytest.mark.parametrize("rows,past", LARGE, ids=str)
def test_many_rows(ctx, type_, shape, rows, past):  # noqa: F811
    say("many rows", type_, shape, rows, past)
    heads, group, width, page = shape
    n = len(rows)
    slots = np.random.default_rng(n).permutation(n + 1)[:n].tolist()
    a = Attention(sum(rows), type_, heads, group, width, page, past, rows, slots, n + 1, lead=1,
                  gap=2, pad=4)
    a.check(a.got(ctx, pad=4))


@pytest.mark.parametrize("mode", [dict(window=1), dict(window=100), dict(causal=False),
                                  dict(causal=False, window=70), dict(sinks=True, gate=True),
                                  dict(scale=-0.2)], ids=str)
@pytest.mark.parametrize("type_,width", [("f16", 64), ("bf16", 128), ("f16", 256)])
def test_many_rows_forms(ctx, mode, type_, width):  # noqa: F811
    say("many rows, forms", mode, type_, width)
    a = Attention(5, type_, 32, 2, width, 16, [400, 64, 1000], [200, 301, 128], **mode)
    a.check(a.got(ctx))


@pytest.mark.parametrize("where", ["query", "value"])
def test_many_rows_non_finite(ctx, where):  # noqa: F811
    say("many rows, non-finite", where)
    a = Attention(2, "f16", 8, 4, 128, 16, [1500], [300])
    if where == "query":
        a.q[211, 77] = np.nan
    else:
        a.k.values[a.k.table[0, 70], 3, 3, 9] = NAN
    assert attending(ctx, a) == "NUMERIC_DOMAIN"


def test_many_rows_nothing_outside_the_window(ctx):  # noqa: F811
    """Pages that a window has left behind do not exist any more."""
    say("many rows, pages gone")
    for width, rows in ((64, 400), (128, 300), (256, 260), (128, 1), (128, 9)):
        a = Attention(2, "bf16", 32, 2, width, 16, [3000], [rows], window=200)
        gone = (3000 + 1 - 200) // 16
        for p in a.k.table[0, :gone]:
            a.k.keys[p] = a.k.values[p] = NAN
        clean = a.k.table.copy()
        a.k.table[0, :gone] = 0xFFFFFFFF
        got = a.got(ctx)
        a.k.table = clean
        for p in a.k.table[0, :gone]:
            a.k.keys[p] = a.k.values[p] = 0
        # places of the first page that is left, before the window
        a.check(got)


def test_small_items_of_many_heads(ctx):  # noqa: F811
    """Items of few rows for a small call would be more than its workgroups."""
    say("many heads")
    for count, rows in ((7, 32), (70, 7)):
        a = Attention(5, "f16", 64, 4, 64, 16, [0] * count, [rows] * count)
        a.check(a.got(ctx))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("width,tiles", [(64, 12), (128, 6), (256, 3)])
@pytest.mark.parametrize("over", [0, 1])
def test_short_lines(ctx, type_, width, tiles, over):  # noqa: F811
    """Lines of the table at the size where a workgroup takes an item whole, and past
    it; sequences of every length that fits, with the window and the sink besides."""
    say("short lines", type_, width, tiles, over)
    keys = (tiles + over) * 64
    past = [0, 1, 31, 32, 63, 64, 127, keys - 65, keys - 33, keys - 3]
    a = Attention(12, type_, 2, 8, width, 32, past, [1] * 10, line=keys // 32, sinks=True)
    a.check(a.got(ctx))
    a = Attention(13, type_, 2, 4, width, 64, [keys - 3], [3], line=keys // 64, window=130)
    a.check(a.got(ctx))
    a = Attention(14, type_, 4, 2, width, 16, past[-4:], [2, 0, 1, 3], line=keys // 16,
                  causal=False, gate=True, lead=1, gap=1)
    a.check(a.got(ctx))


@pytest.mark.parametrize("type_,width", [("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("rows", [1, 60])
@pytest.mark.parametrize("line", [8, 12])
def test_lines_of_two_and_three_tiles(ctx, type_, width, rows, line):  # noqa: F811
    # no item has two parts in lines of two tiles; long lines behind a window of two
    say("two and three tiles", type_, width, rows, line)
    past = [line * 16 - rows, 3, 0, 65]
    a = Attention(15, type_, 2, 4, width, 16, past, [rows] * 4, line=line)
    a.check(a.got(ctx))
    a = Attention(16, type_, 80, 1, width, 16, past, [1] * 4, line=line)  # 320 items
    a.check(a.got(ctx))
    a = Attention(17, type_, 2, 4, width, 16, [5000, 20, 700], [1, 1, 1], window=60)
    a.check(a.got(ctx))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("width,tiles", [(64, 14), (128, 7), (256, 3)])
@pytest.mark.parametrize("over", [0, 1])
def test_short_lines_of_many_rows(ctx, type_, width, tiles, over):  # noqa: F811
    say("short lines, many rows", type_, width, tiles, over)
    keys = (tiles + over) * 64
    for seed, heads, rows in ((19, 1, [20, 1, 0, 65, 129]), (20, 24, [190, 60, 5, 128, 190])):
        past = [keys - rows[0], 3, 0, 64, keys - 190]
        a = Attention(seed, type_, heads, 3, width, 64, past, rows, line=keys // 64)
        a.check(a.got(ctx))
    a = Attention(21, type_, 2, 5, width, 32, [1000], [70], window=40, gate=True)
    a.check(a.got(ctx))
    a = Attention(22, type_, 2, 2, width, 32, [3] * 70, [7] * 70, line=keys // 32, causal=False)
    a.check(a.got(ctx))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("mode", [{}, dict(window=300), dict(causal=False, gate=True)], ids=str)
def test_middle_calls(ctx, type_, width, mode):  # noqa: F811
    """Calls that do not fill the device: items of 64 rows (heads of 256: of 128)."""
    say("middle", type_, width, mode)
    for seed, heads, group, past, rows in ((23, 4, 4, [2000], [301]), (24, 4, 3, [0], [917]),
                                           (25, 2, 5, [0, 900, 70, 3], [333, 1, 250, 407])):
        a = Attention(seed, type_, heads, group, width, 64, past, rows, line=64, **mode)
        a.check(a.got(ctx))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("width", [64, 128, 256])
def test_rows_of_two_waves(ctx, type_, width):  # noqa: F811
    """17 to 32 rows for a key head, beside sequences of one and of many rows."""
    say("two waves", type_, width)
    for seed, rows, past in ((28, [4, 3, 1, 4], [9000, 70, 5000, 8200]), (29, [4], [30000]),
                             (30, [3, 500, 4, 1], [4000, 3000, 64, 63])):
        a = Attention(seed, type_, 2, 8, width, 64, past, rows, line=512)
        a.check(a.got(ctx))


def test_middle_calls_of_many_sequences(ctx):  # noqa: F811
    say("middle, many sequences")
    a = Attention(26, "f16", 4, 4, 64, 32, [400 - 5 * i for i in range(70)], [30] * 70)
    a.check(a.got(ctx))


@pytest.mark.parametrize("type_,width", [("f16", 128), ("bf16", 64)])
def test_uneven_calls(ctx, type_, width):  # noqa: F811
    say("uneven", type_, width)
    a = Attention(27, type_, 4, 8, width, 128, [0], [1500])
    a.check(a.got(ctx))


def test_bad_slot_in_a_short_line(ctx):  # noqa: F811
    say("bad slot, short lines")
    a = Attention(18, "f16", 2, 4, 128, 32, [5, 90], [1, 1], line=4)
    a.k.slots = [0, 2]
    assert attending(ctx, a) == "INVALID_ARGUMENT"


def test_slots_may_be_shared(ctx):  # noqa: F811
    # several rows' worth of queries over one sequence's pages: read, not written
    say("shared")
    a = Attention(4, "f16", 2, 4, 128, 32, [100], [1], [0])
    a.k.slots = [0, 0, 0]
    a.off, a.spans, a.total = None, [(0, 1), (1, 2), (2, 3)], 3
    a.q = Gen(9).normal(3, a.w)
    a.mine = np.ones(3, bool)
    a.check(a.got(ctx))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("rows,past", [([1], [700]), ([50], [200])], ids=str)
@pytest.mark.parametrize("size", [30.0, 1e-20, 1e20])
def test_sizes_of_queries(ctx, type_, rows, past, size):  # noqa: F811
    """Rows of very different sizes: a query's own scale is kept. Scores of up to
    30 x 4 units leave one or a few keys; their errors grow with their size."""
    say("sizes", type_, rows, past, size)
    a = Attention(6, type_, 1, 4, 128, 64, past, rows)
    a.q[:, ::2] *= np.float32(1e-3)     # within a row
    a.q *= np.float32(size if size < 1e3 else 1.0)
    if size >= 1e3:                     # huge queries, tiny keys' factor
        a.q *= np.float32(size)
        a.scale = np.float32(1e-20 * 128 ** -0.5)
    grow = 16.0 if size == 30.0 else 1.0
    a.check(a.got(ctx), rel=2e-6 * grow, big=3e-5 * grow)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("rows,past", [([1], [200]), ([300], [900])], ids=str)
def test_tiny_queries_and_a_huge_scale(ctx, type_, rows, past):  # noqa: F811
    # near the ends of binary32 both; queries below 2^-114 keep their bits too
    say("tiny queries", type_, rows, past)
    a = Attention(8, type_, 8, 2, 64, 32, past, rows)
    a.q *= np.float32(1e-36)
    a.scale = np.float32(1e36 * 64 ** -0.5)
    a.check(a.got(ctx))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("rows,past", [([1], [200]), ([300], [900])], ids=str)
@pytest.mark.parametrize("scale", [0.0, 1e-30])
def test_scores_of_nothing(ctx, type_, rows, past, scale):  # noqa: F811
    """Scores far below binary32's range, and a scale of 0: all keys that a row sees
    weigh the same, and those that its mask leaves out nothing."""
    say("scores of nothing", type_, rows, past, scale)
    a = Attention(9, type_, 8, 2, 64, 32, past, rows, window=150)
    a.q *= np.float32(1e-30)
    a.scale = np.float32(scale)
    a.check(a.got(ctx))


@pytest.mark.parametrize("rows,past", [([1], [60]), ([1], [3000]), ([300], [900])], ids=str)
def test_sinks_of_any_size(ctx, rows, past):  # noqa: F811
    """-inf: no sink; a large one takes all the weight."""
    say("sinks", rows, past)
    a = Attention(8, "f16", 2, 4, 64, 32, past, rows, sinks=True)
    a.sinks[:] = [-np.inf, -80.0, 0.0, 3.0, 12.0, 30.0, -3e38, 5.0]
    a.check(a.got(ctx))
    a.sinks[:] = 3e38
    assert not a.got(ctx)[a.mine].any()


def test_growing_scores(ctx):  # noqa: F811
    """Keys whose scores grow along the sequence: each tile moves the maximum, by
    little (within the slack) and by much. Scores up to 100: errors 12 times."""
    say("growing scores")
    for step in (0.002, 0.05):
        for rows, past in (([1], [1800]), ([40], [1800])):
            a = Attention(7, "f16", 1, 4, 128, 64, past, rows)
            k, _ = a.k.floats()
            unit = np.ones(128) / np.sqrt(128)
            a.q[:] = np.tile((unit * 128 ** 0.5).astype(np.float32), 4)[None] + a.q * 0.1
            for i in range(past[0] + rows[0]):
                p = a.k.table[0, i // 64]
                a.k.keys[p, 0, i % 64] = paged64.to_bits((unit * i * step).astype(np.float32), False)
            a.check(a.got(ctx), rel=2.4e-5, big=4e-4)


def attending(ctx, a, off=None, slots=None, edit=None):  # noqa: F811
    with Call(ctx) as c:
        at, k, seqs = a.describe(c)
        if edit:
            edit(c, at, k, seqs)
        out = np.full((a.total, a.w), SENTINEL)
        y = c.up(out)
        n = kq_hip.paged_attention_scratch_bytes(at, k, seqs)
        with pytest.raises(kq_hip.KqError) as e:
            ctx.paged_attention(at, k, seqs, c.up(a.q), a.q.shape[1],
                                None if a.gate is None else c.up(a.gate), a.w + 4, y, a.w,
                                c.scratch(n), n)
        assert (c.down(y, out) == SENTINEL).all()
        return e.value.name


@pytest.mark.parametrize("what", ["slot", "page", "line", "length", "offsets", "offsets back"])
@pytest.mark.parametrize("many", [False, True])
def test_bad_indexes(ctx, what, many):  # noqa: F811
    say("bad", what, many)
    n = 80 if many else 3
    rows, past = [1, 20, 2] + [1] * (n - 3), [40, 50, 60] + [5] * (n - 3)
    a = Attention(1, "f16", 1, 4, 64, 16, past, rows)
    if what == "slot":
        a.k.slots[1] = n
    elif what == "page":
        a.k.table[1, 2] = a.k.pages + 5
    elif what == "line":
        a.k.lengths[2] = a.k.line * 16 - 1
    elif what == "length":
        a.k.lengths[2] = 0xFFFFFFFF
    elif what == "offsets":
        a.off[n] = a.total + 1
    else:
        a.off[1], a.off[2] = a.off[2], a.off[1]
    assert attending(ctx, a) == "INVALID_ARGUMENT"


def test_offsets_that_overlap(ctx):  # noqa: F811
    """Spans that go back again and again claim more rows than there are: refused,
    and no partial result leaves the scratch."""
    say("overlapping offsets")
    for n in (41, 201):
        a = Attention(1, "f16", 1, 4, 64, 16, [4000] * 2 + [0] * (n - 2), [60] + [0] * (n - 1))
        a.k.slots = [0] * n
        a.off[:] = [0, 60] * ((n + 1) // 2) + [0] * ((n + 1) % 2)
        assert attending(ctx, a) == "INVALID_ARGUMENT"


@pytest.mark.parametrize("where", ["query", "gate", "sink", "key", "value"])
@pytest.mark.parametrize("rows,past", [([1], [90]), ([30], [90]), ([1], [5000])], ids=str)
def test_non_finite(ctx, where, rows, past):  # noqa: F811
    say("non-finite", where, rows, past)
    a = Attention(2, "f16", 1, 4, 64, 16, past, rows, gate=True, sinks=True)
    if where == "query":
        a.q[-1, 77] = np.inf
    elif where == "gate":
        a.gate[-1, 3] = np.nan
    elif where == "sink":
        a.sinks[2] = np.nan
    else:
        (a.k.keys if where == "key" else a.k.values)[a.k.table[0, 1], 0, 3, 9] = NAN
    assert attending(ctx, a) == "NUMERIC_DOMAIN"


def test_non_finite_outside_the_window(ctx):  # noqa: F811
    """Keys and values that no row of the call sees are not looked at, also where
    they share a page and a tile with those that are seen."""
    say("outside the window")
    for rows, past in (([1], [150]), ([20], [150])):
        for type_ in TYPES:
            a = Attention(2, type_, 2, 4, 64, 64, past, rows, window=30)
            a.check(a.got(ctx))
            first = past[0] + 1 - 30
            for pos in range(first):
                p = a.k.table[0, pos // 64]
                a.k.keys[p, :, pos % 64] = a.k.values[p, :, pos % 64] = NAN
            k, v = a.k.keys.copy(), a.k.values.copy()
            clean = a.got(ctx)
            a.k.keys[a.k.keys == NAN] = a.k.values[a.k.values == NAN] = 0
            a.check(clean)
            a.k.keys, a.k.values = k, v


def test_offsets_past_4_gib(ctx):  # noqa: F811
    """Pages whose bytes lie 5 GiB into the pool."""
    say("far pages")
    a = Attention(3, "f16", 2, 4, 128, 64, [100, 30], [3, 20])
    page_bytes = 2 * 64 * 128 * 2
    shift = (5 << 30) // page_bytes
    with Call(ctx) as c:
        at, k, seqs = a.describe(c)
        big = [ctx.alloc((shift + a.k.pages) * page_bytes) for _ in range(2)]
        c.bufs += big
        d = kq_hip.Diagnostic()
        for b, host in zip(big, (a.k.keys, a.k.values)):
            kq_hip.check(kq_hip.lib().kq_hip_upload(C.c_void_p(ctx.handle),
                                                    C.c_void_p(b.ptr + shift * page_bytes),
                                                    host.ctypes.data, host.nbytes, C.byref(d)), d)
        far = a.k.table.copy()
        far[far != 0xFFFFFFFF] += shift
        k = kq_hip.paged_cache(a.k.type_id, 2, 128, 64, shift + a.k.pages, a.k.line, big[0].ptr,
                               big[1].ptr, c.up(far), c.up(a.k.lengths))
        out = np.full((a.total, a.w), SENTINEL)
        y = c.up(out)
        n = kq_hip.paged_attention_scratch_bytes(at, k, seqs)
        ctx.paged_attention(at, k, seqs, c.up(a.q), a.w, None, 0, y, a.w, c.scratch(n), n)
        a.check(c.down(y, out))
        # and rows written there
        qkv = Gen(4).normal(a.total, 2 * 256)
        p = c.up(qkv)
        ctx.cache_append(k, seqs, kq_hip.cache_rows(p, 512, p + 1024, 512))
        got = ctx.download(big[0].ptr + shift * page_bytes, np.uint16, a.k.keys.size)
        got = got.reshape(a.k.keys.shape)
        for t, s, pos in paged64.places(a.spans, a.k.slots, None, a.k.lengths):
            assert np.array_equal(got[a.k.table[s, pos // 64], :, pos % 64],
                                  paged64.to_bits(qkv[t, :256].reshape(2, 128), False))


# ---------------------------------------------------------------- together


class Layer:
    """Norms of the heads, rotation and append, attention with its gate: what an
    attention layer does between its projections, on buffers that stay."""

    def __init__(self, ctx, c, seqs_count, rows, pages_each, type_="f16", hk=2, group=4, width=64,
                 page=16):
        self.ctx, self.c = ctx, c
        self.hk, self.hq, self.width, self.page = hk, hk * group, width, page
        self.type_id, self.bf16 = TYPES[type_]
        self.n = seqs_count
        self.kv, self.qw = hk * width, hk * group * width
        self.stride = 2 * self.qw + 2 * self.kv  # query, gate, key, value
        pages = seqs_count * pages_each + 1
        order = np.random.default_rng(1).permutation(pages)[:seqs_count * pages_each]
        self.table = order.reshape(seqs_count, pages_each).astype(np.uint32)
        self.pools = [c.up(np.full((pages, hk, page, width), NAN, np.uint16)) for _ in range(2)]
        self.shape = (pages, hk, page, width)
        self.lengths = np.zeros(seqs_count, np.uint32)
        self.d_lengths = c.up(self.lengths)
        self.cache = kq_hip.paged_cache(self.type_id, hk, width, page, pages, pages_each,
                                        *self.pools, c.up(self.table), self.d_lengths)
        self.freq, _ = kq_hip.rotary_frequencies(width // 2, 1e4)
        self.rot = kq_hip.rotary(width // 2, c.up(self.freq))
        self.norm_w = 1 + 0.1 * Gen(3).normal(width)
        w = c.up(self.norm_w.astype(np.float32))
        self.norms = [kq_hip.gated_norm(h, width, 1e-6, w) for h in (self.hq, hk)]
        self.x = c.up(np.zeros((rows, self.stride), np.float32))
        self.y = c.up(np.zeros((rows, self.qw), np.float32))
        self.att = kq_hip.paged_attention(self.hq, width ** -0.5, gate="sigmoid")
        self.need, self.scratch = 0, None
        self.tokens = [np.zeros((0, self.stride)) for _ in range(seqs_count)]

    def plan(self, seqs):
        self.need = kq_hip.paged_attention_scratch_bytes(self.att, self.cache, seqs)
        self.scratch = self.c.scratch(self.need)

    def step(self, seqs):
        s, x, f = self.stride, self.x, 4
        gate, key = x + f * self.qw, x + 2 * f * self.qw
        n = seqs.token_count
        self.ctx.gated_norm(self.norms[0], n, x, s, None, 0, x, s)
        self.ctx.gated_norm(self.norms[1], n, key, s, None, 0, key, s)
        rows = kq_hip.cache_rows(key, s, key + f * self.kv, s, self.hq, x, s, x, s)
        self.ctx.cache_append(self.cache, seqs, rows, self.rot)
        self.ctx.paged_attention(self.att, self.cache, seqs, x, s, gate, s, self.y, self.qw,
                                 self.scratch, self.need)

    def exact(self, x, spans):
        """The call's outputs from all rows so far, the cache's rounding included."""
        out = []
        for i, (a, b) in enumerate(spans):
            self.tokens[i] = np.concatenate([self.tokens[i], x[a:b].astype(np.float64)])
            t = self.tokens[i]
            n = len(t)
            if a == b:
                continue
            rms = lambda v: v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-6) * self.norm_w  # noqa: E731
            q = rms(t[:, :self.qw].reshape(n, self.hq, -1))
            k = rms(t[:, 2 * self.qw:2 * self.qw + self.kv].reshape(n, self.hk, -1))
            v = t[:, -self.kv:].reshape(n, self.hk, -1)
            q, k = (paged64.turn(z, np.arange(n), self.freq)[0] for z in (q, k))
            k, v = (paged64.to_values(paged64.to_bits(z.astype(np.float32), self.bf16), self.bf16)
                    for z in (k, v))
            pool = [np.zeros((1, self.hk, n, self.width)) for _ in range(2)]
            pool[0][0], pool[1][0] = k.swapaxes(0, 1), v.swapaxes(0, 1)
            g = t[n - (b - a):, self.qw:2 * self.qw].reshape(b - a, self.hq, -1)
            y = paged64.attention(q[n - (b - a):], *pool, [[0]], [n - (b - a)], [(0, b - a)], [0],
                                  None, self.width ** -0.5, gate=g, out=np.zeros(g.shape))
            out.append(y.reshape(b - a, -1))
        return np.concatenate(out)


@pytest.mark.parametrize("type_", TYPES)
def test_layer_prompt_then_decoding(type_):
    """Prompts in one call, more rows in another, then decoding steps from a
    replayed graph whose lengths change. Keys whose binary64 value lies next to a
    border of the cache's type are rounded the other way now and then: their
    norm and rotation are 16 u off, so about 16 u / (eps / 2) of the keys' values
    (2^-9 fp16, 2^-12 bf16), each by a step eps. A score of 64 terms then moves by
    about eps sqrt(64) 8^-1 2^-4.5 (fp16; 2^-6 bf16), 4e-5 (1.2e-4), and an
    output's 2-norm by less than that: 1e-4 and 3e-4, an element 15 times."""
    say("layer", type_)
    rows = [37, 1, 70, 0, 16]
    bar = (1e-4, 1.5e-3) if type_ == "f16" else (3e-4, 4.5e-3)
    with kq_hip.Context(0) as ctx, Call(ctx) as c:  # noqa: F811
        n = len(rows)
        lay = Layer(ctx, c, n, 128, 12, type_)
        g = Gen(21)

        def fill(count):
            x = g.normal(count, lay.stride)
            put(ctx, lay.x, x)
            return x

        def compare(x, spans):
            want = lay.exact(x, spans)
            near(ctx.download(lay.y, np.float32, want.size).reshape(want.shape), want, *bar)
            lay.lengths += np.array([b - a for a, b in spans], np.uint32)
            put(ctx, lay.d_lengths, lay.lengths)

        for lengths in (rows, [3, 40, 1, 22, 0]):
            off, spans, total = table(lengths)
            seqs = kq_hip.sequences(total, n, n, c.up(off))
            lay.plan(seqs)
            x = fill(total)
            lay.step(seqs)
            compare(x, spans)
        one = [(i, i + 1) for i in range(n)]
        seqs = kq_hip.sequences(n, n, n)
        lay.plan(seqs)
        x = fill(n)
        lay.step(seqs)                 # eagerly once
        compare(x, one)
        ctx.set_async(True)
        h, graph = capture(ctx, lambda: lay.step(seqs))
        for i in range(20):
            x = fill(n)
            if i % 7 == 3:             # other work of the program between two replays
                lay.step(seqs)
                ctx.synchronize()
                compare(x, one)
                x = fill(n)
            assert h.hipGraphLaunch(graph, C.c_void_p(ctx.stream)) == 0
            ctx.synchronize()
            compare(x, one)
        ctx.set_async(False)
        h.hipGraphExecDestroy(graph)


def test_prompt_graph_lengths():
    """A graph of ragged calls replayed with other offsets, lengths and slots."""
    say("graph lengths")
    with kq_hip.Context(0) as ctx, Call(ctx) as c:  # noqa: F811
        a = Attention(3, "f16", 2, 4, 64, 16, [900, 30, 400, 0], [30, 4, 20, 10])
        at, k, seqs = a.describe(c)
        n = kq_hip.paged_attention_scratch_bytes(at, k, seqs)
        scr, y, q = c.scratch(n), c.up(np.zeros((a.total, a.w), np.float32)), c.up(a.q)
        run = lambda: ctx.paged_attention(at, k, seqs, q, a.w, None, 0, y, a.w, scr, n)  # noqa: E731
        run()
        ctx.set_async(True)
        h, graph = capture(ctx, run)
        for off, past, slots in (([0, 30, 34, 54, 64], [900, 30, 400, 0], [0, 1, 2, 3]),
                                 ([0, 1, 2, 3, 4], [929, 33, 0, 9], [0, 1, 2, 3]),
                                 ([0, 0, 0, 60, 64], [5, 6, 300, 6], [1, 3, 0, 2]),
                                 ([0, 10, 10, 20, 30], [100, 3, 12, 0], [NO, 1, 2, 0])):
            a.off = np.array(off, np.uint32)
            a.spans = list(zip(off[:-1], off[1:]))
            a.k.slots = slots
            for s, slot in enumerate(slots):
                if slot != NO:
                    a.k.lengths[slot] = past[s]
            a.q = Gen(off[1] + 5).normal(a.total, a.w)
            a.mine = np.zeros(a.total, bool)
            for (b, e), s in zip(a.spans, slots):
                a.mine[b:e] = s != NO
            put(ctx, seqs.offsets, a.off)
            put(ctx, seqs.slots, np.array(slots, np.uint32))
            put(ctx, k.lengths, a.k.lengths)
            put(ctx, q, a.q)
            for _ in range(2):
                put(ctx, y, np.full((a.total, a.w), SENTINEL))
                assert h.hipGraphLaunch(graph, C.c_void_p(ctx.stream)) == 0
                ctx.synchronize()
                got = ctx.download(y, np.float32, a.total * a.w).reshape(a.total, a.w)
                a.check(got)
        ctx.set_async(False)
        h.hipGraphExecDestroy(graph)


def test_two_contexts_at_once():
    """Calls of two contexts side by side, each with scratch of its own."""
    say("two contexts")
    with kq_hip.Context(0) as one, kq_hip.Context(0) as two:
        calls = []
        for i, cx in enumerate((one, two)):
            c = Call(cx)
            a = Attention(i, "f16", 2, 4, 128, 64, [9000 + i, 50], [1 + i, 40])
            at, k, seqs = a.describe(c)
            n = kq_hip.paged_attention_scratch_bytes(at, k, seqs)
            y = c.up(np.full((a.total, a.w), SENTINEL))
            calls.append((cx, c, a, at, k, seqs, c.up(a.q), y, c.scratch(n), n))
            cx.set_async(True)
        for _ in range(10):
            for cx, c, a, at, k, seqs, q, y, scr, n in calls:
                cx.paged_attention(at, k, seqs, q, a.w, None, 0, y, a.w, scr, n)
        for cx, c, a, at, k, seqs, q, y, scr, n in calls:
            cx.synchronize()
            a.check(cx.download(y, np.float32, a.total * a.w).reshape(a.total, a.w))
            cx.set_async(False)
            c.__exit__()


def test_same_bits_again(ctx):  # noqa: F811
    say("same bits")
    a = Attention(3, "f16", 2, 8, 128, 64, [5000, 40, 700], [1, 90, 3])
    first = a.got(ctx)
    for _ in range(3):
        assert np.array_equal(a.got(ctx), first, equal_nan=True)
