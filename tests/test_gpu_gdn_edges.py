"""The operators between a GDN layer's projections and its residual where
values or places are at an edge: what lies behind a sequence's rows, decays
that differ by orders of magnitude, long memories, small columns beside large
ones, the ends of the type's range. Against binary64 (tests/gdn64.py), with
the bars of tests/test_gpu_gdn.py where no other is derived here.
"""
import numpy as np
import pytest

import gdn64
import kq_hip
from test_gpu_gdn import (NO, Attention, Call, Conv, Gen, check, ctx, near, say,  # noqa: F401
                          table)

pytestmark = pytest.mark.gpu


# What follows a sequence in the arrays (rows of nobody, rows of a sequence taken
# out) is never looked at: not its values, not their size, not whether they are
# numbers.
@pytest.mark.parametrize("tail", [1, 31, 32, 33, 63])
@pytest.mark.parametrize("heads,delta", [((2, 4, 128, 128), True), ((1, 2, 64, 64), True),
                                         ((16, 48, 128, 128), True), ((1, 2, 64, 64), False),
                                         ((2, 4, 128, 128), False)], ids=str)
@pytest.mark.parametrize("behind", [np.nan, 1e30])
def test_attention_rows_behind_a_tail(ctx, tail, heads, delta, behind):  # noqa: F811
    say("behind a tail", tail, heads, delta, behind)
    for lengths, slots in (([64 + tail], [1]), ([tail], [0]), ([tail, 40, 128 + tail], [2, NO, 0])):
        off, spans, rows = table(lengths, lead=1, gap=70)
        n = len(lengths)
        a = Attention(tail, *heads, rows, 3, delta=delta)
        mine = np.zeros(rows, bool)
        for (b, e), s in zip(spans, slots):
            mine[b:e] = s != NO
        clean = a.got(ctx, off, slots, None, n)
        for x in (a.qkv, a.alpha, a.beta):
            if x is not None:
                x[~mine] = behind
        got = a.got(ctx, off, slots, None, n)
        assert np.array_equal(got[0], clean[0]) and np.array_equal(got[1], clean[1])
        check(a, got, spans, slots, [0] * n)


def near_parts(got, want):
    """Every head's rows, 64 at a time, by themselves."""
    for b in range(0, len(got), 64):
        for h in range(got.shape[1]):
            near(got[b:b + 64, h], want[b:b + 64, h])


# Rows that wipe a head's state out (a gate that resets it) between ordinary rows.
@pytest.mark.parametrize("alpha", [1e3, 1e10, 1e12, 1e15, 1e17, 1e30])
@pytest.mark.parametrize("heads", [(2, 4, 128, 64), (1, 2, 64, 64)], ids=str)
@pytest.mark.parametrize("delta", [True, False])
def test_attention_decays_behind_a_strong_one(ctx, alpha, heads, delta):  # noqa: F811
    say("behind a strong decay", alpha, heads, delta)
    off, spans, rows = table([200, 90, 12])
    a = Attention(61, *heads, rows, 3, delta=delta)
    for t in (3, 20, 21, 70, 100, 150, 203, 230, 295):
        a.alpha[t, :heads[1] - (t % 2)] = np.float32(alpha) * np.float32(1 + t / 64)
    got = a.got(ctx, off, None, None, 3)
    wy, ws = a.want(spans, [0, 1, 2], [0] * 3)
    near_parts(got[0], wy)
    for s in range(3):
        for h in range(heads[1]):
            near(got[1][s, h], ws[s, h])


def awkward_rates(n):
    r = np.linspace(-1e-4, -1e-5, 4000).astype(np.float32)
    e = np.exp(64.0 * r.astype(np.float64))
    off = (e.astype(np.float32) - e) / e
    return r[np.argsort(off)[[0, -1, 1, -2][:n]]]


@pytest.mark.parametrize("count", [1, 17])
@pytest.mark.parametrize("delta", [True, False])
def test_attention_long_memory(ctx, delta, count):  # noqa: F811
    say("long memory", delta, count)
    off, spans, rows = table([16384] + [1] * (count - 1))
    a = Attention(62, 1, 4, 64, 64, rows, count, delta=delta, alpha=False)
    a.qkv[:, 64:96] = 0
    a.rate[:] = awkward_rates(4)
    got = a.got(ctx, off, None, None, count)
    wy, ws = a.want(spans, list(range(count)), [0] * count)
    for h in range(4):
        near(got[1][0, h, :32], ws[0, h, :32])
        near(got[1][0, h, 32:], ws[0, h, 32:])
    near_parts(got[0], wy)


def awkward_size(n):
    m = np.linspace(2.4e38, 3.4e38, 20001).astype(np.float32)
    want = 1.0 / (m.astype(np.float64) * np.sqrt(n))
    off = np.abs(want.astype(np.float32).astype(np.float64) - want) / want
    return m[np.argmax(off)], off.max()


@pytest.mark.parametrize("rows", [1, 7, 40])
@pytest.mark.parametrize("dk", [64, 128])
def test_attention_largest_keys(ctx, rows, dk):  # noqa: F811
    m, off_ = awkward_size(dk)
    say("largest keys", rows, dk, m, off_)
    off, spans, _ = table([rows])
    a = Attention(63, 1, 2, dk, 64, rows, 1)
    a.qkv[:, :2 * dk] = np.sign(a.qkv[:, :2 * dk]) * m
    check(a, a.got(ctx, off, None, None, 1), spans, [0], [0])


@pytest.mark.parametrize("channels", [64, 67])
def test_conv_empty_sequence_non_finite(ctx, channels):  # noqa: F811
    say("conv, empty sequence", channels)
    v = Conv(64, channels, 4, 20, 2)
    v.state[1, 2, 33] = np.inf
    assert v.failing(ctx, [0, 20, 20], [0, 1], None, 2) == "NUMERIC_DOMAIN"


# The join in the place of the gated residual's write leaves the same bits.
@pytest.mark.parametrize("tokens", [1, 9, 600])
@pytest.mark.parametrize("hidden", [2560, 640, 36])
def test_join_is_gr_write(ctx, hidden, tokens):  # noqa: F811
    say("join as gr_write", hidden, tokens)
    g, b = Gen(65), 4
    block, res = g.normal(tokens, hidden), g.normal(tokens, b, hidden)
    gate = 2 * gdn64.sigmoid(g.normal(tokens, b)).astype(np.float32)
    with Call(ctx) as c:
        out, same, norm = (c.up(np.empty_like(res)) for _ in range(3))
        pb, pr, pg = c.up(block), c.up(res), c.up(gate)
        ctx.gr_write(kq_hip.gr_dims(b, hidden, 1), pr, pb, pg, tokens, same)
        want = c.down(same, res)
        assert np.array_equal(want, res + block[:, None] * gate[:, :, None])
        ctx.block_join(kq_hip.block_join(b, hidden, 1e-6), tokens, pb, None, pr, pg, out)
        assert np.array_equal(c.down(out, res), want)
        j = kq_hip.block_join(b, hidden, 1e-6, pre=c.up(g.normal(b, hidden)), pre_offset=1.0)
        ctx.block_join(j, tokens, pb, None, pr, pg, pr, norm)
        assert np.array_equal(c.down(pr, res), want)


def terms(a, b, rows, slot):
    """Of outputs q.S of a sequence from row b on, the 2-norms of the terms q_i S_i: what
    an output's error is a fraction of. Its own size is about that, but for cancellation,
    which leaves one output in ten at a tenth; a norm over few rows shows that."""
    hk, hv, dk, dv = a.dims
    q = a.parts()[0].astype(np.float64)
    q = q / np.sqrt((q * q).sum(-1, keepdims=True) + a.eps) * float(a.scale)
    out = []
    for t in rows:
        S = a.want([(b, t + 1)], [slot], [0])[1][slot]
        out.append(np.sqrt((q[t].repeat(hv // hk, 0)[:, :, None] ** 2 * S * S).sum(1)))
    return np.array(out)


# Columns of v have nothing to do with each other: each keeps its own bits, however
# small beside its neighbours (factors of 2^-spread .. 1), and from chunk to chunk
# as they grow and fall.
@pytest.mark.parametrize("spread", [8, 24, 60])
@pytest.mark.parametrize("lengths", [[17], [150], [70, 12, 130]], ids=str)
@pytest.mark.parametrize("heads,delta", [((2, 4, 128, 64), True), ((1, 2, 64, 64), True),
                                         ((2, 4, 128, 64), False), ((1, 9, 128, 128), False)],
                         ids=str)
def test_attention_columns(ctx, spread, lengths, heads, delta):  # noqa: F811
    say("columns", spread, lengths, heads, delta)
    off, spans, rows = table(lengths)
    n, (hk, hv, dk, dv) = len(lengths), heads
    g = Gen(67)
    a = Attention(66, *heads, rows, n, delta=delta)
    f = np.float32(2.0) ** -np.round(g.uniform(0, spread, hv, dv))
    # and each chunk's values by up to 2^6 either way, a column by itself
    wave = np.float32(2.0) ** np.round(g.uniform(-6, 6, rows // 64 + 1, hv, dv))
    a.qkv[:, 2 * hk * dk:a.width] *= (f * np.repeat(wave, 64, 0)[:rows]).reshape(rows, -1)
    a.state *= f[None, :, None, :]
    got = a.got(ctx, off, None, None, n)
    wy, ws = a.want(spans, list(range(n)), [0] * n)
    for s, (b, e) in enumerate(spans):
        for x in range(b, e, 64):  # 64 rows at a time, and the state
            x = slice(x, min(x + 64, e))
            size = np.linalg.norm(wy[x], axis=0)
            if x.stop - x.start < 16:
                t = terms(a, b, range(x.start, x.stop), s)
                size = np.maximum(size, np.linalg.norm(t, axis=0))
            err = np.linalg.norm(got[0][x] - wy[x], axis=0) / size
            assert err.max() <= 2e-6, (s, x, err.max())
        err = np.linalg.norm(got[1][s] - ws[s], axis=1) / np.linalg.norm(ws[s], axis=1)
        say("   worst column of the state", err.max())
        assert err.max() <= 2e-6, (s, err.max())


# Rows of one column share a scale in their chunk, under which a value's error is
# 2^-22 of it or 2^-31 of the column's largest: rows 2^k below those behind them.
@pytest.mark.parametrize("k", [10, 20, 30])
@pytest.mark.parametrize("heads,delta", [((2, 4, 128, 64), True), ((1, 2, 64, 64), True),
                                         ((2, 4, 128, 64), False), ((1, 9, 128, 128), False)],
                         ids=str)
def test_attention_rows_before_large_ones(ctx, k, heads, delta):  # noqa: F811
    say("before large rows", k, heads, delta)
    off, spans, rows = table([160])
    hk, hv, dk, dv = heads
    a = Attention(68, *heads, rows, 1, delta=delta)
    v = a.qkv[:, 2 * hk * dk:a.width]
    v[100:] *= np.float32(2.0 ** k)
    got = a.got(ctx, off, None, None, 1)
    wy, ws = a.want(spans, [0], [0])
    near(got[0][:64], wy[:64])
    near(got[0][100:], wy[100:])
    near(got[1], ws)
    # |d| is at most twice |v| and what the state gives; a row takes up to 64 of them
    # times |q.k| <= dk^-1/2
    floor = 64 * dk ** -0.5 * 2.0 ** -31 * 4 * np.abs(v).max()
    y = wy[64:100]
    bar = 3e-5 * np.maximum(np.abs(y), np.sqrt((y * y).mean())) + floor
    assert (np.abs(got[0][64:100] - y) <= bar).all()


# The heads, and 64 rows at a time, by themselves where they differ most in size.
@pytest.mark.parametrize("rows", [16, 17, 200])
@pytest.mark.parametrize("what", ["decays", "values", "keys", "no decay"])
@pytest.mark.parametrize("delta", [True, False])
def test_attention_parts_of_different_size(ctx, what, rows, delta):  # noqa: F811
    say("parts", what, rows, delta)
    off, spans, _ = table([rows])
    hk, hv, dk, dv = heads = (2, 4, 128, 64)
    a = Attention(69, *heads, rows, 1, delta=delta, normalize=what != "keys")
    qk = 2 * hk * dk
    if what == "decays":  # a head forgets at once, another hardly
        a.rate[:] = [-1e30, -200.0, -1.0, -1e-6]
    elif what == "values":  # heads 2^60 apart, their states with them
        f = np.float32(2.0) ** np.array([0, -20, 20, 40], np.float32)
        a.qkv[:, qk:a.width] *= np.repeat(f, dv)
        a.state *= f[None, :, None, None]
    elif what == "keys":  # rows of q, k and v of very different sizes, not normalized
        f = np.float32(10.0) ** Gen(70).uniform(-3, 0, rows, 1)
        a.qkv[:, :hk * dk] *= f
        a.qkv[:, hk * dk:qk] *= f[::-1]
        a.qkv[:, qk:a.width] *= f[::-1] ** -1
    else:
        a.rate[:] = 0.0
    got = a.got(ctx, off, None, None, 1)
    wy, ws = a.want(spans, [0], [0])
    near_parts(got[0], wy)
    for h in range(hv):
        near(got[1][0, h], ws[0, h])


# Rows and states of sequences taken out of a call of single rows are nobody's
def test_single_rows_taken_out(ctx):  # noqa: F811
    say("single rows taken out")
    slots = [2, NO, 0, NO, 4, 1]
    spans = [(i, i + 1) for i in range(6)]
    a = Attention(71, 2, 6, 128, 128, 6, 5)
    v = Conv(72, 260, 4, 6, 5, bias=True)
    for t in (1, 3):
        a.qkv[t], a.alpha[t], a.beta[t], v.x[t] = np.nan, np.inf, np.nan, np.nan
    a.state[3], v.state[3] = np.nan, np.nan
    check(a, a.got(ctx, None, slots, None, 6), spans, slots, [0] * 6)
    v.check(v.got(ctx, None, slots, None, 6), spans, slots, [0] * 6)


# States and values near the type's largest: what leaves the range is a sum with
# rows of q and k that are not yet divided by their norm, not the result.
@pytest.mark.parametrize("rows", [1, 12, 40])
@pytest.mark.parametrize("delta", [True, False])
def test_attention_largest_states(ctx, rows, delta):  # noqa: F811
    say("largest states", rows, delta)
    off, spans, _ = table([rows])
    a = Attention(73, 2, 4, 128, 64, rows, 1, delta=delta)
    a.qkv[:, :2 * 2 * 128] *= np.float32(30.0)
    a.qkv[:, 2 * 2 * 128:a.width] *= np.float32(1e36)
    a.state *= np.float32(3e37)
    check(a, a.got(ctx, None if rows == 1 else off, None, None, 1), spans, [0], [0])
