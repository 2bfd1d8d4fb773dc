"""The operators between a GDN layer's projections and its residual, on the
device, against their definitions in binary64 (tests/gdn64.py).

Bars, from the arithmetic (u = 2^-24, half a step of binary32):
- norms: an output is a product of at most 6 rounded factors, two of which
  carry the errors of a sum of squares (random signs: a few u; its root
  halves it) and of an exponential (2 u): |err| <= 16 u |y|, and where a
  residual is added 16 u (|residual| + |term|);
- convolution: taps products added in binary32, |err| <= (taps + 2) u S with S
  the sum of the terms' magnitudes; the SiLU has slope at most 1.1 and its own
  6 u: (taps + 10) u S;
- attention: an output is a sum over dk state values and 64 rows at a time,
  each product with operands within 2^-22 (three roundings of split
  operands); independent signs leave the 2-norm of the error within a few
  2^-22 of the 2-norm of the terms, which cancellation makes up to 4 times
  the output's: 2e-6 of the output's 2-norm for a whole array; a single
  element's error has the root-mean-square of the others' and stays within
  15 of it among a few million: 3e-5 of max(|y|, rms y).
"""
import ctypes as C

import numpy as np
import pytest

import gdn64
import kq_hip
import kq_oracle
import kq_synth as S

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SENTINEL = np.float32(-1234.5)
NO = gdn64.NO_SLOT


@pytest.fixture(scope="module")
def ctx():
    c = kq_hip.Context(0)
    yield c
    c.close()


def say(*a):
    print(*a, flush=True)


class Gen:
    """Seeded values."""

    def __init__(self, seed):
        self.r = np.random.default_rng(seed)

    def normal(self, *shape, scale=1.0):
        return (self.r.standard_normal(shape) * scale).astype(np.float32)

    def uniform(self, lo, hi, *shape):
        return self.r.uniform(lo, hi, shape).astype(np.float32)


def near(got, want, rel=2e-6, big=3e-5):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape and np.isfinite(got).all()
    norm = np.linalg.norm(want)
    err = np.abs(got - want)
    if norm == 0.0:
        assert not err.any()
        return
    rms = norm / np.sqrt(want.size)
    say("   rel", np.linalg.norm(err) / norm, "max", (err / np.maximum(np.abs(want), rms)).max())
    assert np.linalg.norm(err) <= rel * norm
    assert (err <= big * np.maximum(np.abs(want), rms)).all()


def table(lengths, lead=0, gap=0):
    """offsets and spans of sequences of these lengths, `lead` rows of nobody before."""
    off = np.cumsum([lead] + list(lengths)).astype(np.uint32)
    spans = list(zip(off[:-1].tolist(), off[1:].tolist()))
    return off, spans, int(off[-1]) + gap


class Call:
    """Uploads arrays, hands out addresses and frees everything at the end."""

    def __init__(self, ctx):
        self.ctx, self.bufs = ctx, []

    def up(self, a):
        if a is None:
            return None
        b = self.ctx.upload(a)
        self.bufs.append(b)
        return b.ptr

    def scratch(self, n):
        b = self.ctx.upload(np.full(max(n, 1), 0xFF, np.uint8))  # NaN for whoever reads it unset
        self.bufs.append(b)
        return b.ptr

    def down(self, p, a):
        return self.ctx.download(p, a.dtype, a.size).reshape(a.shape)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for b in self.bufs:
            b.close()


# ---------------------------------------------------------------- attention


class Attention:
    def __init__(self, seed, hk, hv, dk, dv, rows, pool, delta=True, alpha=True, bias=True,
                 normalize=True, eps=1e-6, pad=0):
        g = Gen(seed)
        self.dims = (hk, hv, dk, dv)
        self.rows, self.eps, self.normalize = rows, eps, normalize
        self.width = 2 * hk * dk + hv * dv
        # q, k and v side by side in a row, with `pad` more values behind them
        self.qkv = g.normal(rows, self.width + pad)
        if not normalize:
            self.qkv[:, :2 * hk * dk] /= np.float32(np.sqrt(dk))
        self.rate = -g.uniform(1.0, 16.0, hv) if alpha else -g.uniform(0.001, 0.2, hv)
        self.bias = g.uniform(-7.0, -2.0, hv) if alpha and bias else None
        self.alpha = g.normal(rows, hv + 3) if alpha else None
        self.beta = g.normal(rows, hv) if delta else None
        self.state = g.normal(pool, hv, dk, dv, scale=0.2)
        self.scale = np.float32(dk ** -0.5)

    def parts(self):
        hk, hv, dk, dv = self.dims
        n = self.rows
        return (self.qkv[:, :hk * dk].reshape(n, hk, dk),
                self.qkv[:, hk * dk:2 * hk * dk].reshape(n, hk, dk),
                self.qkv[:, 2 * hk * dk:self.width].reshape(n, hv, dv))

    def want(self, spans, slots, fresh):
        hk, hv, dk, dv = self.dims
        y = np.full((self.rows, hv, dv), SENTINEL)
        so = np.full(self.state.shape, SENTINEL)
        alpha = None if self.alpha is None else self.alpha[:, :hv]
        return gdn64.attention(*self.parts(), alpha, self.beta, self.rate, self.bias,
                               float(self.scale), self.eps if self.normalize else None,
                               self.state, spans, slots, fresh, y, so)

    def describe(self, c, off, slots, fresh, count):
        hk, hv, dk, dv = self.dims
        u32 = lambda a: None if a is None else c.up(np.asarray(a, np.uint32))  # noqa: E731
        seqs = kq_hip.sequences(self.rows, count, self.state.shape[0], u32(off), u32(slots),
                                u32(fresh))
        la = kq_hip.linear_attention(hk, hv, dk, dv, float(self.scale), c.up(self.rate),
                                     c.up(self.bias), self.normalize, self.eps)
        qkv, row = c.up(self.qkv), self.qkv.shape[1]
        inp = kq_hip.linear_attention_inputs(qkv, row, qkv + 4 * hk * dk, row, qkv + 8 * hk * dk,
                                             row, c.up(self.alpha), hv + 3, c.up(self.beta), hv)
        return la, seqs, inp

    def got(self, ctx, off, slots, fresh, count, in_place=False, pad=0):
        hk, hv, dk, dv = self.dims
        with Call(ctx) as c:
            la, seqs, inp = self.describe(c, off, slots, fresh, count)
            st = c.up(self.state)
            so = st if in_place else c.up(np.full(self.state.shape, SENTINEL))
            out = np.full((self.rows, hv * dv + pad), SENTINEL)
            y = c.up(out)
            n = kq_hip.linear_attention_scratch_bytes(la, seqs)
            ctx.linear_attention(la, seqs, inp, st, so, y, hv * dv + pad, c.scratch(n), n)
            got = c.down(y, out)
            assert (got[:, hv * dv:] == SENTINEL).all()
            return got[:, :hv * dv].reshape(self.rows, hv, dv), c.down(so, self.state)


def check(a, got, spans, slots, fresh, in_place=False):
    """Rows and states against binary64; what belongs to no sequence untouched."""
    y, so = got
    wy, ws = a.want(spans, slots, fresh)
    mine = np.zeros(a.rows, bool)
    held = np.zeros(a.state.shape[0], bool)
    for (b, e), s in zip(spans, slots):
        if s != NO:
            mine[b:e], held[s] = True, True
    assert (y[~mine] == SENTINEL).all()
    if in_place:
        assert np.array_equal(so[~held], a.state[~held])
    else:
        assert (so[~held] == SENTINEL).all()
    if mine.any():
        near(y[mine], wy[mine])
    if held.any():
        near(so[held], ws[held])


HEADS = [(1, 1, 64, 64), (2, 6, 128, 64), (3, 3, 64, 128), (16, 48, 128, 128), (1, 5, 128, 128)]


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("seqs", [1, 3, 70])
def test_attention_single_rows(ctx, heads, seqs):
    if heads[1] == 48 and seqs == 70:
        seqs = 9
    say("single rows", heads, seqs)
    pool = seqs + 4
    a = Attention(seqs, *heads, seqs, pool)
    slots = np.random.default_rng(seqs).permutation(pool)[:seqs].tolist()
    fresh = [i % 3 == 1 for i in range(seqs)]
    spans = [(i, i + 1) for i in range(seqs)]
    got = a.got(ctx, None, slots, fresh, seqs)
    check(a, got, spans, slots, fresh)
    # in place, and slots in order
    a = Attention(seqs + 100, *heads, seqs, pool)
    check(a, a.got(ctx, None, None, None, seqs, in_place=True), spans, list(range(seqs)),
          [0] * seqs, in_place=True)


MODES = [dict(), dict(delta=False), dict(alpha=False), dict(delta=False, alpha=False),
         dict(normalize=False), dict(normalize=False, delta=False), dict(bias=False)]
LENGTHS = [[1], [2], [15], [16], [17], [63], [64], [65], [127], [128], [129], [300], [0],
           [0, 5, 64, 0, 131, 1, 0], [200, 1, 1, 1, 77], [1] * 20 + [90], [33] * 7]


@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: "-".join(map(str, v[:6])))
@pytest.mark.parametrize("heads", HEADS[:3] + HEADS[4:], ids=str)
def test_attention_sequences(ctx, heads, lengths):
    say("sequences", heads, lengths)
    off, spans, rows = table(lengths, lead=3 if len(lengths) > 1 else 0, gap=2)
    n, pool = len(lengths), len(lengths) + 3
    a = Attention(sum(lengths) + n, *heads, rows, pool, pad=4 * (n % 3))
    slots = np.random.default_rng(n).permutation(pool)[:n].tolist()
    if n > 4:
        slots[3] = NO
    fresh = [i % 2 for i in range(n)]
    check(a, a.got(ctx, off, slots, fresh, n, pad=4), spans, slots, fresh)
    check(a, a.got(ctx, off, slots, None, n, in_place=True), spans, slots, [0] * n,
          in_place=True)


@pytest.mark.parametrize("mode", MODES, ids=lambda m: "-".join(m) or "all")
@pytest.mark.parametrize("lengths", [[1, 1, 1], [40], [150, 3, 260]], ids=str)
def test_attention_forms(ctx, mode, lengths):
    say("forms", mode, lengths)
    off, spans, rows = table(lengths)
    n = len(lengths)
    a = Attention(17, 2, 4, 128, 128, rows, n, **mode)
    check(a, a.got(ctx, off, None, None, n), spans, list(range(n)), [0] * n)
    if lengths == [1, 1, 1]:
        check(a, a.got(ctx, None, None, None, n), spans, list(range(n)), [0] * n)


def test_attention_long_prompt(ctx):
    # many chunks of one sequence, the layer's own heads
    say("long prompt")
    off, spans, rows = table([1999])
    a = Attention(5, 16, 48, 128, 128, rows, 1)
    check(a, a.got(ctx, off, None, [1], 1), spans, [0], [1])


# many heads: the operands of 15 chunks (960 rows) fill a round of the work, so
# that sequences go on from the state that an earlier round left
@pytest.mark.parametrize("lengths", [[1100], [960, 30], [40, 700, 0, 500, 16, 17, 300]], ids=str)
@pytest.mark.parametrize("delta", [True, False])
def test_attention_rounds(ctx, lengths, delta):
    say("rounds", lengths, delta)
    off, spans, rows = table(lengths, lead=1, gap=1)
    n = len(lengths)
    a = Attention(11, 2, 256, 64, 64, rows, n + 1, delta=delta)
    slots = [n - i for i in range(n)]
    fresh = [i % 2 == 0 for i in range(n)]
    if delta:
        check(a, a.got(ctx, off, slots, fresh, n, in_place=True), spans, slots, fresh,
              in_place=True)
    else:
        check(a, a.got(ctx, off, slots, fresh, n), spans, slots, fresh)


# without the delta correction and with few heads: chunks side by side
@pytest.mark.parametrize("heads", [(1, 1, 64, 64), (1, 2, 128, 64), (2, 4, 64, 128),
                                   (1, 3, 128, 128)], ids=str)
@pytest.mark.parametrize("lengths", [[17], [64], [900], [70, 0, 200]], ids=str)
def test_attention_chunks_at_once(ctx, heads, lengths):
    say("chunks at once", heads, lengths)
    off, spans, rows = table(lengths, lead=2, gap=1)
    n = len(lengths)
    a = Attention(n, *heads, rows, n + 1, delta=False, alpha=n != 1, pad=8)
    slots = [n - i for i in range(n)]
    fresh = [i % 2 for i in range(n)]
    check(a, a.got(ctx, off, slots, fresh, n, pad=4), spans, slots, fresh)
    check(a, a.got(ctx, off, slots, None, n, in_place=True), spans, slots, [0] * n, in_place=True)


def test_attention_chunks_at_once_rounds(ctx):
    # more chunks than a round of the work has (236), the state carried on
    say("chunks at once, rounds")
    off, spans, rows = table([15200, 33])
    a = Attention(3, 1, 16, 64, 64, rows, 2, delta=False)
    check(a, a.got(ctx, off, None, [1, 0], 2), spans, [0, 1], [1, 0])


@pytest.mark.parametrize("where", ["q", "v", "state"])
def test_attention_chunks_at_once_non_finite(ctx, where):
    say("chunks at once, non-finite", where)
    off, _, _ = table([200])
    a = Attention(9, 1, 2, 64, 64, 200, 1, delta=False)
    if where == "state":
        a.state[0, 1, 5, 7] = np.nan
    else:
        a.qkv[150, 3 if where == "q" else 130] = np.inf
    assert failing(ctx, a, off, None, None, 1) == "NUMERIC_DOMAIN"


def test_attention_many_sequences(ctx):
    # more than a workgroup looks at at a time, chunks among them here and there
    say("many sequences")
    lengths = [1, 0, 2, 1] * 160 + [70, 1, 17, 1] + [1] * 300 + [200, 18]
    off, spans, rows = table(lengths, lead=1, gap=2)
    n = len(lengths)
    a = Attention(31, 1, 2, 64, 64, rows, n)
    slots = np.random.default_rng(31).permutation(n).tolist()
    slots[100] = slots[641] = NO
    fresh = [i % 5 == 0 for i in range(n)]
    check(a, a.got(ctx, off, slots, fresh, n), spans, slots, fresh)


# a call's only sequence among rows of nobody
@pytest.mark.parametrize("lead,length,gap", [(0, 0, 40), (30, 0, 0), (3, 5, 30), (20, 200, 7)])
@pytest.mark.parametrize("heads", [(2, 6, 128, 128), (1, 2, 64, 64)], ids=str)
@pytest.mark.parametrize("delta", [True, False])
def test_attention_one_sequence(ctx, heads, lead, length, gap, delta):
    say("one sequence", heads, lead, length, gap, delta)
    off, spans, rows = table([length], lead=lead, gap=gap)
    a = Attention(41, *heads, rows, 3, delta=delta)
    for slot in (2, NO):
        for fresh in (0, 1):
            check(a, a.got(ctx, off, [slot], [fresh], 1), spans, [slot], [fresh])
        check(a, a.got(ctx, off, [slot], None, 1, in_place=True), spans, [slot], [0], in_place=True)


@pytest.mark.parametrize("off,slot", [([5, 2], 0), ([0, 51], 0), ([60, 70], 0), ([0, 50], 3),
                                      ([0xFFFFFFF0, 50], 0)], ids=str)
@pytest.mark.parametrize("delta", [True, False])
def test_attention_one_bad_sequence(ctx, off, slot, delta):
    say("one bad sequence", off, slot, delta)
    a = Attention(42, 1, 2, 64, 64, 50, 3, delta=delta)
    assert failing(ctx, a, off, [slot], None, 1) == "INVALID_ARGUMENT"


@pytest.mark.parametrize("delta", [True, False])
def test_attention_one_empty_sequence_non_finite(ctx, delta):
    say("one empty sequence, non-finite", delta)
    a = Attention(43, 1, 2, 64, 64, 50, 2, delta=delta)
    a.state[1, 1, 63, 63] = np.inf
    assert failing(ctx, a, [9, 9], [1], None, 1) == "NUMERIC_DOMAIN"


def test_attention_split_prompt_is_one(ctx):
    # a prompt in two calls, its state carried on, against the prompt in one
    say("split prompt")
    off, spans, rows = table([333])
    a = Attention(6, 2, 4, 128, 128, rows, 1)
    want = a.want(spans, [0], [1])
    whole = a.got(ctx, off, None, [1], 1)
    near(whole[0], want[0])
    for cut in (1, 64, 100, 332):
        one = Attention(6, 2, 4, 128, 128, rows, 1)
        y1, s1 = one.got(ctx, [0, cut], None, [1], 1)
        one.state = s1
        y2, s2 = one.got(ctx, [cut, 333], None, None, 1)
        near(np.concatenate([y1[:cut], y2[cut:]]), want[0])
        near(s2, want[1])


@pytest.mark.parametrize("rows", [1, 9, 80])
def test_attention_fresh_state_is_not_read(ctx, rows):
    say("fresh over NaN", rows)
    off, spans, _ = table([rows])
    a = Attention(7, 2, 4, 64, 128, rows, 2)
    a.state[:] = np.nan
    check(a, a.got(ctx, None if rows == 1 else off, [1], [1], 1), spans, [1], [1])


@pytest.mark.parametrize("rows", [1, 12, 150])
@pytest.mark.parametrize("what", ["strong decay", "no decay", "same key", "zero rows", "large",
                                  "tiny", "large values", "mixed"])
def test_attention_edges(ctx, what, rows):
    say("edges", what, rows)
    off, spans, _ = table([rows])
    hk, hv, dk, dv = 2, 4, 128, 64
    raw = what == "mixed"
    a = Attention(8, hk, hv, dk, dv, rows, 1, normalize=not raw)
    qk = 2 * hk * dk
    if what == "strong decay":
        a.rate[:] = [-1e4, -200.0, -1e30, -16.0]
        a.alpha[:] = np.abs(a.alpha) * 20
    elif what == "no decay":
        a.rate[:] = 0.0
        a.state *= 0
    elif what == "same key":  # the delta rule's hardest case: each row overwrites the last
        a.qkv[:, hk * dk:qk] = a.qkv[0, hk * dk:qk]
        a.beta[:] = 30.0
        a.rate[:] = -1e-3
    elif what == "zero rows":
        a.qkv[rows // 2:, :qk] = 0.0
    elif what == "large":  # squares beyond the type's range
        a.qkv[:, :qk] *= np.float32(1e25)
    elif what == "tiny":  # far below the epsilon: a key's weight is |k| / 1e-3
        a.qkv[:, :qk] *= np.float32(1e-9)
    elif what == "large values":
        a.qkv[:, qk:a.width] *= np.float32(1e30)
        a.state *= np.float32(1e30)
    else:  # rows of very different sizes, not normalized
        f = np.float32(10.0) ** Gen(9).uniform(-6, 0, rows, 1)
        a.qkv[:, :hk * dk] *= f
        a.qkv[:, hk * dk:qk] *= f[::-1]
        a.qkv[:, qk:a.width] *= f[::-1] ** -1
    check(a, a.got(ctx, off, None, None, 1), spans, [0], [0])


def failing(ctx, a, off, slots, fresh, count):
    """The status of a call that fails, and whether its outputs were left alone."""
    hk, hv, dk, dv = a.dims
    with Call(ctx) as c:
        la, seqs, inp = a.describe(c, off, slots, fresh, count)
        st, so = c.up(a.state), c.up(np.full(a.state.shape, SENTINEL))
        out = np.full((a.rows, hv * dv), SENTINEL)
        y = c.up(out)
        n = kq_hip.linear_attention_scratch_bytes(la, seqs)
        with pytest.raises(kq_hip.KqError) as e:
            ctx.linear_attention(la, seqs, inp, st, so, y, hv * dv, c.scratch(n), n)
        assert (c.down(y, out) == SENTINEL).all()
        assert (c.down(so, a.state) == SENTINEL).all()
        return e.value.name


@pytest.mark.parametrize("where", ["q", "k", "v", "alpha", "beta", "rate", "growth", "state"])
@pytest.mark.parametrize("rows", [1, 70])
def test_attention_non_finite(ctx, where, rows):
    say("non-finite", where, rows)
    off, _, _ = table([rows])
    a = Attention(10, 2, 4, 128, 128, rows, 1)
    t = rows - 1
    if where in "qkv":
        a.qkv[t, {"q": 3, "k": 2 * 128 + 5, "v": a.width - 1}[where]] = np.inf
    elif where == "alpha":
        a.alpha[t, 1] = -np.inf  # a decay of one, but not a number
    elif where == "beta":
        a.beta[t, 2] = np.inf
    elif where == "rate":
        a.rate[3] = np.nan
    elif where == "growth":
        a.rate[3] = 0.5
    else:
        a.state[0, 1, 2, 3] = np.nan
    assert failing(ctx, a, off, None, None, 1) == "NUMERIC_DOMAIN"


BAD_SEQUENCES = [([0, 5, 4, 9], None), ([0, 5, 9, 11], None), ([0, 5, 0xFFFFFFF0, 9], None),
                 ([12, 12, 12, 12], None), ([0, 3, 6, 9], [0, 5, 1]), ([0, 3, 6, 9], [0, 1, 0]),
                 ([0, 3, 3, 9], [2, 3, 2]), (None, [0, 1, 7]), (None, [1, 1, 0])]


@pytest.mark.parametrize("off,slots,scale", [(o, s, k) for o, s in BAD_SEQUENCES for k in (1, 70)
                                             if o is not None or k == 1], ids=str)
def test_bad_sequences(ctx, off, slots, scale):
    # offsets that decrease or pass the rows, slots that are not there or
    # named twice: refused on the device, by every operator, nothing written
    say("bad sequences", off, slots, scale)
    rows = 3 if off is None else 10 * scale
    off = None if off is None else [min(o * scale, 0xFFFFFFF0) for o in off]
    a = Attention(11, 1, 2, 64, 64, rows, 5)
    assert failing(ctx, a, off, slots, None, 3) == "INVALID_ARGUMENT"
    v = Conv(12, 64, 4, rows, 5)
    assert v.failing(ctx, off, slots, None, 3) == "INVALID_ARGUMENT"


# -------------------------------------------------------------- convolution


@pytest.mark.parametrize("first,second", [(0, 1), (63, 299), (64, 65), (150, 298), (255, 256),
                                          (200, 299)])
@pytest.mark.parametrize("rows", ["one each", "mixed"])
def test_slot_taken_among_many(ctx, first, second, rows):
    # one head: a workgroup has more threads than columns, and all of them look
    say("slot taken", first, second, rows)
    n = 300
    lengths = [1] * n if rows == "one each" else [i % 3 for i in range(n)]
    off, _, total = table(lengths)
    off = None if rows == "one each" else off
    slots = np.random.default_rng(1).permutation(n).tolist()
    slots[second] = slots[first]
    a = Attention(51, 1, 1, 64, 64, total, n)
    assert failing(ctx, a, off, slots, None, n) == "INVALID_ARGUMENT"
    assert Conv(52, 12, 4, total, n).failing(ctx, off, slots, None, n) == "INVALID_ARGUMENT"


class Conv:
    def __init__(self, seed, channels, taps, rows, pool, bias=False, silu=True, pad=0):
        g = Gen(seed)
        self.x = g.normal(rows, channels + pad)
        self.w = g.normal(channels, taps, scale=taps ** -0.5)
        self.bias = g.normal(channels) if bias else None
        self.state = g.normal(pool, taps - 1, channels)
        self.silu, self.channels, self.taps, self.rows = silu, channels, taps, rows

    def describe(self, c, off, slots, fresh, count):
        u32 = lambda a: None if a is None else c.up(np.asarray(a, np.uint32))  # noqa: E731
        return (kq_hip.causal_conv(self.channels, self.taps, c.up(self.w), c.up(self.bias),
                                   "silu" if self.silu else "none"),
                kq_hip.sequences(self.rows, count, self.state.shape[0], u32(off), u32(slots),
                                 u32(fresh)))

    def got(self, ctx, off, slots, fresh, count, in_place=False, pad=0):
        with Call(ctx) as c:
            cv, seqs = self.describe(c, off, slots, fresh, count)
            st = c.up(self.state)
            so = st if in_place else c.up(np.full(self.state.shape, SENTINEL))
            out = np.full((self.rows, self.channels + pad), SENTINEL)
            y = c.up(out)
            ctx.causal_conv(cv, seqs, c.up(self.x), self.x.shape[1], st, so, y, out.shape[1])
            got = c.down(y, out)
            assert (got[:, self.channels:] == SENTINEL).all()
            return got[:, :self.channels], c.down(so, self.state)

    def failing(self, ctx, off, slots, fresh, count):
        with Call(ctx) as c:
            cv, seqs = self.describe(c, off, slots, fresh, count)
            st, so = c.up(self.state), c.up(np.full(self.state.shape, SENTINEL))
            out = np.full((self.rows, self.channels), SENTINEL)
            y = c.up(out)
            with pytest.raises(kq_hip.KqError) as e:
                ctx.causal_conv(cv, seqs, c.up(self.x), self.x.shape[1], st, so, y, self.channels)
            assert (c.down(y, out) == SENTINEL).all()
            assert (c.down(so, self.state) == SENTINEL).all()
            return e.value.name

    def check(self, got, spans, slots, fresh, in_place=False):
        fill = self.state if in_place else np.full(self.state.shape, SENTINEL)
        x = self.x[:, :self.channels]
        args = (spans, slots, fresh, np.full((self.rows, self.channels), SENTINEL), fill)
        wy, ws = gdn64.conv(x, self.w, self.bias, self.silu, self.state, *args)
        big, _ = gdn64.conv(np.abs(x), np.abs(self.w),
                            None if self.bias is None else np.abs(self.bias), False,
                            np.abs(self.state), *args)
        assert (np.abs(got[0] - wy) <= (self.taps + 10) * U * np.abs(big)).all()
        assert np.array_equal(got[1], ws.astype(np.float32))  # inputs, moved


@pytest.mark.parametrize("taps", range(2, 9))
@pytest.mark.parametrize("channels", [1, 4, 63, 260, 1030])
def test_conv(ctx, channels, taps):
    say("conv", channels, taps)
    lengths = [0, 5, 1, 40, 0, 2, 17, 3, 100]
    off, spans, rows = table(lengths, lead=2, gap=3)
    n = len(lengths)
    for k, pad in enumerate((0, 4, 1)):
        v = Conv(taps + k, channels, taps, rows, n + 2, bias=k > 0, silu=k != 1, pad=pad)
        slots = np.random.default_rng(k).permutation(n + 2)[:n].tolist()
        slots[5] = NO
        fresh = [(i + k) % 2 for i in range(n)]
        v.check(v.got(ctx, off, slots, fresh, n, pad=pad), spans, slots, fresh)
        v.check(v.got(ctx, off, slots, fresh, n, in_place=True), spans, slots, fresh, True)
    # one row a sequence
    one = [(i, i + 1) for i in range(7)]
    v = Conv(taps, channels, taps, 7, 7, bias=True)
    v.check(v.got(ctx, None, None, None, 7), one, list(range(7)), [0] * 7)
    v.check(v.got(ctx, None, [6, 0, NO, 1, 2, 3, 4], [0, 1, 0, 0, 1, 0, 0], 7, in_place=True),
            one, [6, 0, NO, 1, 2, 3, 4], [0, 1, 0, 0, 1, 0, 0], True)


@pytest.mark.parametrize("taps", [2, 4, 8])
def test_conv_many_sequences(ctx, taps):
    # sequences shorter and longer than the taps, more of them than a wave
    # counts, next to ones that fill several walks of rows
    lengths = [(7 * i) % 12 for i in range(90)] + [1] * 70 + [100, 0, 33] + [0] * 5
    off, spans, rows = table(lengths, lead=2, gap=3)
    n = len(lengths)
    c = Conv(taps, 36, taps, rows, n + 2)
    slots = np.random.default_rng(taps).permutation(n + 2)[:n].tolist()
    slots[91] = slots[4] = NO
    fresh = [i % 3 == 0 for i in range(n)]
    c.check(c.got(ctx, off, slots, fresh, n), spans, slots, fresh)
    c.check(c.got(ctx, off, slots, fresh, n, in_place=True), spans, slots, fresh, True)


def test_conv_layer(ctx):
    # the layer's channels, prompts whose walks begin inside other sequences
    say("conv layer")
    off, spans, rows = table([129, 1, 700, 1, 31])
    v = Conv(3, 10240, 4, rows, 5)
    v.check(v.got(ctx, off, None, [1, 0, 1, 0, 0], 5), spans, list(range(5)), [1, 0, 1, 0, 0])


@pytest.mark.parametrize("rows", [1, 40])
def test_conv_fresh_and_non_finite(ctx, rows):
    say("conv fresh over NaN", rows)
    off, spans, _ = table([rows])
    v = Conv(4, 68, 4, rows, 1)
    state = v.state.copy()
    v.state[:] = np.nan
    v.check(v.got(ctx, off, None, [1], 1), spans, [0], [1])
    assert v.failing(ctx, off, None, None, 1) == "NUMERIC_DOMAIN"
    v.state = state
    v.x[-1, 5] = np.inf
    assert v.failing(ctx, off, None, None, 1) == "NUMERIC_DOMAIN"


# -------------------------------------------------------------------- norms

WIDTHS = [1, 3, 4, 17, 60, 64, 65, 96, 128, 131, 256, 260, 1000, 1024, 1025, 2560, 4096, 4100,
          4099, 16384, 16383]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("gate", ["none", "sigmoid", "silu"])
def test_gated_norm(ctx, width, gate):
    say("norm", width, gate)
    tokens, groups = (7, 5) if width < 2000 else (3, 2)
    g = Gen(width)
    w = groups * width
    for k, pad in enumerate((0, 4, 1)):
        x = g.normal(tokens, w + pad) * np.float32(10.0) ** g.uniform(-6, 6, tokens, 1)
        x[0, :width] = 0.0
        z = g.normal(tokens, w + pad, scale=4.0)
        weight = None if k == 0 and width > 64 else g.normal(groups if k == 1 else 1, width)
        off = 0.0 if k == 0 else 1.0
        want = gdn64.gated_norm(x[:, :w].reshape(tokens, groups, width),
                                weight, off, z[:, :w].reshape(tokens, groups, width), gate, 1e-6)
        with Call(ctx) as c:
            n = kq_hip.gated_norm(groups, width, 1e-6, c.up(weight), off, k == 1, gate)
            px, pz = c.up(x), c.up(z)
            out = np.full((tokens, w + pad), SENTINEL)
            y = c.up(out)
            ctx.gated_norm(n, tokens, px, w + pad, pz, w + pad, y, w + pad)
            got = c.down(y, out)
            assert (got[:, w:] == SENTINEL).all()
            # over the input, over the gate
            ctx.gated_norm(n, tokens, px, w + pad, pz, w + pad, pz, w + pad)
            if gate != "none":
                assert np.array_equal(c.down(pz, z)[:, :w], got[:, :w])
                pz = c.up(z)
            ctx.gated_norm(n, tokens, px, w + pad, pz, w + pad, px, w + pad)
            assert np.array_equal(c.down(px, x)[:, :w], got[:, :w])
        got = got[:, :w].reshape(tokens, groups, width)
        assert (np.abs(got - want) <= 16 * U * np.abs(want)).all()


@pytest.mark.parametrize("scale", [1e-38, 1e-25, 1e-16, 1e16, 1e19, 1e30, 1e38])
@pytest.mark.parametrize("width", [64, 131, 2560, 5000])
def test_gated_norm_range(ctx, width, scale):
    # squares beyond the type's range on either side
    say("norm range", width, scale)
    x = np.clip(Gen(1).normal(3, width), -3, 3) * np.float32(scale)
    eps = 1e-30 if scale < 1 else 1e-6
    want = gdn64.gated_norm(x, None, 0, None, "none", np.float64(np.float32(eps)))
    with Call(ctx) as c:
        out = np.empty_like(x)
        y = c.up(out)
        ctx.gated_norm(kq_hip.gated_norm(1, width, eps), 3, c.up(x), width, None, 0, y, width)
        got = c.down(y, out)
    assert (np.abs(got - want) <= 16 * U * np.abs(want)).all()


def test_norm_many_rows(ctx):
    # more rows than one launch has workgroups for
    say("norm many rows")
    x = Gen(2).normal(200000, 48 * 3)
    want = gdn64.gated_norm(x.reshape(200000, 48, 3), None, 0, None, "none", 1e-6)
    with Call(ctx) as c:
        out = np.empty_like(x)
        y = c.up(out)
        ctx.gated_norm(kq_hip.gated_norm(48, 3, 1e-6), 200000, c.up(x), 144, None, 0, y, 144)
        got = c.down(y, out).reshape(want.shape)
    assert (np.abs(got - want) <= 16 * U * np.abs(want)).all()


@pytest.mark.parametrize("hidden", [1, 5, 640, 1001, 1028, 2048, 2560, 4100, 5001, 16384])
@pytest.mark.parametrize("form", range(4))
def test_block_join(ctx, hidden, form):
    say("join", hidden, form)
    post, gate, pre, branch = [(True, "silu", True, True), (False, "none", False, False),
                               (True, "none", False, True), (False, "sigmoid", True, False)][form]
    for tokens, branches in ((1, 4), (5, 1), (3, 7), (520, 4)):
        if tokens * branches * hidden > 6_000_000:
            continue
        g = Gen(hidden + tokens)
        block, z = g.normal(tokens, hidden), g.normal(tokens, hidden, scale=3.0)
        res = g.normal(tokens, branches, hidden, scale=2.0)
        cg = 2 * gdn64.sigmoid(g.normal(tokens, branches)).astype(np.float32) if branch else None
        pw = g.normal(hidden, scale=0.1) if post else None
        nw = g.normal(branches, hidden, scale=0.1) if pre else None
        scale = np.float32(0.7)
        r, n = gdn64.block_join(block, pw, 1.0, z, gate, float(scale), res, cg, nw, 1.0, 1e-6)
        term = np.abs(r - res) + np.abs(res)
        for in_place in (False, True):
            with Call(ctx) as c:
                j = kq_hip.block_join(branches, hidden, 1e-6, c.up(pw), 1.0, gate, float(scale),
                                      c.up(nw), 1.0)
                pr = c.up(res)
                po = pr if in_place else c.up(np.empty_like(res))
                pn = c.up(np.empty_like(res)) if pre else None
                ctx.block_join(j, tokens, c.up(block), c.up(z) if gate != "none" else None, pr,
                               c.up(cg), po, pn)
                gr = c.down(po, res)
                gn = c.down(pn, res) if pre else None
            assert (np.abs(gr - r) <= 16 * U * term).all()
            if pre:
                # the norm's factor times the residual's own error
                inv = np.abs(n) / np.maximum(np.abs(r), 1e-30)
                assert (np.abs(gn - n) <= 16 * U * (np.abs(n) + inv * term)).all()


@pytest.mark.parametrize("where", ["block", "gate", "residual", "branch", "post", "pre"])
def test_join_non_finite(ctx, where):
    say("join non-finite", where)
    g = Gen(3)
    a = {"block": g.normal(4, 64), "gate": g.normal(4, 64), "residual": g.normal(4, 2, 64),
         "branch": g.normal(4, 2), "post": g.normal(64), "pre": g.normal(2, 64)}
    a[where].flat[-1] = np.inf
    with Call(ctx) as c:
        p = {k: c.up(v) for k, v in a.items()}
        ro, no = c.up(np.full((4, 2, 64), SENTINEL)), c.up(np.full((4, 2, 64), SENTINEL))
        j = kq_hip.block_join(2, 64, 1e-6, p["post"], 1.0, "silu", 1.0, p["pre"], 1.0)
        with pytest.raises(kq_hip.KqError) as e:
            ctx.block_join(j, 4, p["block"], p["gate"], p["residual"], p["branch"], ro, no)
        assert e.value.name == "NUMERIC_DOMAIN"
        assert (c.down(ro, a["residual"]) == SENTINEL).all()
        assert (c.down(no, a["residual"]) == SENTINEL).all()


# ------------------------------------------------------- the layer's run


class Layer:
    """A GDN layer behind the gated residual's read: Q8_0 projections of a
    hidden state, convolution, attention, head norm with its gate, the output
    projection and the join. `step` puts the state of every sequence on."""

    HK, HV, D, H, TAPS = 2, 6, 64, 256, 4

    def __init__(self, ctx, c, rows, seqs):
        self.ctx, g = ctx, Gen(20)
        self.rows, self.seqs = rows, seqs
        hk, hv, d, h = self.HK, self.HV, self.D, self.H
        self.ch, self.val = 2 * hk * d + hv * d, hv * d

        def mat(key, r, n):
            return S.quant_matrix("Q8_0", S.stream_key(S.W_MATVEC_Q8_0, S.R_WEIGHT, key), r, n)

        self.w = {"qkv": (mat(1, self.ch, h), self.ch, h), "gate": (mat(2, self.val, h), self.val, h),
                  "alpha": (mat(3, hv, h), hv, h), "beta": (mat(4, hv, h), hv, h),
                  "out": (mat(5, h, self.val), h, self.val)}
        self.p = {k: c.up(v[0]) for k, v in self.w.items()}
        self.dense = {k: kq_oracle.dequantize(kq_hip.TYPE_Q8_0, v[0].reshape(-1)).reshape(v[1], v[2])
                      .astype(np.float64) for k, v in self.w.items()}
        self.conv_w = g.normal(self.ch, self.TAPS, scale=0.5)
        self.rate, self.bias = -g.uniform(1, 8, hv), g.uniform(-5, -2, hv)
        self.norm_w, self.pre_w = 1 + g.normal(d, scale=0.1), g.normal(1, h, scale=0.1)
        self.state_c = np.zeros((seqs, self.TAPS - 1, self.ch), np.float32)
        self.state_a = np.zeros((seqs, hv, d, d), np.float32)
        self.buf = {k: c.up(np.zeros((rows, n), np.float32)) for k, n in
                    [("x", h), ("res", h), ("qkv", self.ch), ("conv", self.ch), ("gate", self.val),
                     ("alpha", hv), ("beta", hv), ("y", self.val), ("o", h), ("norm", h)]}
        self.sc, self.sa = c.up(self.state_c), c.up(self.state_a)
        self.fresh_none = None
        self.cv = kq_hip.causal_conv(self.ch, self.TAPS, c.up(self.conv_w))
        self.la = kq_hip.linear_attention(hk, hv, d, d, d ** -0.5, c.up(self.rate), c.up(self.bias))
        b = self.buf
        self.inp = kq_hip.linear_attention_inputs(b["conv"], self.ch, b["conv"] + 4 * hk * d,
                                                  self.ch, b["conv"] + 8 * hk * d, self.ch,
                                                  b["alpha"], hv, b["beta"], hv)
        self.gn = kq_hip.gated_norm(hv, d, 1e-6, c.up(self.norm_w), gate="silu")
        self.jn = kq_hip.block_join(1, h, 1e-6, pre=c.up(self.pre_w), pre_offset=1.0)
        self.scr = c.scratch(1 << 24)

    def project(self, name, x, y, rows):
        w, r, n = self.w[name]
        for at in range(0, rows, 8):
            self.ctx.matvec(kq_hip.TYPE_Q8_0, self.p[name], r, n, x + 4 * at * n,
                            min(8, rows - at), y + 4 * at * r)

    def step(self, seqs, rows):
        b, ctx = self.buf, self.ctx
        for k in ("qkv", "gate", "alpha", "beta"):
            self.project(k, b["x"], b[k], rows)
        ctx.causal_conv(self.cv, seqs, b["qkv"], self.ch, self.sc, self.sc, b["conv"], self.ch)
        ctx.linear_attention(self.la, seqs, self.inp, self.sa, self.sa, b["y"], self.val, self.scr,
                             kq_hip.linear_attention_scratch_bytes(self.la, seqs))
        ctx.gated_norm(self.gn, rows, b["y"], self.val, b["gate"], self.val, b["y"], self.val)
        self.project("out", b["y"], b["o"], rows)
        ctx.block_join(self.jn, rows, b["o"], None, b["res"], None, b["res"], b["norm"])

    def exact(self, x, res, spans):
        """The same in binary64 from the layer's own running state."""
        n, hk, hv, d = len(x), self.HK, self.HV, self.D
        p = {k: x.astype(np.float64) @ self.dense[k].T for k in ("qkv", "gate", "alpha", "beta")}
        slots, fresh = list(range(self.seqs)), [0] * self.seqs
        cv, self.state_c = gdn64.conv(p["qkv"], self.conv_w, None, True, self.state_c, spans, slots,
                                      fresh, np.zeros((n, self.ch)), self.state_c)
        q, k, v = np.split(cv, [hk * d, 2 * hk * d], axis=1)
        y, self.state_a = gdn64.attention(q.reshape(n, hk, d), k.reshape(n, hk, d),
                                          v.reshape(n, hv, d), p["alpha"], p["beta"], self.rate,
                                          self.bias, d ** -0.5, 1e-6, self.state_a, spans, slots,
                                          fresh, np.zeros((n, hv, d)), self.state_a)
        y = gdn64.gated_norm(y, self.norm_w, 0, p["gate"].reshape(n, hv, d), "silu", 1e-6)
        o = y.reshape(n, -1) @ self.dense["out"].T
        r, nx = gdn64.block_join(o, None, 0, None, "none", 1.0, res[:, None], None, self.pre_w, 1.0,
                                 1e-6)
        return r[:, 0], nx[:, 0]


def put(ctx, ptr, a):
    d = kq_hip.Diagnostic()
    a = np.ascontiguousarray(a)
    kq_hip.check(kq_hip.lib().kq_hip_upload(ctx._h, C.c_void_p(ptr), a.ctypes.data, a.nbytes,
                                            C.byref(d)), d)


class Far:
    """Rows 4 MiB apart: from the 1024th on past 32-bit offsets."""
    STRIDE = 1 << 20

    def __init__(self, ctx, c, a):
        self.ctx, self.a = ctx, a
        b = ctx.alloc(((a.shape[0] - 1) * self.STRIDE + a.shape[1]) * 4)
        c.bufs.append(b)
        self.ptr = b.ptr
        for t in range(a.shape[0]):
            put(ctx, self.ptr + 4 * t * self.STRIDE, a[t])

    def down(self):
        return np.stack([self.ctx.download(self.ptr + 4 * t * self.STRIDE, self.a.dtype,
                                           self.a.shape[1]) for t in range(self.a.shape[0])])


def far_slots(ctx, c, slots, held):
    """A pool in which the slots named lie far apart: its address, slot by slot upload."""
    size = held[0].nbytes
    b = ctx.alloc((max(slots) + 1) * size)
    c.bufs.append(b)
    for s, h in zip(slots, held):
        put(ctx, b.ptr + s * size, h)
    return b.ptr, size


@pytest.mark.parametrize("delta", [True, False])
def test_far_rows_and_slots(delta):
    # rows and states past 4 GiB of their arrays
    say("far", delta)
    lengths = [1000, 90, 10]
    off, spans, rows = table(lengths)
    with kq_hip.Context(0) as ctx, Call(ctx) as c:
        ctx.set_commit_on_success(False)
        hk, hv, dk, dv = dims = (2, 4, 64, 64) if delta else (1, 2, 64, 64)
        a = Attention(21, *dims, rows, 3, delta=delta)
        slots = [(9 << 29) // (hv * dk * dv), 7, (9 << 28) // (hv * dk * dv)]
        x, y = Far(ctx, c, a.qkv), Far(ctx, c, np.full((rows, hv * dv), SENTINEL))
        pool, size = far_slots(ctx, c, slots, a.state)
        la, _, _ = a.describe(c, off, None, None, 3)
        seqs = kq_hip.sequences(rows, 3, max(slots) + 1, c.up(off),
                                c.up(np.asarray(slots, np.uint32)),
                                c.up(np.asarray([0, 1, 0], np.uint32)))
        inp = kq_hip.linear_attention_inputs(
            x.ptr, Far.STRIDE, x.ptr + 4 * hk * dk, Far.STRIDE, x.ptr + 8 * hk * dk, Far.STRIDE,
            c.up(a.alpha), hv + 3, c.up(a.beta), hv)
        n = kq_hip.linear_attention_scratch_bytes(la, seqs)
        ctx.linear_attention(la, seqs, inp, pool, pool, y.ptr, Far.STRIDE, c.scratch(n), n)
        got = np.stack([ctx.download(pool + s * size, np.float32, a.state[0].size)
                        .reshape(a.state[0].shape) for s in slots])
        heads = y.down()
        check(a, (heads.reshape(rows, hv, dv), got), spans, [0, 1, 2], [0, 1, 0], in_place=True)
        # and the norm over them, in place
        w = Gen(22).normal(dv)
        ctx.gated_norm(kq_hip.gated_norm(hv, dv, 1e-6, c.up(w)), rows, y.ptr, Far.STRIDE, None, 0,
                       y.ptr, Far.STRIDE)
        h = heads.reshape(rows, hv, dv).astype(np.float64)
        want = h / np.sqrt((h * h).mean(2, keepdims=True) + 1e-6) * w
        assert (np.abs(y.down().reshape(rows, hv, dv) - want) <= 16 * U * np.abs(want)).all()


def test_far_conv():
    say("far conv")
    lengths = [1000, 2, 98]
    off, spans, rows = table(lengths)
    with kq_hip.Context(0) as ctx, Call(ctx) as c:
        ctx.set_commit_on_success(False)
        v = Conv(23, 256, 4, rows, 3)
        slots = [(9 << 29) // (3 * 256), 5, (9 << 28) // (3 * 256)]
        x, y = Far(ctx, c, v.x), Far(ctx, c, np.full((rows, 256), SENTINEL))
        pool, size = far_slots(ctx, c, slots, v.state)
        cv, _ = v.describe(c, off, None, None, 3)
        seqs = kq_hip.sequences(rows, 3, max(slots) + 1, c.up(off),
                                c.up(np.asarray(slots, np.uint32)), None)
        ctx.causal_conv(cv, seqs, x.ptr, Far.STRIDE, pool, pool, y.ptr, Far.STRIDE)
        got = np.stack([ctx.download(pool + s * size, np.float32, v.state[0].size)
                        .reshape(v.state[0].shape) for s in slots])
        v.check((y.down(), got), spans, [0, 1, 2], [0, 0, 0], in_place=True)


def hip_lib():
    h = C.CDLL("libamdhip64.so")
    h.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    h.hipStreamEndCapture.argtypes = [C.c_void_p, C.c_void_p]
    h.hipGraphInstantiate.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    h.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    h.hipGraphExecDestroy.argtypes = [C.c_void_p]
    h.hipGraphDestroy.argtypes = [C.c_void_p]
    return h


def capture(ctx, fn):
    """fn's calls on the context's stream as an executable graph."""
    h, g, ge = hip_lib(), C.c_void_p(), C.c_void_p()
    stream = C.c_void_p(ctx.stream)
    assert h.hipStreamBeginCapture(stream, 2) == 0
    fn()
    assert h.hipStreamEndCapture(stream, C.byref(g)) == 0
    assert h.hipGraphInstantiate(C.byref(ge), g, None, None, 0) == 0
    h.hipGraphDestroy(g)
    return h, ge


def test_layer_prompt_then_decoding():
    """A batch of prompts, then decoding steps from a replayed graph, each
    against binary64. The bars add up through the layer: projections of 256
    columns, the attention, a norm that scales by 1 / rms and another
    projection: 2e-5 of the residual's 2-norm."""
    say("layer")
    lengths = [130, 1, 65, 20]
    off, spans, rows = table(lengths)
    n = len(lengths)
    with kq_hip.Context(0) as ctx, Call(ctx) as c:
        lay = Layer(ctx, c, rows, n)
        g = Gen(21)
        b = lay.buf

        def fill(r):
            x, res = g.normal(r, lay.H), g.normal(r, lay.H)
            put(ctx, b["x"], x)
            put(ctx, b["res"], res)
            return x, res

        def compare(x, res, spans):
            r, nx = lay.exact(x, res, spans)
            near(ctx.download(b["res"], np.float32, r.size).reshape(r.shape), r, 2e-5, 4e-4)
            near(ctx.download(b["norm"], np.float32, r.size).reshape(r.shape), nx, 2e-5, 4e-4)

        x, res = fill(rows)
        lay.step(kq_hip.sequences(rows, n, n, c.up(off)), rows)
        compare(x, res, spans)
        one = [(i, i + 1) for i in range(n)]
        seqs = kq_hip.sequences(n, n, n)
        x, res = fill(n)
        lay.step(seqs, n)          # eagerly once
        compare(x, res, one)
        ctx.set_async(True)
        h, graph = capture(ctx, lambda: lay.step(seqs, n))
        for i in range(4):
            x, res = fill(n)
            if i == 2:             # other work of the program between two replays
                lay.step(seqs, n)
                ctx.synchronize()
                compare(x, res, one)
                x, res = fill(n)
            assert h.hipGraphLaunch(graph, C.c_void_p(ctx.stream)) == 0
            ctx.synchronize()
            compare(x, res, one)
        near(ctx.download(lay.sa, np.float32, lay.state_a.size).reshape(lay.state_a.shape),
             lay.state_a, 2e-5, 4e-4)
        ctx.set_async(False)
        h.hipGraphExecDestroy(graph)


def test_prompt_graph_replays():
    """The chunked form captured once and replayed with other inputs and other
    offsets in the same buffers."""
    say("prompt graph")
    with kq_hip.Context(0) as ctx, Call(ctx) as c:
        a = Attention(30, 2, 4, 128, 128, 400, 4)
        hk, hv, dk, dv = a.dims
        off = c.up(np.zeros(5, np.uint32))
        la, _, inp = a.describe(c, None, None, None, 1)
        seqs = kq_hip.sequences(400, 4, 4, off)
        st, so = c.up(a.state), c.up(np.zeros_like(a.state))
        y = c.up(np.zeros((400, hv * dv), np.float32))
        n = kq_hip.linear_attention_scratch_bytes(la, seqs)
        scr = c.scratch(n)
        ctx.set_async(True)
        h, graph = capture(ctx, lambda: ctx.linear_attention(la, seqs, inp, st, so, y, hv * dv, scr,
                                                             n))
        for lengths in ([400, 0, 0, 0], [1, 150, 200, 20], [0, 64, 128, 3], [100, 100, 100, 100]):
            o, spans, rows = table(lengths)
            b = Attention(sum(lengths[:2]), 2, 4, 128, 128, 400, 4)
            b.rate, b.bias = a.rate, a.bias
            put(ctx, off, o)
            put(ctx, inp.query, b.qkv)
            put(ctx, inp.alpha, b.alpha)
            put(ctx, inp.beta, b.beta)
            put(ctx, st, b.state)
            put(ctx, so, np.full_like(b.state, SENTINEL))
            put(ctx, y, np.full((400, hv * dv), SENTINEL))
            assert h.hipGraphLaunch(graph, C.c_void_p(ctx.stream)) == 0
            ctx.synchronize()
            got = (ctx.download(y, np.float32, 400 * hv * dv).reshape(400, hv, dv),
                   ctx.download(so, np.float32, b.state.size).reshape(b.state.shape))
            check(b, got, spans, list(range(4)), [0] * 4)
        ctx.set_async(False)
        h.hipGraphExecDestroy(graph)


@pytest.mark.parametrize("count,dims,delta", [(1, (2, 4, 128, 64), True), (1, (1, 2, 64, 128), False),
                                              (2, (1, 2, 64, 64), False)], ids=str)
def test_attention_graph_lengths(count, dims, delta):
    """Captured calls whose lengths change between replays, down to none."""
    say("graph lengths", count, dims, delta)
    with kq_hip.Context(0) as ctx, Call(ctx) as c:
        a = Attention(31, *dims, 300, 2, delta=delta)
        hk, hv, dk, dv = dims
        off = c.up(np.zeros(count + 1, np.uint32))
        la, _, inp = a.describe(c, None, None, None, 1)
        seqs = kq_hip.sequences(300, count, 2, off)
        st, so = c.up(a.state), c.up(np.zeros_like(a.state))
        out = np.full((300, hv * dv), SENTINEL)
        y = c.up(out)
        n = kq_hip.linear_attention_scratch_bytes(la, seqs)
        scr = c.scratch(n)
        ctx.set_async(True)
        h, graph = capture(ctx, lambda: ctx.linear_attention(la, seqs, inp, st, so, y, hv * dv, scr,
                                                             n))
        for lengths in ([300, 0], [0, 150], [5, 100], [129, 171], [0, 0], [64, 16]):
            o, spans, _ = table(lengths[:count], lead=0)
            put(ctx, off, o)
            put(ctx, so, np.full_like(a.state, SENTINEL))
            put(ctx, y, out)
            assert h.hipGraphLaunch(graph, C.c_void_p(ctx.stream)) == 0
            ctx.synchronize()
            check(a, (c.down(y, out).reshape(300, hv, dv), c.down(so, a.state)), spans,
                  list(range(count)), [0] * count)
        ctx.set_async(False)
        h.hipGraphExecDestroy(graph)


def test_conv_graph_lengths():
    say("conv graph lengths")
    with kq_hip.Context(0) as ctx, Call(ctx) as c:
        v = Conv(32, 260, 4, 90, 3)
        off = c.up(np.zeros(4, np.uint32))
        cv, _ = v.describe(c, None, None, None, 1)
        seqs = kq_hip.sequences(90, 3, 3, off)
        x, st, so = c.up(v.x), c.up(v.state), c.up(np.zeros_like(v.state))
        out = np.full((90, 260), SENTINEL)
        y = c.up(out)
        ctx.set_async(True)
        h, graph = capture(ctx, lambda: ctx.causal_conv(cv, seqs, x, 260, st, so, y, 260))
        for lengths in ([90, 0, 0], [1, 2, 3], [0, 0, 0], [30, 17, 43], [0, 16, 74]):
            o, spans, _ = table(lengths)
            put(ctx, off, o)
            put(ctx, so, np.full_like(v.state, SENTINEL))
            put(ctx, y, out)
            assert h.hipGraphLaunch(graph, C.c_void_p(ctx.stream)) == 0
            ctx.synchronize()
            v.check((c.down(y, out), c.down(so, v.state)), spans, [0, 1, 2], [0, 0, 0])
        ctx.set_async(False)
        h.hipGraphExecDestroy(graph)


def test_same_inputs_same_bits(ctx):
    # no sum depends on the order in which workgroups run
    say("same bits")
    off, spans, rows = table([150, 700, 1, 64])
    a = Attention(40, 2, 4, 128, 128, rows, 4)
    one = a.got(ctx, off, None, None, 4)
    for _ in range(3):
        two = a.got(ctx, off, None, None, 4)
        assert np.array_equal(one[0], two[0]) and np.array_equal(one[1], two[1])


def test_two_contexts_at_once():
    # two streams of their own, enqueued without waiting between
    say("two contexts")
    off, spans, rows = table([200, 3])
    with kq_hip.Context(0) as x, kq_hip.Context(0) as y:
        runs = []
        for k, ctx in enumerate((x, y)):
            c = Call(ctx)
            a = Attention(50 + k, 2, 4, 128, 128, rows, 2)
            la, seqs, inp = a.describe(c, off, None, None, 2)
            n = kq_hip.linear_attention_scratch_bytes(la, seqs)
            out = np.full((rows, 4 * 128), SENTINEL)
            runs.append((ctx, c, a, la, seqs, inp, c.up(a.state), c.up(np.full_like(a.state, SENTINEL)),
                         c.up(out), c.scratch(n), n, out))
        for ctx, *_ in runs:
            ctx.set_async(True)
        for _ in range(3):
            for ctx, c, a, la, seqs, inp, st, so, py, scr, n, out in runs:
                ctx.linear_attention(la, seqs, inp, st, so, py, 512, scr, n)
        for ctx, c, a, la, seqs, inp, st, so, py, scr, n, out in runs:
            ctx.synchronize()
            check(a, (c.down(py, out).reshape(rows, 4, 128), c.down(so, a.state)), spans, [0, 1],
                  [0, 0])
            c.__exit__()
