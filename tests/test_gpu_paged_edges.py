"""Rotary positions and attention over a paged cache where their arithmetic and
their launches end, on the device, against the definitions in binary64
(tests/paged64.py)."""
import numpy as np
import pytest

import kq_hip
import paged64
from test_gpu_gdn import Call, Gen, ctx, near, say  # noqa: F401
from test_gpu_paged import SENTINEL, TYPES, Attention, Cache, u32

pytestmark = pytest.mark.gpu


# ------------------------------------------- weights far below a row's largest

# where a workgroup takes an item, where items have parts, and items of 64 and 128 rows
FORMS = [(1, [1], [200]), (1, [1], [3000]), (4, [3, 1, 40], [90, 700, 300]), (8, [300], [900]),
         (8, [700, 1, 300], [0, 64, 1500])]


def leading_key(ctx, type_, width, heads, rows, past, ahead, at, value):  # noqa: F811
    """One key leads the others by `ahead` (nats) and its value is next to nothing, so
    that the others' small weights are what counts. Every weight of a row stands beside
    one number of its own, the leading key's score of up to `ahead`, whose query is held
    to 2^-23, rounded with its factor (2^-24) and summed of two terms (2^-24 each): at
    most 1.25 2^-22 of `ahead`, 1.5 2^-22 allowed beside the 2e-6 of scores of the order
    of 1 (15 times that for an element)."""
    a = Attention(ahead, type_, heads, 4, width, 64, past, rows)
    q = a.q.reshape(a.total, a.hq, width)
    q *= np.float32(0.5)
    g = np.random.default_rng(ahead)
    q[:, :, 0] = g.uniform(3.5, 4.0, (a.total, a.hq))
    lead = np.zeros(width, np.float32)
    lead[0] = ahead * width ** 0.5 / 4.0
    for s in a.k.slots:
        ids = a.k.table[s][a.k.table[s] < a.k.pages]
        a.k.keys[ids, :, :, 0] = 0
        a.k.keys[ids[0], :, at] = paged64.to_bits(lead, a.k.bf16)
        a.k.values[ids[0], :, at] = paged64.to_bits(
            g.normal(size=(heads, width)).astype(np.float32) * np.float32(value), a.k.bf16)
    bar = 2e-6 + ahead * 1.5 * 2.0 ** -22
    got = a.got(ctx).astype(np.float64).reshape(a.total, a.hq, width)
    want = a.want().reshape(a.total, a.hq, width)
    size = np.linalg.norm(want, axis=2, keepdims=True)
    assert not got[size[..., 0] == 0].any()  # rows that see the leading key alone
    size[size == 0] = 1.0
    near(got / size, want / size, bar, 15 * bar)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("heads,rows,past", FORMS, ids=str)
@pytest.mark.parametrize("ahead", [6, 12, 18, 24, 36])
@pytest.mark.parametrize("at", [0, 60])
def test_a_leading_key_without_a_value(ctx, type_, width, heads, rows, past, ahead, at):  # noqa: F811
    say("leading key", type_, width, heads, rows, past, ahead, at)
    leading_key(ctx, type_, width, heads, rows, past, ahead, at, 0.0)


@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("heads,rows,past", FORMS[2:], ids=str)
@pytest.mark.parametrize("ahead", [12, 16])
@pytest.mark.parametrize("value", [1e-1, 1e-2, 1e-3, 1e-5])
def test_a_leading_key_of_a_small_value(ctx, width, heads, rows, past, ahead, value):  # noqa: F811
    # on both sides of where the small weights' last bits are looked at
    say("leading key", width, heads, rows, past, ahead, value)
    leading_key(ctx, "f16", width, heads, rows, past, ahead, 0, value)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("heads,rows,past", FORMS[:4], ids=str)
@pytest.mark.parametrize("ahead", [60, 76, 80, 84, 86])
def test_sinks_far_above_the_scores(ctx, type_, width, heads, rows, past, ahead):  # noqa: F811
    """A sink's weight against weights that are held times up to 2^15: outputs are normal
    numbers still. What a row is multiplied by is held to 2^-150 where it is not, that is
    2^-135 e^ahead of itself, as the largest scores are above 0; the sink's own exponent
    has a relative error of 2^-24 beside the 2e-6 of the scores, and the outputs a last
    half step, 2^-150."""
    say("sinks ahead", type_, width, heads, rows, past, ahead)
    a = Attention(ahead, type_, heads, 4, width, 64, [max(p, 60) for p in past], rows, sinks=True)
    a.sinks[:] = ahead
    bar = 2e-6 + ahead * 2.0 ** -23 + 2.0 ** -135 * np.exp(ahead)
    got, want = a.got(ctx).astype(np.float64), a.want()
    assert np.linalg.norm(got - want) <= bar * np.linalg.norm(want) + 2.0 ** -150 * want.size ** 0.5


# ------------------------------------------------------------- the largest calls


def test_more_workgroups_than_a_launch(ctx):  # noqa: F811
    """As many sequences as a call may have, of as many key heads: 16.8 million items of
    a workgroup each, more than 2^32 threads. The rows repeat, and so do their results."""
    say("65535 sequences of 256 heads")
    n, heads, width, again = 65535, 256, 64, 60
    past = [0, 3, 64, 130, 255]
    k = Cache(4, "f16", heads, width, 64, past, [1] * 5, line=4)
    slots = np.arange(n) % 5
    few = Gen(9).normal(again, heads * width)
    with Call(ctx) as c:
        seqs = kq_hip.sequences(n, n, 5, None, u32(c, slots))
        at = kq_hip.paged_attention(heads, width ** -0.5)
        cache = k.describe(c)
        q = c.up(few[np.arange(n) % again])
        out = np.full((n, heads * width), SENTINEL)
        y = c.up(out)
        size = kq_hip.paged_attention_scratch_bytes(at, cache, seqs)
        say("launching")
        ctx.paged_attention(at, cache, seqs, q, heads * width, None, 0, y, heads * width,
                            c.scratch(size), size)
        say("done")
        got = c.down(y, out)
    fk, fv = k.floats()
    want = paged64.attention(few.reshape(again, heads, width), fk, fv, k.table, k.lengths,
                             [(i, i + 1) for i in range(again)], slots[:again], None, width ** -0.5,
                             out=np.zeros((again, heads, width)))
    near(got[:again], want.reshape(again, -1))
    for i in range(again, n, again):
        assert np.array_equal(got[i:i + again], got[:min(again, n - i)])


# ------------------------------------------------------------------- the rotation


@pytest.mark.parametrize("rows,first", [(700, 1 << 23), (4096, 0), (4096, (1 << 24) - 4096)])
def test_angles(ctx, rows, first):  # noqa: F811
    """Sines and cosines of angles up to 2^24, seen by a vector of length 1: rounded once,
    2^-25 below 1, of an angle held to 2^-27 and by series 2^-27 off."""
    say("angles", rows, first)
    half = 512
    freq = np.exp(-np.sort(Gen(rows).uniform(0.0, 7.0, half).astype(np.float64)))
    at = first + np.arange(rows, dtype=np.uint32)
    x = np.zeros((rows, 2 * half), np.float32)
    x[:, :half] = 1.0
    with Call(ctx) as c:
        y = c.up(np.zeros_like(x))
        ctx.rotary(kq_hip.rotary(2 * half, c.up(freq)), 1, 2 * half, rows, u32(c, at), c.up(x),
                   2 * half, y, 2 * half)
        got = c.down(y, x)
    angle = at.astype(np.longdouble)[:, None] * freq.astype(np.longdouble)
    off = np.abs(got - np.concatenate([np.cos(angle), np.sin(angle)], 1)).max()
    say("   off", float(off) * 2.0 ** 25, "times 2^-25")
    assert off <= 2.0 ** -25 + 2.0 ** -27 + 2.0 ** -27
