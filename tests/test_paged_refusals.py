"""What rotary positions, the paged cache and the attention over it refuse
before any device work, and the frequencies that the host makes. CPU only: a
context that was never opened stands in for one, and a call that passes every
check ends at it."""
import ctypes as C
import math

import numpy as np
import pytest

import kq_hip
import paged64
from test_gdn_refusals import at, call, passes, seqs


def rotary(r=None, heads=4, width=64, tokens=5, positions=at(1), x=at(0), xs=256, y=at(2), ys=256):
    r = r or kq_hip.rotary(64, at(3))
    return call("kq_hip_rotary_f32", C.byref(r), heads, width, tokens, positions, x, xs, y, ys)


def test_rotary():
    R = kq_hip.rotary
    assert passes(rotary())
    assert passes(rotary(positions=None)) and passes(rotary(y=at(0)))
    assert passes(rotary(R(2, at(3), "pairs", 1.2)))
    assert passes(rotary(xs=512, y=at(0, 1024), ys=512))   # beside the input, in its rows
    for kw, want in [(dict(tokens=0), "INVALID_ARGUMENT"), (dict(heads=0), "INVALID_ARGUMENT"),
                     (dict(width=0), "INVALID_ARGUMENT"), (dict(x=None), "INVALID_ARGUMENT"),
                     (dict(y=None), "INVALID_ARGUMENT"),
                     (dict(r=R(64, None)), "INVALID_ARGUMENT"),
                     (dict(r=R(64, at(3), magnitude=math.inf)), "INVALID_ARGUMENT"),
                     (dict(r=kq_hip.Rotary(64, 2, 1.0, at(3))), "INVALID_ARGUMENT"),
                     (dict(r=R(0, at(3))), "LIMIT_EXCEEDED"), (dict(r=R(63, at(3))), "LIMIT_EXCEEDED"),
                     (dict(r=R(1026, at(3)), width=1024, heads=1, xs=1024, ys=1024),
                      "LIMIT_EXCEEDED"),
                     (dict(r=R(66, at(3))), "DIMENSION_MISMATCH"),
                     (dict(width=1025, heads=1, xs=1025, ys=1025), "LIMIT_EXCEEDED"),
                     (dict(heads=4097, width=1024), "LIMIT_EXCEEDED"),
                     (dict(tokens=262145), "LIMIT_EXCEEDED"),
                     (dict(xs=255), "DIMENSION_MISMATCH"), (dict(ys=255), "DIMENSION_MISMATCH"),
                     (dict(xs=(1 << 22) + 1), "DIMENSION_MISMATCH"),
                     (dict(x=at(0, 2)), "INVALID_ALIGNMENT"),
                     (dict(positions=at(1, 1)), "INVALID_ALIGNMENT"),
                     (dict(r=R(64, at(3, 4))), "INVALID_ALIGNMENT"),
                     (dict(y=at(0, 4)), "ALIASING_VIOLATION"),
                     (dict(y=at(0), ys=260), "ALIASING_VIOLATION"),
                     (dict(xs=512, y=at(0, 1020), ys=512), "ALIASING_VIOLATION"),
                     (dict(xs=512, x=at(0, 1020), y=at(0), ys=512), "ALIASING_VIOLATION"),
                     (dict(y=at(1)), "ALIASING_VIOLATION"), (dict(y=at(3)), "ALIASING_VIOLATION")]:
        assert rotary(**kw)[0] == want, kw
    assert passes(rotary(xs=512, x=at(0, 1024), y=at(0), ys=512))


def cache(type_id=kq_hip.TYPE_F16, heads=2, width=64, page=16, pages=9, line=4, keys=at(10),
          values=at(11), table=at(12), lengths=at(13)):
    return kq_hip.paged_cache(type_id, heads, width, page, pages, line, keys, values, table, lengths)


BAD_CACHES = [(dict(heads=0), "INVALID_ARGUMENT"), (dict(pages=0), "INVALID_ARGUMENT"),
              (dict(line=0), "INVALID_ARGUMENT"), (dict(keys=None), "INVALID_ARGUMENT"),
              (dict(values=None), "INVALID_ARGUMENT"), (dict(table=None), "INVALID_ARGUMENT"),
              (dict(lengths=None), "INVALID_ARGUMENT"),
              (dict(type_id=kq_hip.TYPE_F32), "UNSUPPORTED_TENSOR_TYPE"),
              (dict(type_id=kq_hip.TYPE_Q8_0), "UNSUPPORTED_TENSOR_TYPE"),
              (dict(heads=257), "LIMIT_EXCEEDED"), (dict(width=96), "LIMIT_EXCEEDED"),
              (dict(page=8), "LIMIT_EXCEEDED"), (dict(page=48), "LIMIT_EXCEEDED"),
              (dict(page=512), "LIMIT_EXCEEDED"),
              (dict(line=(1 << 20) + 1), "LIMIT_EXCEEDED"),
              (dict(keys=at(10, 8)), "INVALID_ALIGNMENT"),
              (dict(values=at(11, 2)), "INVALID_ALIGNMENT"),
              (dict(table=at(12, 2)), "INVALID_ALIGNMENT"),
              (dict(lengths=at(13, 1)), "INVALID_ALIGNMENT")]


def append(c=None, q=None, i=None, r=None, **rows):
    good = dict(key=at(0), key_stride=512, value=at(0, 512), value_stride=512, query_heads=4,
                query=at(0, 1024), query_stride=512, query_output=at(2), query_output_stride=256)
    i = kq_hip.cache_rows(**{**good, **rows})
    r = kq_hip.rotary(64, at(3)) if r is None else r
    return call("kq_hip_cache_append_f32", C.byref(c or cache()), C.byref(q or seqs()),
                C.byref(i), C.byref(r) if r else None)


def test_cache_append():
    R = kq_hip.rotary
    assert passes(append())
    assert passes(append(r=False))
    assert passes(append(query_heads=0, query=None, query_output=None, query_stride=0,
                         query_output_stride=0))
    assert passes(append(query_output=at(0, 1024), query_output_stride=512))  # in its own rows
    assert passes(append(cache(kq_hip.TYPE_BF16, page=256)))
    assert passes(append(q=seqs(3, 3, 5, None)))
    for kw, want in BAD_CACHES:
        assert append(cache(**kw))[0] == want, kw
    for kw, want in [(dict(key=None), "INVALID_ARGUMENT"), (dict(value=None), "INVALID_ARGUMENT"),
                     (dict(query=None), "INVALID_ARGUMENT"),
                     (dict(query_output=None), "INVALID_ARGUMENT"),
                     (dict(r=R(64, None)), "INVALID_ARGUMENT"),
                     (dict(r=R(66, at(3))), "DIMENSION_MISMATCH"),
                     (dict(r=R(64, at(3, 4))), "INVALID_ALIGNMENT"),
                     (dict(q=seqs(0)), "INVALID_ARGUMENT"), (dict(q=seqs(262145)), "LIMIT_EXCEEDED"),
                     (dict(q=seqs(4, 3, 5, None)), "DIMENSION_MISMATCH"),
                     (dict(query_heads=257, query_stride=1 << 15, query_output_stride=1 << 15),
                      "LIMIT_EXCEEDED"),
                     (dict(key_stride=124), "DIMENSION_MISMATCH"),
                     (dict(value_stride=124), "DIMENSION_MISMATCH"),
                     (dict(query_stride=252), "DIMENSION_MISMATCH"),
                     (dict(query_output_stride=252), "DIMENSION_MISMATCH"),
                     (dict(key_stride=514), "INVALID_ALIGNMENT"),
                     (dict(key=at(0, 8)), "INVALID_ALIGNMENT"),
                     (dict(value=at(0, 516)), "INVALID_ALIGNMENT"),
                     (dict(query_output=at(2, 4)), "INVALID_ALIGNMENT"),
                     (dict(query_output=at(0), query_output_stride=512), "ALIASING_VIOLATION"),
                     (dict(query_output=at(0, 1024)), "ALIASING_VIOLATION"),
                     (dict(query_output=at(10)), "ALIASING_VIOLATION"),
                     (dict(query_output=at(21)), "ALIASING_VIOLATION"),
                     (dict(query_output=at(3)), "ALIASING_VIOLATION"),
                     (dict(c=cache(values=at(10))), "ALIASING_VIOLATION"),
                     (dict(c=cache(values=at(10, 9 * 2 * 16 * 64 * 2 - 16))), "ALIASING_VIOLATION"),
                     (dict(c=cache(keys=at(0))), "ALIASING_VIOLATION"),
                     (dict(c=cache(keys=at(12))), "ALIASING_VIOLATION"),
                     (dict(c=cache(values=at(3))), "ALIASING_VIOLATION")]:
        assert append(**kw)[0] == want, kw
    assert passes(append(c=cache(values=at(10, 9 * 2 * 16 * 64 * 2))))


def attn(a=None, c=None, q=None, query=at(0), qs=256, gate=at(1), gs=256, y=at(2), ys=256,
         scratch=at(4), nbytes=1 << 27):
    a = a or kq_hip.paged_attention(4, 0.125, gate="sigmoid", sinks=at(5))
    return call("kq_hip_paged_attention_f32", C.byref(a), C.byref(c or cache()),
                C.byref(q or seqs()), query, qs, gate, gs, y, ys, scratch, nbytes)


def test_paged_attention():
    A = kq_hip.paged_attention
    assert passes(attn())
    assert passes(attn(A(4, -0.5, causal=False, window=7), gate=None, gs=0))
    assert passes(attn(qs=512, y=at(0, 1024), ys=512))
    assert passes(attn(q=seqs(3, 3, 5, None)))
    for kw, want in BAD_CACHES:
        assert attn(c=cache(**kw))[0] == want, kw
    need = kq_hip.paged_attention_scratch_bytes(A(4, 1.0), cache(), seqs())
    for kw, want in [(dict(query=None), "INVALID_ARGUMENT"), (dict(y=None), "INVALID_ARGUMENT"),
                     (dict(gate=None), "INVALID_ARGUMENT"), (dict(scratch=None), "INVALID_ARGUMENT"),
                     (dict(a=A(0, 1.0)), "INVALID_ARGUMENT"),
                     (dict(a=A(4, math.nan)), "INVALID_ARGUMENT"),
                     (dict(a=A(4, 1.0, gate="silu")), "INVALID_ARGUMENT"),
                     (dict(a=kq_hip.PagedAttention(4, 1.0, 2, 0, None, 0)), "INVALID_ARGUMENT"),
                     (dict(a=A(3, 1.0)), "DIMENSION_MISMATCH"),
                     (dict(a=A(258, 1.0), qs=1 << 15, ys=1 << 15), "LIMIT_EXCEEDED"),
                     (dict(q=seqs(count=0)), "INVALID_ARGUMENT"),
                     (dict(q=seqs(4, 3, 5, None)), "DIMENSION_MISMATCH"),
                     (dict(qs=252), "DIMENSION_MISMATCH"), (dict(gs=252), "DIMENSION_MISMATCH"),
                     (dict(ys=252), "DIMENSION_MISMATCH"),
                     (dict(nbytes=need - 1), "BUFFER_TOO_SMALL"),
                     (dict(query=at(0, 8)), "INVALID_ALIGNMENT"), (dict(qs=258), "INVALID_ALIGNMENT"),
                     (dict(y=at(2, 4)), "INVALID_ALIGNMENT"), (dict(gate=at(1, 8)), "INVALID_ALIGNMENT"),
                     (dict(scratch=at(4, 8)), "INVALID_ALIGNMENT"),
                     (dict(a=A(4, 1.0, sinks=at(5, 2))), "INVALID_ALIGNMENT"),
                     (dict(y=at(0)), "ALIASING_VIOLATION"), (dict(y=at(1)), "ALIASING_VIOLATION"),
                     (dict(y=at(4)), "ALIASING_VIOLATION"), (dict(y=at(10)), "ALIASING_VIOLATION"),
                     (dict(y=at(5)), "ALIASING_VIOLATION"), (dict(y=at(13)), "ALIASING_VIOLATION"),
                     (dict(scratch=at(0)), "ALIASING_VIOLATION"),
                     (dict(scratch=at(11)), "ALIASING_VIOLATION"),
                     (dict(scratch=at(12)), "ALIASING_VIOLATION")]:
        assert attn(**kw)[0] == want, kw


@pytest.mark.parametrize("name", ["kq_hip_rotary_f32", "kq_hip_cache_append_f32",
                                  "kq_hip_paged_attention_f32", "kq_hip_rotary_frequencies"])
def test_nothing_given(name):
    d = kq_hip.Diagnostic()
    fn = getattr(kq_hip.lib(), name)
    args = [None if t is C.c_void_p else 0 for t in fn.argtypes[:-1]]
    assert kq_hip.STATUS[fn(*args, C.byref(d))] == "INVALID_ARGUMENT"


def test_scratch_bytes():
    A, f = kq_hip.paged_attention, kq_hip.paged_attention_scratch_bytes
    assert f(A(3, 1.0), cache(), seqs()) == 0            # refused
    assert f(A(4, 1.0), cache(width=80), seqs()) == 0
    assert f(A(4, 1.0), cache(), seqs(0)) == 0
    # what the pointers are does not matter, nor how long the pool is
    assert f(A(4, 1.0), cache(keys=None, table=None, pages=1 << 20), seqs()) == \
        f(A(4, 1.0), cache(), seqs()) > 0
    # bounded for the largest calls
    big = kq_hip.paged_cache(kq_hip.TYPE_F16, 32, 256, 256, 1 << 20, 1 << 16, 0, 0, 0, 0)
    assert f(A(256, 1.0), big, seqs(262144, 65535, 65535)) < 400 << 20


@pytest.mark.parametrize("window", [0, 40, 500])
@pytest.mark.parametrize("group", [1, 8, 16, 17])
def test_scratch_of_the_largest_call_is_enough(group, window):
    f = kq_hip.paged_attention_scratch_bytes
    for heads in (1, 8):
        a = kq_hip.paged_attention(heads * group, 1.0, True, window)
        for width in (64, 128, 256):
            for line in (1, 8, 12, 20, 28, 40, 400):
                c = kq_hip.paged_cache(kq_hip.TYPE_F16, heads, width, 16, 9, line, 0, 0, 0, 0)
                largest = 0
                for n in (1, 2, 16, 33, 64, 65, 300):
                    one = f(a, c, kq_hip.sequences(n, n, n))
                    few, many = (f(a, c, kq_hip.sequences(t, n, n, 64)) for t in (n, 50 * n))
                    assert 0 < one <= many and few <= many and largest <= many
                    largest = many


def test_frequencies():
    """Against the formulas; powers and products of binary64 in another order are
    a few 2^-53 apart, each times its exponent's size (log of 1e7 is 16)."""
    F = kq_hip.rotary_frequencies
    for dims, base in ((2, 10000.0), (64, 10000.0), (126, 1e6), (1024, 1e7)):
        i = np.arange(dims // 2)
        plain = np.exp(-2 * i / dims * math.log(base))
        f, m = F(dims, base)
        assert m == 1.0 and np.allclose(f, plain, rtol=1e-14, atol=0)
        f, m = F(dims, base, "linear", 4.0)
        assert m == 1.0 and np.allclose(f, plain / 4, rtol=1e-14, atol=0)
        div = np.linspace(1, 8, dims // 2).astype(np.float32)
        f, m = F(dims, base, divisors=div)
        assert np.allclose(f, plain / div, rtol=1e-14, atol=0)
        f, m = F(dims, base, "bands", 8.0, 32768.0)
        assert m == np.float32(0.1 * math.log(8.0) + 1)
        turns = plain * 32768 / (2 * math.pi)
        ends = np.sort(np.stack([plain, plain / 8]), 0)
        assert (f >= ends[0] * (1 - 1e-14)).all() and (f <= ends[1] * (1 + 1e-14)).all()
        assert (np.diff(f) < 0).all()
        # an index away from both borders, frequencies are all of one kind
        step = base ** (2.0 / dims)
        assert np.allclose(f[turns > 32 * step], plain[turns > 32 * step], rtol=1e-14, atol=0)
        assert np.allclose(f[turns < 1 / step], plain[turns < 1 / step] / 8, rtol=1e-14, atol=0)
    # an original context in which nothing, or everything, turns often enough
    plain = F(64, 1e4)[0]
    assert np.array_equal(F(64, 1e4, "bands", 8.0, 6.0)[0], plain / 8)
    assert np.array_equal(F(64, 1e4, "bands", 8.0, 1e9)[0], plain)
    f, _ = F(128, 1e6, "bands", 8.0, 32768.0)
    # a straight line between the borders
    low = math.floor(128 * math.log(32768 / (32 * 2 * math.pi)) / (2 * math.log(1e6)))
    high = math.ceil(128 * math.log(32768 / (2 * math.pi)) / (2 * math.log(1e6)))
    i = (low + high) // 2
    slow = (i - low) / (high - low)
    want = 1e6 ** (-2 * i / 128) * (1 - slow + slow / 8)
    assert 0 < slow < 1 and abs(f[i] / want - 1) < 1e-14


@pytest.mark.parametrize("kw,want", [
    (dict(dims=0), "LIMIT_EXCEEDED"), (dict(dims=7), "LIMIT_EXCEEDED"),
    (dict(dims=1026), "LIMIT_EXCEEDED"), (dict(base=1.0), "INVALID_ARGUMENT"),
    (dict(base=math.nan), "INVALID_ARGUMENT"),
    (dict(scaling="linear", factor=0.5), "INVALID_ARGUMENT"),
    (dict(scaling="bands", factor=2.0), "INVALID_ARGUMENT"),
    (dict(scaling="bands", factor=2.0, original_context=4096.0, slow=0.0), "INVALID_ARGUMENT"),
    (dict(scaling="bands", factor=2.0, original_context=4096.0, fast=1.0), "INVALID_ARGUMENT"),
    (dict(divisors=[1.0] * 31 + [0.0]), "INVALID_ARGUMENT"),
    (dict(divisors=[math.inf] + [1.0] * 31), "INVALID_ARGUMENT")])
def test_frequencies_refused(kw, want):
    with pytest.raises(kq_hip.KqError) as e:
        kq_hip.rotary_frequencies(**{**dict(dims=64, base=1e4), **kw})
    assert e.value.name == want


def test_definitions():
    """The binary64 definitions that the device tests compare with: a rotation
    keeps a pair's length, bf16 rounds to even, a uniform attention is a mean."""
    x = np.random.default_rng(1).standard_normal((3, 2, 8))
    for pairs in (False, True):
        y, _ = paged64.turn(x, [0, 5, 1 << 20], np.array([1.0, 0.1, 0.01]), pairs=pairs)
        assert np.array_equal(y[0], x[0]) and np.array_equal(y[..., 6:], x[..., 6:])
        assert np.allclose((y[..., :6] ** 2).sum(-1), (x[..., :6] ** 2).sum(-1))
    assert list(paged64.bf16_bits(np.array([1.0, 1.00390625, 1.01171875], np.float32))) == [
        0x3F80, 0x3F80, 0x3F82]
    keys = np.zeros((3, 1, 16, 4), np.float32)
    values = np.random.default_rng(2).standard_normal((3, 1, 16, 4)).astype(np.float32)
    y = paged64.attention(np.ones((2, 1, 4)), keys, values, [[2, 0]], [16], [(0, 2)], [0], None,
                          1.0, out=np.zeros((2, 1, 4)))
    assert np.allclose(y[0, 0], np.concatenate([values[2, 0], values[0, 0, :1]]).mean(0))
    assert np.allclose(y[1, 0], np.concatenate([values[2, 0], values[0, 0, :2]]).mean(0))
