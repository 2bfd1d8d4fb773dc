"""What the operators around the GDN attention refuse before any device work:
statuses of the host's checks. CPU only: a context that was never opened
stands in for one, and a call that passes every check ends at it."""
import ctypes as C

import pytest

import kq_hip

NO_CONTEXT = C.create_string_buffer(4096)  # zeros: no stream
A = 0x10000000  # addresses that no check may read through


def at(i, offset=0):
    return A + i * 0x10000000 + offset


def call(name, *args):
    d = kq_hip.Diagnostic()
    st = getattr(kq_hip.lib(), name)(C.cast(NO_CONTEXT, C.c_void_p), *args, C.byref(d))
    return kq_hip.STATUS[st], d.message.decode()


def passes(got):
    return got == ("INVALID_ARGUMENT", "valid context is required")


def seqs(tokens=10, count=3, pool=5, offsets=at(20), slots=at(21), fresh=at(22)):
    return kq_hip.sequences(tokens, count, pool, offsets, slots, fresh)


def conv(c=None, q=None, x=at(0), xs=64, state=at(1), out=at(2), y=at(3), ys=64):
    c = c or kq_hip.causal_conv(64, 4, at(4), at(5))
    q = q or seqs()
    return call("kq_hip_causal_conv_f32", C.byref(c), C.byref(q), x, xs, state, out, y, ys)


def test_conv():
    assert passes(conv())
    assert passes(conv(state=at(1), out=at(1)))
    assert passes(conv(kq_hip.causal_conv(64, 2, at(4)), seqs(3, 3, 3, None, None, None)))
    bad = [(dict(c=kq_hip.causal_conv(0, 4, at(4))), "INVALID_ARGUMENT"),
           (dict(c=kq_hip.causal_conv(64, 4, None)), "INVALID_ARGUMENT"),
           (dict(c=kq_hip.causal_conv(64, 4, at(4), activation="sigmoid")), "INVALID_ARGUMENT"),
           (dict(c=kq_hip.causal_conv(64, 1, at(4))), "LIMIT_EXCEEDED"),
           (dict(c=kq_hip.causal_conv(64, 9, at(4))), "LIMIT_EXCEEDED"),
           (dict(x=None), "INVALID_ARGUMENT"), (dict(state=None), "INVALID_ARGUMENT"),
           (dict(q=seqs(0)), "INVALID_ARGUMENT"), (dict(q=seqs(count=0)), "INVALID_ARGUMENT"),
           (dict(q=seqs(pool=0)), "INVALID_ARGUMENT"),
           (dict(q=seqs(262145)), "LIMIT_EXCEEDED"), (dict(q=seqs(count=65536)), "LIMIT_EXCEEDED"),
           (dict(q=seqs(offsets=None)), "DIMENSION_MISMATCH"),
           (dict(q=seqs(count=6, slots=None)), "DIMENSION_MISMATCH"),
           (dict(q=seqs(offsets=at(20, 2))), "INVALID_ALIGNMENT"),
           (dict(xs=63), "DIMENSION_MISMATCH"), (dict(ys=63), "DIMENSION_MISMATCH"),
           (dict(x=at(0, 1)), "INVALID_ALIGNMENT"),
           (dict(y=at(0)), "ALIASING_VIOLATION"),                 # over the input
           (dict(out=at(1, 16)), "ALIASING_VIOLATION"),           # a part of the state
           (dict(out=at(3)), "ALIASING_VIOLATION"),               # two outputs
           (dict(y=at(21)), "ALIASING_VIOLATION")]                # over the slots
    for kw, want in bad:
        assert conv(**kw)[0] == want, kw


def attn(a=None, q=None, i=None, state=at(1), out=at(2), y=at(3), ys=256, scratch=at(9),
         nbytes=1 << 27):
    a = a or kq_hip.linear_attention(2, 4, 64, 64, 0.125, at(4), at(5))
    q = q or seqs()
    i = i or kq_hip.linear_attention_inputs(at(6), 512, at(6, 512), 512, at(6, 1024), 512, at(7), 4,
                                            at(8), 4)
    return call("kq_hip_linear_attention_f32", C.byref(a), C.byref(q), C.byref(i), state, out, y,
                ys, scratch, nbytes)


def test_linear_attention():
    L, I = kq_hip.linear_attention, kq_hip.linear_attention_inputs
    assert passes(attn())
    assert passes(attn(out=at(1)))
    assert passes(attn(i=I(at(6), 128, at(10), 128, at(11), 256)))
    assert passes(attn(q=seqs(3, 3, 5, None), scratch=None, nbytes=0))
    good = dict(key_heads=2, value_heads=4, key_width=64, value_width=64, scale=0.1, rate=at(4))
    for change, want in [(dict(key_heads=0), "INVALID_ARGUMENT"),
                         (dict(scale=float("nan")), "INVALID_ARGUMENT"),
                         (dict(epsilon=0.0), "INVALID_ARGUMENT"),
                         (dict(epsilon=1e-21), "INVALID_ARGUMENT"),
                         (dict(rate=None), "INVALID_ARGUMENT"),
                         (dict(key_heads=3), "DIMENSION_MISMATCH"),
                         (dict(value_heads=258), "LIMIT_EXCEEDED"),
                         (dict(key_width=96), "LIMIT_EXCEEDED"),
                         (dict(value_width=32), "LIMIT_EXCEEDED")]:
        assert attn(a=L(**{**good, **change}))[0] == want, change
    assert passes(attn(a=L(**{**good, "normalize": False, "epsilon": 0.0})))
    inp = dict(query=at(6), query_stride=128, key=at(10), key_stride=128, value=at(11),
               value_stride=256, alpha=at(7), alpha_stride=4, beta=at(8), beta_stride=4)
    for change, want in [(dict(query=None), "INVALID_ARGUMENT"),
                         (dict(query_stride=124), "DIMENSION_MISMATCH"),
                         (dict(value_stride=252), "DIMENSION_MISMATCH"),
                         (dict(alpha_stride=3), "DIMENSION_MISMATCH"),
                         (dict(beta_stride=3), "DIMENSION_MISMATCH"),
                         (dict(query_stride=130), "INVALID_ALIGNMENT"),
                         (dict(key=at(10, 4)), "INVALID_ALIGNMENT"),
                         (dict(alpha=at(7, 2)), "INVALID_ALIGNMENT")]:
        assert attn(i=I(**{**inp, **change}))[0] == want, change
    assert attn(ys=255)[0] == "DIMENSION_MISMATCH"
    assert attn(y=at(6))[0] == "ALIASING_VIOLATION"
    assert attn(out=at(1, 64))[0] == "ALIASING_VIOLATION"
    assert attn(y=at(2))[0] == "ALIASING_VIOLATION"
    assert attn(q=seqs(9, 3, 5, None))[0] == "DIMENSION_MISMATCH"


def norm(n=None, tokens=5, x=at(0), xs=256, gate=at(1), gs=256, y=at(2), ys=256):
    n = n or kq_hip.gated_norm(4, 64, 1e-6, at(3), gate="silu")
    return call("kq_hip_gated_norm_f32", C.byref(n), tokens, x, xs, gate, gs, y, ys)


def test_gated_norm():
    N = kq_hip.gated_norm
    assert passes(norm())
    assert passes(norm(y=at(0))) and passes(norm(y=at(1)))
    assert passes(norm(N(4, 64, 1e-6), gate=None, gs=0))
    for kw, want in [(dict(tokens=0), "INVALID_ARGUMENT"), (dict(gate=None), "INVALID_ARGUMENT"),
                     (dict(n=N(0, 64, 1e-6)), "INVALID_ARGUMENT"),
                     (dict(n=N(4, 64, 0.0)), "INVALID_ARGUMENT"),
                     (dict(n=N(4, 64, 1e-6, weight_offset=float("inf"))), "INVALID_ARGUMENT"),
                     (dict(n=N(1, 16385, 1e-6)), "LIMIT_EXCEEDED"),
                     (dict(tokens=262145), "LIMIT_EXCEEDED"),
                     (dict(xs=255), "DIMENSION_MISMATCH"), (dict(gs=255), "DIMENSION_MISMATCH"),
                     (dict(x=at(0, 2)), "INVALID_ALIGNMENT"),
                     (dict(y=at(0), ys=260), "ALIASING_VIOLATION"),
                     (dict(y=at(0, 4)), "ALIASING_VIOLATION"),
                     (dict(y=at(3)), "ALIASING_VIOLATION")]:
        assert norm(**kw)[0] == want, kw


def join(j=None, tokens=5, block=at(0), gate=at(1), residual=at(2), branch=at(3), out=at(4),
         normalized=at(5)):
    j = j or kq_hip.block_join(4, 64, 1e-6, post=at(6), gate="silu", pre=at(7))
    return call("kq_hip_block_join_f32", C.byref(j), tokens, block, gate, residual, branch, out,
                normalized)


def test_block_join():
    J = kq_hip.block_join
    assert passes(join())
    assert passes(join(out=at(2)))
    assert passes(join(J(1, 64, 0.0), gate=None, branch=None, normalized=None))
    for kw, want in [(dict(tokens=0), "INVALID_ARGUMENT"), (dict(gate=None), "INVALID_ARGUMENT"),
                     (dict(normalized=None), "INVALID_ARGUMENT"),
                     (dict(j=J(4, 64, 1e-6)), "INVALID_ARGUMENT"),
                     (dict(j=J(4, 64, 0.0, pre=at(7))), "INVALID_ARGUMENT"),
                     (dict(j=J(4, 64, 1e-6, scale=float("nan"), pre=at(7))), "INVALID_ARGUMENT"),
                     (dict(j=J(65, 64, 1e-6, pre=at(7))), "LIMIT_EXCEEDED"),
                     (dict(j=J(4, 16385, 1e-6, pre=at(7))), "LIMIT_EXCEEDED"),
                     (dict(block=at(0, 1)), "INVALID_ALIGNMENT"),
                     (dict(out=at(2, 16)), "ALIASING_VIOLATION"),
                     (dict(normalized=at(4)), "ALIASING_VIOLATION"),
                     (dict(normalized=at(2)), "ALIASING_VIOLATION"),
                     (dict(out=at(0)), "ALIASING_VIOLATION")]:
        assert join(**kw)[0] == want, kw


@pytest.mark.parametrize("name", ["kq_hip_causal_conv_f32", "kq_hip_linear_attention_f32",
                                  "kq_hip_gated_norm_f32", "kq_hip_block_join_f32"])
def test_nothing_given(name):
    d = kq_hip.Diagnostic()
    fn = getattr(kq_hip.lib(), name)
    args = [None if t is C.c_void_p else 0 for t in fn.argtypes[:-1]]
    assert kq_hip.STATUS[fn(*args, C.byref(d))] == "INVALID_ARGUMENT"


def test_scratch_bytes():
    a = kq_hip.linear_attention(16, 48, 128, 128, 0.1, at(4))
    f = kq_hip.linear_attention_scratch_bytes
    assert f(a, seqs(3, 3, 5, None)) == 0  # one row a sequence: none
    assert f(a, seqs(0)) == 0              # refused
    assert f(kq_hip.linear_attention(16, 40, 128, 128, 0.1, at(4)), seqs()) == 0


# an output that is the input it may be, where another input lies there too: that
# one is read by other workgroups than those that write it
def test_second_input_at_the_output():
    assert conv(x=at(1), state=at(1), out=at(1))[0] == "ALIASING_VIOLATION"
    assert conv(kq_hip.causal_conv(64, 4, at(1)), state=at(1), out=at(1))[0] == "ALIASING_VIOLATION"
    i = kq_hip.linear_attention_inputs(at(1), 128, at(10), 128, at(11), 256)
    assert attn(i=i, state=at(1), out=at(1))[0] == "ALIASING_VIOLATION"
    assert attn(q=seqs(slots=at(1)), state=at(1), out=at(1))[0] == "ALIASING_VIOLATION"
    assert join(block=at(2), out=at(2))[0] == "ALIASING_VIOLATION"
    assert join(gate=at(2), out=at(2))[0] == "ALIASING_VIOLATION"
    assert join(branch=at(2), out=at(2))[0] == "ALIASING_VIOLATION"
    # the other inputs may lie together
    assert passes(join(block=at(2), gate=at(2)))
    assert passes(join(block=at(1), gate=at(1), out=at(2)))
