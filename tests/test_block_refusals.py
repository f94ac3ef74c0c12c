"""What layer norm with statistics, rotary positions and windowed attention
refuse: each call is turned down on the host, before any device is touched, so
these run without one. The packets point at host memory that nothing reads."""
import ctypes

import numpy as np
import pytest

import chelis_amd as C

EDOMAIN, EUNSUPPORTED = 1, 2
F32, F64, I32, I64, BF16, F16 = C.DT_F32, C.DT_F64, C.DT_I32, C.DT_I64, C.DT_BF16, C.DT_F16
KEEP = []


def tensor(shape, dtype=F32, strides=None, room=1 << 20):
    """A packet over `room` bytes of its own."""
    if strides is None:
        strides, step = [], 1
        for n in reversed(shape):
            strides.insert(0, step)
            step *= max(1, n)
    buf = np.zeros(room, np.uint8)
    g, keep = C.make_packet(shape, strides, buf.ctypes.data, room, dtype)
    KEEP.append((buf, keep))
    return g


def at(t, shape, strides, dtype=F32):
    """Another packet over t's storage."""
    g, keep = C.make_packet(shape, strides, t.data, 1 << 20, dtype)
    KEEP.append(keep)
    return g


def refused(status, text, code):
    message = C.lib().chelis_hip_last_error().decode()
    assert status == code, (status, message)
    assert text in message, message


def ref(t):
    return ctypes.byref(t) if t is not None else None


def stats(x=None, gamma=None, beta=None, y=None, mean=None, rstd=None):
    x = x or tensor((4, 16))
    return C.lib().chelis_hip_layer_norm_stats(
        ref(x), ref(gamma or tensor((16,), x.dtype)), ref(beta or tensor((16,), x.dtype)), 1e-5,
        ref(y or tensor((4, 16), x.dtype)), ref(mean or tensor((4,))), ref(rstd or tensor((4,))))


@pytest.mark.parametrize("change,text,code", [
    (lambda: dict(x=tensor((4, 16), I32)), "x must be f32, f64, bf16 or f16", EDOMAIN),
    (lambda: dict(x=tensor((), F32)), "needs a last axis", EDOMAIN),
    (lambda: dict(y=tensor((4, 15))), "y must match x", EDOMAIN),
    (lambda: dict(y=tensor((4, 16), F16)), "y must match x", EDOMAIN),
    (lambda: dict(y=tensor((4, 16), F32, (8, 1))), "y overlaps itself", EDOMAIN),
    (lambda: dict(x=tensor((4, 16), F32, (16, 2))), "last axis must be contiguous", EUNSUPPORTED),
    (lambda: dict(gamma=tensor((15,))), "gamma must be contiguous", EDOMAIN),
    (lambda: dict(gamma=tensor((16,), F32, (2,))), "gamma must be contiguous", EDOMAIN),
    (lambda: dict(beta=tensor((16,), F64)), "beta must have x's dtype", EDOMAIN),
    (lambda: dict(x=tensor((4, 16), BF16), gamma=tensor((16,), F32)), "gamma and beta must share", EDOMAIN),
    (lambda: dict(mean=tensor((4,), F64)), "mean must be f32", EDOMAIN),
    (lambda: dict(rstd=tensor((4, 1))), "rstd must be contiguous", EDOMAIN),
    (lambda: dict(rstd=tensor((4,), F32, (2,))), "rstd must be contiguous", EDOMAIN),
    (lambda: dict(x=tensor((4, 0)), gamma=tensor((0,)), beta=tensor((0,)), y=tensor((4, 0))), "hidden extent", EDOMAIN),
    (lambda: dict(x=tensor((4, 16), F32, room=32)), "past byte_capacity", EDOMAIN),
])
def test_layer_norm_stats(change, text, code):
    refused(stats(**change()), text, code)


def test_layer_norm_stats_in_place_needs_the_same_rows():
    x = tensor((4, 16), F32, (20, 1))
    refused(stats(x=x, y=at(x, (4, 16), (16, 1))), "overlaps an input with other strides", EDOMAIN)


def adjoint(x=None, gamma=None, mean=None, rstd=None, g=None, dx=0, dgamma=0, dbeta=0):
    x = x or tensor((4, 16))
    made = lambda t, shape: tensor(shape, x.dtype) if t == 0 else t
    return C.lib().chelis_hip_layer_norm_adjoint(
        ref(x), ref(gamma or tensor((16,), x.dtype)), ref(mean or tensor((4,))), ref(rstd or tensor((4,))),
        ref(g or tensor((4, 16), x.dtype)), ref(made(dx, (4, 16))), ref(made(dgamma, (16,))), ref(made(dbeta, (16,))))


@pytest.mark.parametrize("change,text,code", [
    (lambda: dict(dx=None, dgamma=None, dbeta=None), "no gradient asked for", EDOMAIN),
    (lambda: dict(dgamma=None), "come together", EDOMAIN),
    (lambda: dict(g=tensor((4, 8))), "g must match x", EDOMAIN),
    (lambda: dict(dx=tensor((4, 16), F64)), "dx must match x", EDOMAIN),
    (lambda: dict(dx=tensor((4, 16), F32, (0, 1))), "dx overlaps itself", EDOMAIN),
    (lambda: dict(dgamma=tensor((16,), F16)), "dgamma must have x's dtype", EDOMAIN),
    (lambda: dict(x=tensor((4, 16), F16), dgamma=tensor((16,)), dbeta=tensor((16,))), "must have gamma's dtype", EDOMAIN),
    (lambda: dict(mean=tensor((5,))), "mean must be contiguous", EDOMAIN),
    (lambda: dict(x=tensor((4, 16), F64)), "mean must be f32 (f64", EDOMAIN),
])
def test_layer_norm_adjoint(change, text, code):
    refused(adjoint(**change()), text, code)


def test_layer_norm_adjoint_weights_apart():
    d = tensor((16,))
    refused(adjoint(dgamma=d, dbeta=at(d, (16,), (1,))), "dgamma and dbeta overlap", EDOMAIN)


def turn(xs=None, ys=None, positions=None, freqs=None, sections=(3, 5), pairing=0, n=None):
    xs = xs or [tensor((2, 4, 6, 16))]
    ys = ys or [tensor(tuple(x.shape[i] for i in range(x.rank)), x.dtype) for x in xs]
    arr = lambda ts: (C.P * len(ts))(*[ctypes.pointer(t) for t in ts])
    return C.lib().chelis_hip_rotary(arr(xs), len(xs) if n is None else n, ref(positions or tensor((2, 2, 6), I32)),
                                     ref(freqs or tensor((8,), F64)), (ctypes.c_int64 * len(sections))(*sections),
                                     len(sections), pairing, arr(ys))


@pytest.mark.parametrize("change,text,code", [
    (lambda: dict(n=0), "one or two tensors", EDOMAIN),
    (lambda: dict(n=3), "one or two tensors", EDOMAIN),
    (lambda: dict(pairing=2), "unknown pairing", EDOMAIN),
    (lambda: dict(sections=(1,) * 9), "1 to 8 position axes", EDOMAIN),
    (lambda: dict(sections=(3, 0)), "sections must be positive", EDOMAIN),
    (lambda: dict(sections=(3, 6)), "9 pairs do not fit a width of 16", EDOMAIN),
    (lambda: dict(sections=(3, 4)), "freqs must be contiguous f64 [pairs]", EDOMAIN),
    (lambda: dict(xs=[tensor((4, 6, 16))]), "[batch, heads, seq, width]", EDOMAIN),
    (lambda: dict(xs=[tensor((2, 4, 6, 16), I32)]), "[batch, heads, seq, width]", EDOMAIN),
    (lambda: dict(xs=[tensor((2, 4, 6, 16)), tensor((2, 4, 7, 16))]), "differ in more than their heads", EDOMAIN),
    (lambda: dict(xs=[tensor((2, 4, 6, 16)), tensor((2, 4, 6, 16), F16)]), "differ in more than their heads", EDOMAIN),
    (lambda: dict(ys=[tensor((2, 4, 6, 16), F16)]), "share a shape and a dtype", EDOMAIN),
    (lambda: dict(ys=[tensor((2, 4, 6, 16), F32, (384, 0, 16, 1))]), "y overlaps itself", EDOMAIN),
    (lambda: dict(xs=[tensor((2, 4, 6, 16), F32, (768, 192, 32, 2))]), "last axis must be contiguous", EUNSUPPORTED),
    (lambda: dict(positions=tensor((2, 2, 6), F32)), "positions must be i32 or i64", EDOMAIN),
    (lambda: dict(positions=tensor((1, 2, 6), I32)), "positions must be i32 or i64", EDOMAIN),
    (lambda: dict(freqs=tensor((8,), F32)), "freqs must be contiguous f64", EDOMAIN),
])
def test_rotary(change, text, code):
    refused(turn(**change()), text, code)


def test_rotary_in_place_needs_the_same_view():
    x = tensor((2, 4, 6, 16))
    other = at(x, (2, 4, 6, 16), (384, 16, 64, 1))
    refused(turn(xs=[x], ys=[other]), "overlaps an input with other strides", EDOMAIN)
    y = tensor((2, 4, 6, 16))
    refused(turn(xs=[x, tensor((2, 4, 6, 16))], ys=[y, at(y, (2, 4, 6, 16), (384, 96, 16, 1))]), "results overlap", EDOMAIN)


def attend(q=None, k=None, v=None, lengths=None, starts=None, window=4, sinks=1, scale=0.1, o=None, lse=None):
    q = q or tensor((2, 4, 6, 16))
    k = k or tensor((2, 2, 9, 16), q.dtype)
    return C.lib().chelis_hip_window_attention(
        ref(q), ref(k), ref(v or tensor(tuple(k.shape[i] for i in range(k.rank)), k.dtype)), ref(lengths), ref(starts),
        window, sinks, scale, ref(o or tensor(tuple(q.shape[i] for i in range(q.rank)), q.dtype)), ref(lse))


WINDOW = [
    (lambda: dict(q=tensor((2, 4, 6, 16), F64)), "q must be f32, bf16 or f16", EDOMAIN),
    (lambda: dict(q=tensor((4, 6, 16))), "[batch, heads, seq, width]", EDOMAIN),
    (lambda: dict(k=tensor((2, 2, 9, 16), BF16)), "k must have q's dtype", EDOMAIN),
    (lambda: dict(k=tensor((1, 2, 9, 16))), "share batch and width", EDOMAIN),
    (lambda: dict(k=tensor((2, 2, 9, 8))), "share batch and width", EDOMAIN),
    (lambda: dict(k=tensor((2, 3, 9, 16))), "4 query heads over 3 key heads", EDOMAIN),
    (lambda: dict(k=tensor((2, 0, 9, 16))), "4 query heads over 0 key heads", EDOMAIN),
    (lambda: dict(v=tensor((2, 2, 8, 16))), "v must have k's shape", EDOMAIN),
    (lambda: dict(q=tensor((2, 4, 6, 12)), k=tensor((2, 2, 9, 12))), "a multiple of 8 up to 128", EUNSUPPORTED),
    (lambda: dict(q=tensor((2, 4, 6, 136)), k=tensor((2, 2, 9, 136))), "a multiple of 8 up to 128", EUNSUPPORTED),
    (lambda: dict(q=tensor((2, 4, 6, 16), F32, (768, 192, 32, 2))), "last axis must be contiguous", EUNSUPPORTED),
    (lambda: dict(window=0), "window must be at least 1", EDOMAIN),
    (lambda: dict(sinks=-1), "sinks not negative", EDOMAIN),
    (lambda: dict(scale=float("nan")), "scale must be finite", EDOMAIN),
    (lambda: dict(scale=1e39), "scale must be finite", EDOMAIN),
    (lambda: dict(lengths=tensor((2,), F32)), "lengths must be i32 or i64 [batch]", EDOMAIN),
    (lambda: dict(lengths=tensor((3,), I32)), "lengths must be i32 or i64 [batch]", EDOMAIN),
    (lambda: dict(starts=tensor((2, 1), I64)), "starts must be i32 or i64 [batch]", EDOMAIN),
    (lambda: dict(o=tensor((2, 4, 5, 16))), "o must have q's shape", EDOMAIN),
    (lambda: dict(o=tensor((2, 4, 6, 16), F32, (384, 96, 0, 1))), "o overlaps itself", EDOMAIN),
    (lambda: dict(lse=tensor((2, 4, 6), F64)), "lse must be contiguous f32", EDOMAIN),
    (lambda: dict(lse=tensor((2, 6, 4))), "lse must be contiguous f32", EDOMAIN),
]


@pytest.mark.parametrize("change,text,code", WINDOW)
def test_window_attention(change, text, code):
    refused(attend(**change()), text, code)


def test_window_attention_result_apart():
    q = tensor((2, 4, 6, 16))
    refused(attend(q=q, o=at(q, (2, 4, 6, 16), (384, 96, 16, 1))), "o overlaps another operand", EDOMAIN)


def adjoint_of(**change):
    t = dict(q=tensor((2, 4, 6, 16)), k=tensor((2, 2, 9, 16)), v=tensor((2, 2, 9, 16)), o=tensor((2, 4, 6, 16)),
             lse=tensor((2, 4, 6)), g=tensor((2, 4, 6, 16)), lengths=None, starts=None, window=4, sinks=1, scale=0.1,
             dq=tensor((2, 4, 6, 16)), dk=tensor((2, 2, 9, 16)), dv=tensor((2, 2, 9, 16)))
    t.update(change)
    order = ("q", "k", "v", "o", "lse", "g", "lengths", "starts", "window", "sinks", "scale", "dq", "dk", "dv")
    return C.lib().chelis_hip_window_attention_adjoint(*(
        t[n] if n in ("window", "sinks", "scale") else ref(t[n]) for n in order))


@pytest.mark.parametrize("change,text,code", [
    (lambda: dict(g=tensor((2, 4, 6, 8))), "g must have q's shape", EDOMAIN),
    (lambda: dict(o=tensor((2, 4, 6, 16), F16)), "o must have q's dtype", EDOMAIN),
    (lambda: dict(dk=tensor((2, 4, 9, 16))), "dk must have k's shape", EDOMAIN),
    (lambda: dict(dv=tensor((2, 2, 9, 16), F32, (0, 144, 16, 1))), "dv overlaps itself", EDOMAIN),
    (lambda: dict(lse=tensor((2, 4, 7))), "lse must be contiguous f32", EDOMAIN),
    (lambda: dict(lse=None), "null tensor packet", EDOMAIN),
    (lambda: dict(window=-1), "window must be at least 1", EDOMAIN),
    (lambda: dict(dq=None), "null tensor packet", EDOMAIN),
])
def test_window_attention_adjoint(change, text, code):
    refused(adjoint_of(**change()), text, code)


@pytest.mark.parametrize("out,into", [("dq", "q"), ("dk", "k"), ("dv", "k"), ("dv", "dk"), ("dq", "g")])
def test_window_attention_adjoint_results_apart(out, into):
    like = (2, 4, 6, 16) if into in ("q", "g") else (2, 2, 9, 16)
    t = tensor(like)
    refused(adjoint_of(**{into: t, out: at(t, like, (like[1] * like[2] * 16, like[2] * 16, 16, 1))}),
            "overlaps another operand", EDOMAIN)
