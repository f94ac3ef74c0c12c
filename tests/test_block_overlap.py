"""Calls of the block operators whose results share storage with an operand
that they may not share it with: refused on the host, before any device is
touched. The packets lie in one host buffer that nothing reads."""
import ctypes

import numpy as np
import pytest

import chelis_amd as C

EDOMAIN = 1
BYTE = {C.DT_F32: 4, C.DT_F64: 8, C.DT_I32: 4, C.DT_I64: 8, C.DT_BF16: 2, C.DT_F16: 2}
ROOM = 1 << 20
ARENA = np.zeros(ROOM, np.uint8)
KEEP = []


def at(byte, shape, strides=None, dtype=C.DT_F32):
    """A packet whose first element lies at `byte` of the buffer."""
    if strides is None:
        strides, step = [], 1
        for n in reversed(shape):
            strides.insert(0, step)
            step *= max(1, n)
    assert byte % BYTE[dtype] == 0
    g, keep = C.make_packet(shape, strides, ARENA.ctypes.data + byte, ROOM - byte, dtype)
    KEEP.append(keep)
    return g


def refused(status, text):
    message = C.lib().chelis_hip_last_error().decode()
    assert status == EDOMAIN, (status, message)
    assert text in message, message


def ref(t):
    return ctypes.byref(t) if t is not None else None


def step(n):
    """Storage of its own for the n-th operand."""
    return n * 32768


def stats(**change):
    t = dict(x=at(0, (4, 16)), gamma=at(step(1), (16,)), beta=at(step(2), (16,)), y=at(step(3), (4, 16)),
             mean=at(step(4), (4,)), rstd=at(step(5), (4,)))
    t.update(change)
    return C.lib().chelis_hip_layer_norm_stats(ref(t["x"]), ref(t["gamma"]), ref(t["beta"]), 1e-5, ref(t["y"]),
                                               ref(t["mean"]), ref(t["rstd"]))


@pytest.mark.parametrize("change,text", [
    (dict(y=at(64, (4, 16))), "y overlaps an input"),                  # one row further on
    (dict(y=at(4, (4, 16))), "y overlaps an input"),                   # one element further on
    (dict(x=at(0, (4, 16), (32, 1)), y=at(0, (4, 16), (16, 1))), "y overlaps an input"),
    (dict(y=at(step(1), (4, 16))), "y and gamma overlap"),
    (dict(y=at(step(2) - 252, (4, 16))), "y and beta overlap"),        # its last element is beta's first
    (dict(y=at(step(4), (4, 16))), "y and mean overlap"),
    (dict(y=at(step(5) - 64, (4, 16), (17, 1))), "y and rstd overlap"),
    (dict(mean=at(step(5) + 12, (4,))), "mean and rstd overlap"),
    (dict(mean=at(240, (4,))), "mean and x overlap"),
    (dict(rstd=at(step(1), (4,))), "rstd and gamma overlap"),
])
def test_layer_norm_stats(change, text):
    refused(stats(**change), text)


def norm_adjoint(**change):
    t = dict(x=at(0, (4, 16)), gamma=at(step(1), (16,)), mean=at(step(2), (4,)), rstd=at(step(3), (4,)),
             g=at(step(4), (4, 16)), dx=at(step(5), (4, 16)), dgamma=at(step(6), (16,)), dbeta=at(step(7), (16,)))
    t.update(change)
    return C.lib().chelis_hip_layer_norm_adjoint(*(ref(t[n]) for n in (
        "x", "gamma", "mean", "rstd", "g", "dx", "dgamma", "dbeta")))


@pytest.mark.parametrize("change,text", [
    (dict(dx=at(step(4) + 4, (4, 16))), "dx overlaps an input"),
    (dict(dx=at(step(1), (4, 16))), "dx and gamma overlap"),
    (dict(dx=at(step(2), (4, 16))), "dx and mean overlap"),
    (dict(dx=at(step(3) - 64, (4, 16))), "dx and rstd overlap"),
    (dict(dgamma=at(step(5) + 128, (16,))), "dgamma and dx overlap"),
    (dict(dgamma=at(step(1), (16,))), "dgamma and gamma overlap"),
    (dict(dgamma=at(step(7) + 4, (16,))), "dgamma and dbeta overlap"),
    (dict(dbeta=at(step(4), (16,)), dx=None), "dbeta and g overlap"),
    (dict(dbeta=at(step(3), (16,))), "dbeta and rstd overlap"),
    (dict(dbeta=at(128, (16,))), "dbeta and x overlap"),
])
def test_layer_norm_adjoint(change, text):
    refused(norm_adjoint(**change), text)


def turn(xs, ys, positions=None, freqs=None):
    arr = lambda ts: (C.P * len(ts))(*[ctypes.pointer(t) for t in ts])
    return C.lib().chelis_hip_rotary(arr(xs), len(xs), ref(positions or at(step(8), (2, 2, 6), dtype=C.DT_I32)),
                                     ref(freqs or at(step(9), (8,), dtype=C.DT_F64)), (ctypes.c_int64 * 2)(3, 5), 2, 0,
                                     arr(ys))


SHAPE = (2, 4, 6, 16)
PACKED = (6 * 96, 16, 96, 1)  # four of six heads inside the sequence axis


@pytest.mark.parametrize("xs,ys,text", [
    ([at(0, SHAPE)], [at(4, SHAPE)], "y overlaps an input"),
    ([at(0, SHAPE, PACKED)], [at(64, SHAPE, PACKED)], "y overlaps an input"),
    ([at(0, SHAPE), at(step(1), SHAPE)], [at(step(1), SHAPE), at(step(2), SHAPE)], "y overlaps an input"),
    ([at(0, SHAPE), at(step(1), SHAPE)], [at(step(2), SHAPE), at(step(2) + 256, SHAPE)], "the results overlap"),
    ([at(0, SHAPE)], [at(step(8), SHAPE)], "y and positions overlap"),
    ([at(0, SHAPE)], [at(step(9) - 64, SHAPE)], "y and freqs overlap"),
])
def test_rotary(xs, ys, text):
    refused(turn(xs, ys), text)


KEYS = (2, 2, 9, 16)


def attend(**change):
    t = dict(q=at(0, SHAPE), k=at(step(1), KEYS), v=at(step(2), KEYS), lengths=at(step(3), (2,), dtype=C.DT_I32),
             starts=at(step(4), (2,), dtype=C.DT_I64), o=at(step(5), SHAPE), lse=at(step(6), (2, 4, 6)))
    t.update(change)
    return C.lib().chelis_hip_window_attention(*(ref(t[n]) for n in ("q", "k", "v", "lengths", "starts")), 4, 1, 0.1,
                                               ref(t["o"]), ref(t["lse"]))


@pytest.mark.parametrize("change,text", [
    (dict(o=at(16, SHAPE)), "o overlaps another operand (q)"),
    (dict(o=at(step(1) + 128, SHAPE)), "o overlaps another operand (k)"),
    (dict(o=at(step(2) - 64, SHAPE)), "o overlaps another operand (v)"),
    (dict(o=at(0, SHAPE, PACKED), q=at(64, SHAPE, PACKED)), "o overlaps another operand (q)"),
    (dict(o=at(step(3), SHAPE)), "o overlaps another operand (lengths)"),
    (dict(o=at(step(4), SHAPE)), "o overlaps another operand (starts)"),
    (dict(lse=at(step(5), (2, 4, 6))), "o overlaps another operand (lse)"),
    (dict(lse=at(1024, (2, 4, 6))), "lse overlaps another operand (q)"),
    (dict(lse=at(step(4) + 8, (2, 4, 6))), "lse overlaps another operand (starts)"),
])
def test_window_attention(change, text):
    refused(attend(**change), text)


def attend_adjoint(**change):
    t = dict(q=at(0, SHAPE), k=at(step(1), KEYS), v=at(step(2), KEYS), o=at(step(3), SHAPE), lse=at(step(4), (2, 4, 6)),
             g=at(step(5), SHAPE), lengths=at(step(6), (2,), dtype=C.DT_I32), starts=at(step(7), (2,), dtype=C.DT_I32),
             dq=at(step(8), SHAPE), dk=at(step(9), KEYS), dv=at(step(10), KEYS))
    t.update(change)
    return C.lib().chelis_hip_window_attention_adjoint(
        *(ref(t[n]) for n in ("q", "k", "v", "o", "lse", "g", "lengths", "starts")), 4, 1, 0.1,
        *(ref(t[n]) for n in ("dq", "dk", "dv")))


@pytest.mark.parametrize("change,text", [
    (dict(dq=at(step(4), SHAPE)), "dq overlaps another operand (lse)"),
    (dict(dq=at(step(6), SHAPE)), "dq overlaps another operand (lengths)"),
    (dict(dk=at(step(7) - 4, KEYS)), "dk overlaps another operand (starts)"),
    (dict(dv=at(step(5) + 320, KEYS)), "dv overlaps another operand (g)"),
    (dict(dv=at(step(3), KEYS)), "dv overlaps another operand (o)"),
    (dict(dk=at(step(8) + 64, KEYS)), "dq overlaps another operand (dk)"),
    (dict(dv=at(step(9) + 64, KEYS)), "dk overlaps another operand (dv)"),
    (dict(dq=at(64, SHAPE)), "dq overlaps another operand (q)"),
])
def test_window_attention_adjoint(change, text):
    refused(attend_adjoint(**change), text)
