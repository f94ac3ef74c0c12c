"""Windowed attention's gradients with many always-visible keys: any count of
sequences and sinks that the forward call serves, in scratch that does not
outgrow the keys."""
import ctypes

import numpy as np
import pytest

import chelis_amd as C
from block_reference import check, decode, draw, window_adjoint

pytestmark = pytest.mark.gpu


def operands(kind, B, H, KV, S, N, W, seed):
    rng = np.random.default_rng(seed)
    return [draw(kind, rng, s, x)[0] for s, x in (((B, H, S, W), 1.0), ((B, KV, N, W), 1.0), ((B, KV, N, W), 1.0),
                                                  ((B, H, S, W), 0.01))]


def gradients(kind, arrays, window, sinks, scale, some=slice(None)):
    """Checked against binary64 over the sequences `some`."""
    t = [C.to_device(x) for x in arrays]
    o, lse = C.window_attention(*t[:3], window, sinks, scale, lse=True)
    got = [x.numpy() for x in C.window_attention_adjoint(*t[:3], o, lse, t[3], window, sinks, scale)]
    q, k, v, g = (decode(kind, np.ascontiguousarray(x[some])) for x in arrays)
    want = window_adjoint(kind, q, k, v, decode(kind, o.numpy()[some]), lse.numpy()[some].astype(np.float64), g, window,
                          sinks, scale)
    for name, a, (w, bound) in zip(("dq", "dk", "dv"), got, want):
        check(decode(kind, np.ascontiguousarray(a[some])), w, bound, name)
    return got


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_more_sequences_and_sink_blocks_than_a_grid_axis_holds(kind):
    """2100 sequences of 32 sink blocks each: 67200 in all."""
    gradients(kind, operands(kind, 2100, 1, 1, 8, 1200, 8, 1), 3, 1001, 0.3, slice(0, 2100, 419))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,KV,S,W,window,sinks", [(40, 8, 450, 16, 70, 300), (3, 2, 450, 72, 70, 449), (40, 8, 450, 16, 70, 33)])
def test_many_sinks(kind, B, KV, S, W, window, sinks):
    """Sink blocks past what fills the device, whose far rows the keys' own
    workgroups take, and below it, where they are dealt out."""
    gradients(kind, operands(kind, B, 2 * KV, KV, S, S, W, 2), window, sinks, W ** -0.5, slice(0, B, 13))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sinks", [400, 2**40])
def test_sinks_that_hold_every_key_are_a_window_that_does(kind, sinks):
    arrays = operands(kind, 2, 4, 2, 400, 400, 64, 3)
    for a, b in zip(gradients(kind, arrays, 5, sinks, 0.125), gradients(kind, arrays, 400, 0, 0.125)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("sinks", [2000, 2048])
def test_scratch_does_not_outgrow_the_keys(sinks):
    """64 key heads of 2048 bf16 keys, k 32 MB: the gradients of a call with
    nearly every key, and with every key, a sink need less device memory than
    four times that beside their operands."""
    arrays = operands("bf16", 8, 8, 8, 2048, 2048, 128, 4)
    t = [C.to_device(x) for x in arrays]
    out = [C.empty(x.shape, x.dtype) for x in t[:3]]
    o, lse = C.window_attention(*t[:3], 64, sinks, 0.09, lse=True)
    from chelis_amd import hiprt
    free, total = ctypes.c_size_t(), ctypes.c_size_t()

    def available():
        C.synchronize()
        assert hiprt.hip().hipMemGetInfo(ctypes.byref(free), ctypes.byref(total)) == 0
        return free.value

    before = available()
    C.window_attention_adjoint(*t[:3], o, lse, t[3], 64, sinks, 0.09, *out)
    assert before - available() < 4 * arrays[1].nbytes
