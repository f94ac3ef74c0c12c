"""Rotary positions over several axes against the plain binary64 form
(block_reference)."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import check, decode, draw, rotary

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f64", "bf16", "f16"]


def bits(a):
    return np.ascontiguousarray(a).view(np.uint8)


def frequencies(pairs):
    return 10000.0 ** (-np.arange(pairs) / pairs)


def places(rng, axes, batch, seq, dtype=np.int32, far=100000):
    return rng.integers(0, far, (axes, batch, seq)).astype(dtype)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
@pytest.mark.parametrize("batch,seq,heads,kv,sections,width", [
    (1, 1, 1, 1, [1], 2), (1, 1, 1, 1, [1], 5), (2, 3, 3, 1, [2, 3], 13), (64, 1, 16, 4, [16, 24, 24], 128),
    (2, 65, 4, 4, [8, 12, 12], 64), (1, 200, 5, 1, [36], 88), (3, 17, 2, 2, [1, 1, 1, 1, 1, 1, 1, 1], 16),
    (1, 777, 12, 3, [20, 20], 80), (5, 33, 1, 1, [7, 1], 16)])
def test_turn_and_back(kind, pairing, batch, seq, heads, kv, sections, width):
    rng = np.random.default_rng(seq * 7 + width)
    freqs = frequencies(sum(sections))
    pos = places(rng, len(sections), batch, seq)
    (q, qv), (k, kv_) = draw(kind, rng, (batch, heads, seq, width)), draw(kind, rng, (batch, kv, seq, width))
    dq, dk, dp, df = C.to_device(q), C.to_device(k), C.to_device(pos), C.to_device(freqs)
    rq, rk = C.rotary([dq, dk], dp, df, sections, pairing)
    for got, x in ((rq, qv), (rk, kv_)):
        check(decode(kind, got.numpy()), *rotary(kind, x, pos, freqs, sections, pairing), "turned")
    bq = C.rotary_adjoint(dq, dp, df, sections, pairing)
    check(decode(kind, bq.numpy()), *rotary(kind, qv, pos, freqs, sections, pairing, -1.0), "turned back")
    # one tensor at a time and in place: the same bits
    assert np.array_equal(bits(C.rotary(dk, dp, df, sections, pairing).numpy()), bits(rk.numpy()))
    C.rotary([dq, dk], dp, df, sections, pairing, out=[dq, dk])
    assert np.array_equal(bits(dq.numpy()), bits(rq.numpy())) and np.array_equal(bits(dk.numpy()), bits(rk.numpy()))
    # elements past the pairs are copied
    rest = 2 * sum(sections)
    assert np.array_equal(bits(rq.numpy()[..., rest:]), bits(q[..., rest:]))


@pytest.mark.parametrize("kind", KINDS)
def test_heads_inside_the_sequence_axis(kind):
    """Queries and keys as views of one packed [batch, seq, heads + 2 kv,
    width] tensor, turned where they lie; the values beside them stay."""
    B, S, H, KV, W, sections = 2, 19, 4, 2, 24, [5, 7]
    rng = np.random.default_rng(1)
    packed, values = draw(kind, rng, (B, S, H + 2 * KV, W))
    pos, freqs = places(rng, 2, B, S), frequencies(12)
    t = C.to_device(packed)
    row = (H + 2 * KV) * W
    q, k = t.view((B, H, S, W), (S * row, W, row, 1)), t.view((B, KV, S, W), (S * row, W, row, 1), H * W)
    C.rotary([q, k], C.to_device(pos), C.to_device(freqs), sections, "halves", out=[q, k])
    now = t.numpy()
    for part, at, n in ((q, 0, H), (k, H, KV)):
        x = values[:, :, at:at + n].transpose(0, 2, 1, 3)
        check(decode(kind, part.numpy()), *rotary(kind, x, pos, freqs, sections, "halves"))
    assert np.array_equal(bits(now[:, :, H + KV:]), bits(packed[:, :, H + KV:]))


@pytest.mark.parametrize("dtype", [np.int32, np.int64])
def test_positions_of_any_sign_stride_and_size(dtype):
    """Positions shared by the batch (stride 0), negative, and up to 2^30 (the
    angle's own rounding is then 2^30 2^-53 < 2^-22: counted beside the bound)."""
    B, H, S, W = 3, 2, 9, 16
    rng = np.random.default_rng(2)
    x, xv = draw("f32", rng, (B, H, S, W))
    one = rng.integers(-2**30, 2**30, (1, S)).astype(dtype)
    one[0, :3] = [0, -1, 2**30 - 1]
    freqs = frequencies(8)
    t = C.to_device(one)
    y = C.rotary(C.to_device(x), t.view((1, B, S), (S, 0, 1)), C.to_device(freqs), [8])
    want, bound = rotary("f32", xv, np.broadcast_to(one, (1, B, S)), freqs, [8], "halves")
    check(y.numpy().astype(np.float64), want, bound + 2 * 2.0**-22 * np.abs(xv).max())


@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
def test_the_adjoint_is_the_transpose(pairing):
    """<rotary(x), g> = <x, rotary_adjoint(g)> at binary64: both sums are of
    the same 2 n products up to 12 roundings each."""
    rng = np.random.default_rng(4)
    x, g = rng.standard_normal((2, 3, 11, 40)), rng.standard_normal((2, 3, 11, 40))
    pos, freqs = C.to_device(places(rng, 2, 2, 11)), C.to_device(frequencies(18))
    y = C.rotary(C.to_device(x), pos, freqs, [10, 8], pairing).numpy()
    b = C.rotary_adjoint(C.to_device(g), pos, freqs, [10, 8], pairing).numpy()
    assert abs((y * g).sum() - (x * b).sum()) <= 24 * 2.0**-53 * 2 * np.abs(x).max() * np.abs(g).max() * x.size


def test_no_tokens():
    pos, freqs = C.empty((1, 2, 0), np.int32), C.to_device(frequencies(4))
    assert C.rotary(C.empty((2, 3, 0, 8), np.float32), pos, freqs, [4]).shape == (2, 3, 0, 8)
