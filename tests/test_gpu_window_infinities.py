"""Infinities in v that rows see: the formula's sum is infinite in that column
whatever the key weighs (a weight is never 0 beside finite scores), and NaN
only where both infinities or a NaN are seen. Wherever the key stands in a
tile, and however small its weight becomes at the arithmetic's width."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import check, decode, draw, encode, visible, window_forward

pytestmark = pytest.mark.gpu

# batch, heads, kv heads, rows, keys, width, window, sinks: whole rows, rows
# split over waves, one token over few and over many splits
SHAPES = [(8, 16, 8, 200, 200, 64, 200, 0), (8, 16, 8, 200, 200, 72, 90, 3), (2, 4, 2, 40, 300, 64, 200, 0),
          (1, 4, 1, 1, 700, 128, 700, 0), (1, 2, 1, 1, 9000, 64, 9000, 0)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("gap", [0.0, 40.0, 300.0])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_a_seen_infinity_is_infinite_whatever_it_weighs(kind, gap, shape):
    """Keys 70, 90 and 130 score up to `gap` below all others: e^-40 is past
    f16's weights, e^-300 past binary32's. They hold +inf in column 3, -inf in
    column 4 (both in column 5, one NaN in column 6)."""
    B, H, KV, S, N, W, window, sinks = shape
    rng = np.random.default_rng(N + W)
    q, k, v = (draw(kind, rng, s)[0] for s in ((B, H, S, W), (B, KV, N, W), (B, KV, N, W)))
    one, low = encode(kind, np.ones(1))[0], encode(kind, np.full(1, -gap))[0]
    q[..., 0], k[..., 0] = one, encode(kind, np.zeros(1))[0]
    odd = [70, 90, 130]
    k[:, :, odd, 0] = low
    clean = v.copy()
    for at, column, value in ((70, 3, np.inf), (90, 4, -np.inf), (70, 5, np.inf), (130, 5, -np.inf), (90, 6, np.nan)):
        v[:, :, at, column] = encode(kind, np.full(1, value))[0]
    o, lse = C.window_attention(C.to_device(q), C.to_device(k), C.to_device(v), window, sinks, 1.0, lse=True)
    got, values = decode(kind, o.numpy()), [decode(kind, x) for x in (q, k, clean)]
    (want, bound), (wl, bl) = window_forward(kind, *values, window, sinks, 1.0)
    check(lse.numpy().astype(np.float64), wl, bl, "lse")
    vis = visible(S, N, N, N - S, window, sinks)
    rest = [c for c in range(W) if c not in (3, 4, 5, 6)]
    check(got[..., rest], want[..., rest], bound[..., rest], "the other columns")
    a, b, c = (vis[:, n] for n in odd)
    for column, sees, value in ((3, a, np.inf), (4, b, -np.inf), (5, a & ~c, np.inf), (5, c & ~a, -np.inf)):
        assert (got[:, :, sees, column] == value).all(), (column, value)
    assert np.isnan(got[:, :, a & c, 5]).all() and np.isnan(got[:, :, b, 6]).all()
    for column, sees in ((3, a), (4, b), (5, a | c), (6, b)):
        check(got[:, :, ~sees, column], want[:, :, ~sees, column], bound[:, :, ~sees, column], "unseen")


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(8, 16, 8, 200, 200, 64), (1, 4, 1, 1, 700, 128)])
def test_a_later_score_far_above_keeps_it(kind, shape):
    """The key that holds the infinity scores highest until the last key of
    all stands 200 above it: what was summed is scaled down to nothing then."""
    B, H, KV, S, N, W = shape
    rng = np.random.default_rng(9)
    q, k, v = (draw(kind, rng, s, 0.1)[0] for s in ((B, H, S, W), (B, KV, N, W), (B, KV, N, W)))
    q[..., 0] = encode(kind, np.ones(1))[0]
    k[:, :, :, 0] = encode(kind, np.full(1, -8.0))[0]
    k[:, :, 20, 0] = encode(kind, np.zeros(1))[0]
    k[:, :, N - 1, 0] = encode(kind, np.full(1, 200.0))[0]
    v[:, :, 20, 7] = encode(kind, np.full(1, np.inf))[0]
    o = decode(kind, C.window_attention(C.to_device(q), C.to_device(k), C.to_device(v), N, 0, 1.0).numpy())
    sees = np.arange(N - S, N) >= 20
    assert (o[:, :, sees, 7] == np.inf).all() and np.isfinite(o[:, :, ~sees, 7]).all()
    other = np.arange(W) != 7
    assert np.isfinite(o[..., other]).all()
