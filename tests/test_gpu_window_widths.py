"""Windowed attention with heads between the widths its registers hold (64, 96
and 128): the columns that fill a tile up past the width take no part, whatever
the keys, values and cotangents of visible pairs hold."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import decode, draw, encode

pytestmark = pytest.mark.gpu

# batch, heads, kv heads, rows, keys: whole rows (the last ones behind the
# window of the sinks), and one token over a cache
SHAPES = [(8, 16, 8, 200, 200), (2, 8, 2, 1, 300)]
HELD = {8: 64, 40: 64, 72: 96, 104: 128}


def results(q, k, v, g, window=60, sinks=5):
    t = [C.to_device(x) for x in (q, k, v, g)]
    o, lse = C.window_attention(*t[:3], window, sinks, 0.2, lse=True)
    return o.numpy(), lse.numpy(), [x.numpy() for x in C.window_attention_adjoint(*t[:3], o, lse, t[3], window, sinks, 0.2)]


def operands(kind, shape, W, seed):
    B, H, KV, S, N = shape
    rng = np.random.default_rng(seed)
    return [draw(kind, rng, (B, h, n, W), s)[0] for h, n, s in ((H, S, 1.0), (KV, N, 1.0), (KV, N, 1.0), (H, S, 0.01))]


@pytest.mark.parametrize("shape", SHAPES, ids=["rows", "token"])
@pytest.mark.parametrize("W", sorted(HELD))
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_a_key_of_minus_infinity_weighs_nothing(kind, W, shape):
    """Element 0 of every q is 1 and of one visible key -inf: its score is
    -inf and its weight 0, so every row stays finite; of the gradients only
    dq's column 0 (0 times that element) is NaN, at the rows that see it."""
    q, k, v, g = operands(kind, shape, W, W)
    S, N = shape[3:]
    at = N - 20
    q[..., 0] = encode(kind, np.ones(1))[0]
    k[:, :, at, 0] = encode(kind, np.full(1, -np.inf))[0]
    o, lse, (dq, dk, dv) = results(q, k, v, g)
    assert np.isfinite(decode(kind, o)).all() and np.isfinite(lse).all()
    bad = np.isnan(decode(kind, dq))
    assert not bad[..., 1:].any()
    sees = np.arange(N - S, N) >= at
    assert bad[:, :, sees, 0].all() and not bad[:, :, ~sees, 0].any()
    assert np.isfinite(decode(kind, dk)).all() and np.isfinite(decode(kind, dv)).all()


@pytest.mark.parametrize("shape", SHAPES, ids=["rows", "token"])
@pytest.mark.parametrize("W", sorted(HELD))
@pytest.mark.parametrize("which", [1, 2, 3], ids=["k", "v", "g"])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_zeros_up_to_the_held_width_change_nothing(kind, value, which, W, shape):
    """The same heads with zeros from their width up to the held one: products
    with those columns add zeros, so every bit is the same."""
    parts = operands(kind, shape, W, W + which)
    row = parts[which].shape[2] - 1 if which < 3 else 0
    parts[which][0, 0, row, 3] = encode(kind, np.full(1, value))[0]
    wide = [np.concatenate([x, np.zeros(x.shape[:3] + (HELD[W] - W,), x.dtype)], 3) for x in parts]
    (o, lse, grads), (ow, lw, wgrads) = results(*parts), results(*wide)
    assert np.array_equal(lse, lw, equal_nan=True)
    for a, b in zip([o, *grads], [ow, *wgrads]):
        assert np.array_equal(decode(kind, a), decode(kind, np.ascontiguousarray(b[..., :W])), equal_nan=True)
