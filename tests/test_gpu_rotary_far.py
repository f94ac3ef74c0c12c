"""Rotary positions whose binary64 angle is large: the angle is what
position * frequency rounds to, and its sine is exact to the width's rounding
however many turns it holds."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import check, decode, draw, rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f64", "bf16", "f16"])
@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
@pytest.mark.parametrize("scale", [1.0, 1e-3, 1e9])
def test_angles_of_any_size(kind, pairing, scale):
    rng = np.random.default_rng(7)
    W, S = 48, 61
    x, xv = draw(kind, rng, (2, 3, S, W))
    # 0 and both signs of 2^1 .. 2^62, some of the digits behind them random
    far = [0] + [s * (2**k + int(rng.integers(0, 2**max(k - 1, 1)))) for k in range(3, 62, 2) for s in (1, -1)]
    pos = np.broadcast_to(np.array(far[:S], np.int64), (2, 2, S)).copy()
    pos[1] = pos[1, :, ::-1]
    freqs = scale * 10000.0 ** (-np.arange(W // 2) / 24)
    got = C.rotary(C.to_device(x), C.to_device(pos), C.to_device(freqs), [10, 14], pairing)
    check(decode(kind, got.numpy()), *rotary(kind, xv, pos, freqs, [10, 14], pairing), "turned")
    back = C.rotary_adjoint(C.to_device(x), C.to_device(pos), C.to_device(freqs), [10, 14], pairing)
    check(decode(kind, back.numpy()), *rotary(kind, xv, pos, freqs, [10, 14], pairing, -1.0), "turned back")
