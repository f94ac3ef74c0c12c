"""Dense products of a few rows on both sides of every limit between the vector units
and tiles: lengths of the contraction around each, weights in whole vectors and not,
one column to more than a round of workgroups, the widest operands."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import check, decode, draw, encode
from training_reference import dense

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("k", [1, 7, 504, 511, 512, 999, 1000, 1001, 1496, 1504, 1999, 2000, 2001])
@pytest.mark.parametrize("order", ["kn", "nk"])
def test_either_side_of_the_limits(kind, rows, k, order):
    rng = np.random.default_rng(rows * 10 + k)
    for n in (1, 8, 37):
        x, xv = draw(kind, rng, (rows, k))
        w, wv = draw(kind, rng, (k, n), k ** -0.5)
        bias, bv = draw("f32", rng, n, 0.3)
        res, rv = draw(kind, rng, (rows, n))
        t = C.to_device(w) if order == "kn" else C.to_device(np.ascontiguousarray(w.T)).view((k, n), (1, k))
        y, z = C.dense(C.to_device(x), t, C.to_device(bias), "silu", C.to_device(res), z=True)
        wy, wz = dense(kind, xv, wv, bv, "silu", rv)
        check(decode(kind, y.numpy()), *wy, f"y {n}")
        check(decode(kind, z.numpy()), *wz, f"z {n}")


# small whole numbers: every sum is exact, one rounding to bf16
@pytest.mark.parametrize("rows,k,n,order", [(5, 2001, 4096, "nk"), (5, 2001, 4097, "nk"), (8, 8193, 1000, "nk"), (4, 2000, 4097, "nk"),
                                            (3, 1001, 4096, "nk"), (3, 1001, 4097, "nk"), (4, 2001, 4097, "nk"), (1, 515, 32001, "nk"),
                                            (1, 1003, 32001, "kn"), (4, 1 << 20, 3, "nk"), (9, 1 << 20, 8, "nk"),
                                            (3, 1 << 20, 5, "kn"), (2, 8, 1 << 20, "kn"), (3, 7, 1 << 20, "nk"), (40, 16, 1 << 20, "nk")])
def test_wide_operands(rows, k, n, order):
    rng = np.random.default_rng(n + k)
    x, w = rng.integers(-1, 2, (rows, k)).astype(np.float32), rng.integers(-1, 2, (k, n)).astype(np.float32)
    dx = C.to_device(encode("bf16", x))
    dw = C.to_device(encode("bf16", w)) if order == "kn" else C.to_device(np.ascontiguousarray(encode("bf16", w).T)).view((k, n), (1, k))
    got = C.dense(dx, dw)
    want = (x @ w).astype(np.float64)  # binary32 sums of at most 2^20 ones: exact
    assert np.array_equal(decode("bf16", got.numpy()), decode("bf16", encode("bf16", want)))
