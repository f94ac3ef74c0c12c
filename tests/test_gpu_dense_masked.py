"""Gradients of a dense product behind relu where the masked places of the cotangent
hold infinities and NaN: nothing of them arrives, as in relu_adjoint."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import NP, check, decode, draw, encode
from training_reference import dense_adjoint

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows,k,n", [(1, 8, 24), (5, 16, 9), (130, 70, 129), (300, 256, 512)])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_relu_selects(kind, rows, k, n, value):
    rng = np.random.default_rng(rows + n)
    x, xv = draw(kind, rng, (rows, k))
    w, wv = draw(kind, rng, (k, n), k ** -0.5)
    z, zv = draw(kind, rng, (rows, n), 1.5)
    zv[0, 0] = 0.0
    zv[rows // 2, n // 2] = -0.0
    zv[-1, -1] = -np.inf
    z = encode(kind, zv)
    g, gv = draw(kind, rng, (rows, n), 0.1)
    masked = ~(zv > 0)
    put = encode(kind, np.where(masked, value, gv))
    d = [C.to_device(t) for t in (x, w, put, z)]
    got = C.dense_adjoint(*d, "relu", dw=C.empty((k, n), np.float32), dbias=C.empty((n,), np.float32))
    # (the plain form multiplies its bound by z: -1 there stands for the infinity, whose slope is the same 0)
    want = dense_adjoint(kind, "f32", xv, wv, np.maximum(zv, -1.0), "relu", np.where(masked, 0.0, gv))
    for name, t, held, w_ in zip(("dx", "dw", "dbias"), got, (kind, "f32", "f32"), want):
        check(decode(held, t.numpy()), *w_, name)
    # the same step in two calls: the cotangent masked by relu_adjoint, then the product's gradients
    dz = C.relu_adjoint(d[3], d[2])
    apart = C.dense_adjoint(d[0], d[1], dz, dw=C.empty((k, n), np.float32), dbias=C.empty((n,), np.float32))
    for a, b in zip(got, apart):
        assert np.array_equal(a.numpy(), b.numpy())


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_what_passes_arrives(kind):
    """Where z > 0 an infinity or a NaN of g goes on, and a NaN z makes a NaN."""
    rows, k, n = 6, 16, 24
    x, w = (C.to_device(encode(kind, np.ones(s))) for s in ((rows, k), (k, n)))
    z, g = np.ones((rows, n)), np.ones((rows, n))
    g[1, 2], g[2, 3], z[4, 5] = np.inf, np.nan, np.nan
    dx, dw, db = (decode(kind, t.numpy()) for t in C.dense_adjoint(x, w, C.to_device(encode(kind, g)), C.to_device(encode(kind, z)), "relu"))
    assert (dx[[0, 3, 5]] == n).all() and (dx[1] == np.inf).all() and np.isnan(dx[[2, 4]]).all()
    cols = [j for j in range(n) if j not in (2, 3, 5)]
    assert (db[cols] == rows).all() and (dw[:, cols] == rows).all()
    assert db[2] == np.inf and (dw[:, 2] == np.inf).all() and np.isnan(db[[3, 5]]).all() and np.isnan(dw[:, [3, 5]]).all()
