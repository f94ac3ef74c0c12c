"""Dense products, the residual stream and clipping on tensors of more than 2^31
elements, on rows further apart than a tile's offsets reach, and from several threads
at once. But for the threads, inputs are small
integers, so that every product and sum is exact and most results are compared bit
for bit; the large tensors are made on the device by the product itself."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import decode, encode

pytestmark = pytest.mark.gpu
ROWS, K, N = (1 << 21) + 5, 8, 1032  # 2^31 + 1.7e7 elements


@pytest.fixture(scope="module")
def far():
    """x [ROWS, K] of -1, 0, 1 in every 64th row and the last three, w [K, N] of
    -3 .. 3 and their product, whose elements are at most 24."""
    rng = np.random.default_rng(5)
    x = np.zeros((ROWS, K))
    at = np.unique(np.concatenate([np.arange(0, ROWS, 64), np.arange(ROWS - 3, ROWS)]))
    x[at] = rng.integers(-1, 2, (len(at), K))
    w = rng.integers(-3, 4, (K, N)).astype(float)
    dx, dw = C.to_device(encode("bf16", x)), C.to_device(encode("bf16", w))
    return at, x, w, dx, dw, C.dense(dx, dw)


def row_of(t, i, width):
    return decode("bf16", t.view((width,), (1,), i * width).numpy())


CHECKED = (0, 64, ROWS // 2 // 64 * 64, ROWS - 4, ROWS - 3, ROWS - 2, ROWS - 1)


def test_product_and_gradients(far):
    at, x, w, dx, dw, y = far
    assert ROWS * N > 1 << 31
    for i in CHECKED:
        assert np.array_equal(row_of(y, i, N), x[i] @ w), i
    # sums of at most 32772 rows times 24, and 1032 columns times 72: whole numbers under 2^24
    gx, gw, gb = C.dense_adjoint(dx, dw, y, dw=C.empty((K, N), np.float32), dbias=C.empty((N,), np.float32))
    g = x[at] @ w
    assert np.array_equal(gw.numpy(), x[at].T @ g)
    assert np.array_equal(gb.numpy(), g.sum(0))
    for i in CHECKED:
        assert np.array_equal(row_of(gx, i, K), decode("bf16", encode("bf16", (x[i] @ w) @ w.T))), i


def test_rows_far_apart():
    """A result and an operand whose rows lie 2^21 + 8 elements apart, 2^31 in all."""
    rng = np.random.default_rng(6)
    rows, step = 1027, (1 << 21) + 8
    x, w, v = (rng.integers(-1, 2, s).astype(float) for s in ((rows, K), (K, 40), (40, 24)))
    room = C.empty((rows * step,), C.dense(*(C.to_device(encode("bf16", t)) for t in (x, w))).dtype)
    wide = room.view((rows, 40), (step, 1), 0)
    C.dense(C.to_device(encode("bf16", x)), C.to_device(encode("bf16", w)), y=wide)
    got = C.dense(wide, C.to_device(encode("bf16", v)))
    assert np.array_equal(decode("bf16", got.numpy()), decode("bf16", encode("bf16", (x @ w) @ v)))
    dx, dv, _ = C.dense_adjoint(wide, C.to_device(encode("bf16", v)), got, dw=C.empty((40, 24), np.float32))
    g = decode("bf16", got.numpy())
    assert np.array_equal(dv.numpy(), (x @ w).T @ g)
    assert np.array_equal(decode("bf16", dx.numpy()), decode("bf16", encode("bf16", g @ v.T)))


def test_residual_stream(far):
    """u = x + 0.5 x is exact; h and dx: binary32 sums of 1032 terms of at most 48,
    then one rounding to bf16."""
    at, x, w, _, _, y = far
    norm = C.Norm("rms")
    u, h = C.residual_norm(y, y, None, None, 0.5, norm)
    dx, *_ = C.residual_norm_adjoint(u, pre=norm, du=y, dh=y)
    for i in CHECKED:
        row = x[i] @ w
        assert np.array_equal(row_of(u, i, N), 1.5 * row), i
        rstd = 1 / np.sqrt((2.25 * row * row).mean() + 1e-5)
        unit = 1.5 * row * rstd
        assert (np.abs(row_of(h, i, N) - unit) <= (2.0**-8 + 2.0**-18) * np.abs(unit)).all(), i
        want = row + rstd * (row - unit * (row * unit).mean())
        assert (np.abs(row_of(dx, i, N) - want) <= 2.0**-8 * np.abs(want) + 2.0**-13).all(), i


def test_clipping(far):
    """One gradient of more elements than a part holds; its norm is exact but for the
    last roundings. The factor 2^-3 keeps every element."""
    at, x, w, _, _, y = far
    g = x[at] @ w
    want = np.sqrt((g * g).sum())
    norm = C.gradient_norm([y], 1.0, C.empty((), np.float64))
    assert abs(float(norm.numpy()) - want) <= 2.0**-50 * want
    (out,) = C.clip_gradients([y], C.to_device(np.full((), 8.0, np.float64)), 1.0, 1.0, [C.empty(y.shape, y.dtype)])
    for i in CHECKED:
        assert np.array_equal(row_of(out, i, N), 0.125 * (x[i] @ w)), i


def test_threads_at_once():
    """Calls of every operator from four threads: each gives what it gives alone."""
    import threading

    rng = np.random.default_rng(7)
    made = lambda *s: C.to_device(encode("bf16", rng.standard_normal(s)))
    sets = [(made(300 + i, 520), made(520, 264), made(264), made(300 + i, 264)) for i in range(4)]

    def step(x, w, bias, g):
        y, z = C.dense(x, w, bias, "gelu", z=True)
        norm = C.Norm("layer")
        u, h = C.residual_norm(y, g, None, bias, 0.5, norm)
        du, db, dgate, _, _ = C.residual_norm_adjoint(u, g, None, bias, 0.5, norm, du=g, dh=h)
        dx, dw, dbias = C.dense_adjoint(x, w, du, z, "gelu")
        grads = [dw, dbias, dgate]
        held = C.gradient_norm(grads)
        C.clip_gradients(grads, held, 0.5)
        return [t.numpy() for t in (y, h, db, dx, held, *grads)]

    alone = [step(*s) for s in sets]
    wrong = []

    def work(i):
        for _ in range(20):
            if not all(np.array_equal(a, b) for a, b in zip(step(*sets[i]), alone[i])):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
