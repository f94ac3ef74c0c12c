"""Layer norm with statistics and its gradients against the plain binary64
form (block_reference): lengths from one element to rows past the register
capacity, every dtype, strides, aliasing, special values, graph replays."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import NP, Captured, check, decode, draw, encode, norm, norm_adjoint

pytestmark = pytest.mark.gpu
EPS = 1e-5
TYPES = [("f32", "f32"), ("f64", "f64"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")]
SHAPES = [(1, 1), (3, 7), (5, 8), (4, 33), (130, 128), (37, 129), (70, 500), (65, 512), (9, 1000), (1030, 1024),
          (3, 2049), (2, 4104), (5, 8200), (2, 16384), (3, 16389)]


def stat_kind(kind):
    return "f64" if kind == "f64" else "f32"


def bits(a):
    return np.ascontiguousarray(a).view(np.uint8)


def operands(kind, weights, rows, n, seed):
    rng = np.random.default_rng(seed)
    return (draw(kind, rng, (rows, n), 1.5, 0.25), draw(weights, rng, n, 0.1, 1.0), draw(weights, rng, n, 0.1),
            draw(kind, rng, (rows, n), 0.01))


@pytest.mark.parametrize("rows,n", SHAPES)
@pytest.mark.parametrize("kind,weights", TYPES)
def test_forward_and_gradients(kind, weights, rows, n):
    (x, xv), (gm, gv), (bt, bv), (g, gr) = operands(kind, weights, rows, n, rows * 31 + n)
    dx_, dgm, dbt, dg_ = (C.to_device(a) for a in (x, gm, bt, g))
    y, mean, rstd = C.layer_norm_stats(dx_, dgm, dbt, EPS)
    wy, wm, wr = norm(kind, xv, gv, bv, EPS)
    check(decode(kind, y.numpy()), *wy, "y")
    check(mean.numpy().astype(np.float64), *wm, "mean")
    check(rstd.numpy().astype(np.float64), *wr, "rstd")
    if kind in ("f32", "f64"):
        assert np.array_equal(bits(y.numpy()), bits(C.layer_norm(dx_, dgm, dbt, EPS).numpy()))
    m, r = mean.numpy().astype(np.float64), rstd.numpy().astype(np.float64)
    dx, dgamma, dbeta = C.layer_norm_adjoint(dx_, dgm, mean, rstd, dg_)
    wx, wg, wb = norm_adjoint(kind, weights, xv, gv, m, r, gr)
    check(decode(kind, dx.numpy()), *wx, "dx")
    check(decode(weights, dgamma.numpy()), *wg, "dgamma")
    check(decode(weights, dbeta.numpy()), *wb, "dbeta")
    # each part alone, and again: the same bits
    only, none, none2 = C.layer_norm_adjoint(dx_, dgm, mean, rstd, dg_, want_weights=False)
    assert none is None and none2 is None and np.array_equal(bits(only.numpy()), bits(dx.numpy()))
    none, g2, b2 = C.layer_norm_adjoint(dx_, dgm, mean, rstd, dg_, want_dx=False)
    assert none is None
    assert np.array_equal(bits(g2.numpy()), bits(dgamma.numpy())) and np.array_equal(bits(b2.numpy()), bits(dbeta.numpy()))
    # the gradient over x itself, then over g
    over = C.to_device(x)
    C.layer_norm_adjoint(over, dgm, mean, rstd, dg_, dx=over)
    assert np.array_equal(bits(over.numpy()), bits(dx.numpy()))
    C.layer_norm_adjoint(dx_, dgm, mean, rstd, dg_, dx=dg_)
    assert np.array_equal(bits(dg_.numpy()), bits(dx.numpy()))
    C.layer_norm_stats(dx_, dgm, dbt, EPS, y=dx_)
    assert np.array_equal(bits(dx_.numpy()), bits(y.numpy()))


@pytest.mark.parametrize("kind,weights,n", [("f32", "f32", 70000), ("bf16", "f32", 40001), ("f64", "f64", 33000),
                                            ("f16", "f16", 16386)])
def test_rows_past_the_register_capacity(kind, weights, n):
    test_forward_and_gradients(kind, weights, 70, n) if n < 20000 else test_forward_and_gradients(kind, weights, 3, n)


@pytest.mark.parametrize("kind,weights", TYPES)
def test_strided_rows_keep_what_lies_between(kind, weights):
    """Rows of 203 elements 260 apart, from an element off every alignment;
    leading axes that collapse; the gaps of the results stay."""
    rows, n, ld, off = 6, 203, 260, 3
    (x, xv), (gm, gv), (bt, bv), (g, gr) = operands(kind, weights, rows, n, 5)
    rng = np.random.default_rng(9)

    def strided(a):
        back = draw(kind, rng, rows * ld + off)[0]
        whole = back[off:].reshape(rows, ld)
        whole[:, :n] = a
        t = C.to_device(back)
        return t, back, t.view((2, 3, n), (3 * ld, ld, 1), off)

    tx, _, vx = strided(x)
    tg, _, vg = strided(g)
    ty, by, vy = strided(x)
    td, bd, vd = strided(x)
    dgm, dbt = C.to_device(gm), C.to_device(bt)
    _, mean, rstd = C.layer_norm_stats(vx, dgm, dbt, EPS, y=vy)
    wy, wm, _ = norm(kind, xv, gv, bv, EPS)
    check(decode(kind, vy.numpy()).reshape(rows, n), *wy, "y")
    check(mean.numpy().astype(np.float64).reshape(-1), *wm, "mean")
    _, dgamma, dbeta = C.layer_norm_adjoint(vx, dgm, mean, rstd, vg, dx=vd)
    m, r = (t.numpy().astype(np.float64).reshape(-1) for t in (mean, rstd))
    wx, wg, wb = norm_adjoint(kind, weights, xv, gv, m, r, gr)
    check(decode(kind, vd.numpy()).reshape(rows, n), *wx, "dx")
    check(decode(weights, dgamma.numpy()), *wg, "dgamma")
    check(decode(weights, dbeta.numpy()), *wb, "dbeta")
    for t, back in ((ty, by), (td, bd)):
        now = t.numpy()
        assert np.array_equal(bits(now[:off]), bits(back[:off]))
        assert np.array_equal(bits(now[off:].reshape(rows, ld)[:, n:]), bits(back[off:].reshape(rows, ld)[:, n:]))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [100, 1000, 17000])
def test_special_rows_stay_in_their_rows(kind, n):
    """A NaN or an infinity in one row, a constant row, a row far from zero."""
    (x, xv), (gm, gv), (bt, bv), (g, gr) = operands(kind, kind, 8, n, n)
    for row, value in ((2, np.nan), (4, np.inf), (6, 3.0)):
        v = xv.copy()
        v[row, n // 2] = value
        if row == 6:
            v[6] = 3.0
        xs = encode(kind, v)
        y, mean, rstd = C.layer_norm_stats(C.to_device(xs), C.to_device(gm), C.to_device(bt), EPS)
        got = decode(kind, y.numpy())
        keep = [i for i in range(8) if i != row]
        wy, _, _ = norm(kind, decode(kind, xs)[keep], gv, bv, EPS)
        check(got[keep], *wy, f"other rows of {value}")
        if row == 6:
            wy, _, _ = norm(kind, decode(kind, xs)[[6]], gv, bv, EPS)
            check(got[[6]], *wy, "constant row")
        else:
            assert np.isnan(got[row]).all()
        dx, _, _ = C.layer_norm_adjoint(C.to_device(xs), C.to_device(gm), mean, rstd, C.to_device(g))
        m, r = mean.numpy().astype(np.float64), rstd.numpy().astype(np.float64)
        wx, _, _ = norm_adjoint(kind, kind, decode(kind, xs)[keep], gv, m[keep], r[keep], gr[keep])
        check(decode(kind, dx.numpy())[keep], *wx, f"gradient beside {value}")
        if row != 6:
            assert np.isnan(decode(kind, dx.numpy())[row]).all()


@pytest.mark.parametrize("kind,quiet", [("f32", 0x7FC00000), ("bf16", 0x7FC0), ("f16", 0x7E00)])
def test_nan_is_the_canonical_one(kind, quiet):
    x = encode(kind, np.full((2, 64), np.nan))
    one = C.to_device(encode(kind, np.ones(64)))
    y, mean, rstd = C.layer_norm_stats(C.to_device(x), one, one, EPS)
    word = np.uint32 if kind == "f32" else np.uint16
    assert (y.numpy().view(word) == quiet).all()
    assert (mean.numpy().view(np.uint32) == 0x7FC00000).all() and (rstd.numpy().view(np.uint32) == 0x7FC00000).all()
    dx, dg, db = C.layer_norm_adjoint(C.to_device(x), one, mean, rstd, C.to_device(x))
    for t in (dx, dg, db):
        assert (t.numpy().view(word) == quiet).all()


@pytest.mark.parametrize("kind", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("n", [24, 20000])
def test_no_rows_give_zero_weight_gradients(kind, n):
    x = C.empty((0, n), NP[kind])
    w = C.to_device(np.ones(n, NP[kind]))
    stat = C.empty((0,), np.float64 if kind == "f64" else np.float32)
    dg, db = C.to_device(np.ones(n, NP[kind])), C.to_device(np.ones(n, NP[kind]))
    C.layer_norm_stats(x, w, w, EPS)
    C.layer_norm_adjoint(x, w, stat, stat, x, dgamma=dg, dbeta=db)
    assert not dg.numpy().any() and not db.numpy().any()


def test_gradients_against_differences():
    """Central differences of the binary64 forward: for h = 1e-5 their own
    error is below 1e-8 of the gradient's scale at these sizes."""
    rng = np.random.default_rng(3)
    x, gamma, beta, g = rng.standard_normal((4, 37)), rng.standard_normal(37), rng.standard_normal(37), \
        rng.standard_normal((4, 37))
    dev = {k: C.to_device(v) for k, v in dict(x=x, gamma=gamma, beta=beta, g=g).items()}
    _, mean, rstd = C.layer_norm_stats(dev["x"], dev["gamma"], dev["beta"], EPS)
    dx, dgamma, dbeta = C.layer_norm_adjoint(dev["x"], dev["gamma"], mean, rstd, dev["g"])

    def loss(xx, gg, bb):
        return (C.layer_norm(C.to_device(xx), C.to_device(gg), C.to_device(bb), EPS).numpy() * g).sum()

    h = 1e-5
    for grad, which in ((dx, 0), (dgamma, 1), (dbeta, 2)):
        way = rng.standard_normal(grad.shape)
        plus, minus = [x, gamma, beta], [x, gamma, beta]
        plus[which], minus[which] = plus[which] + h * way, minus[which] - h * way
        want = (loss(*plus) - loss(*minus)) / (2 * h)
        assert abs((grad.numpy() * way).sum() - want) < 1e-6 * np.abs(grad.numpy() * way).sum()


@pytest.mark.parametrize("kind,weights,rows,n", [("f32", "f32", 300, 500), ("bf16", "f32", 40, 3000),
                                                 ("bf16", "bf16", 100, 17000)])
def test_captured_gradients_replay(kind, weights, rows, n):
    """Two captured calls replayed in turn, with eager calls of the same sizes
    (which take cached scratch) between them."""
    calls = []
    for seed in (1, 2):
        (x, _), (gm, _), (bt, _), (g, _) = operands(kind, weights, rows, n, seed)
        t = [C.to_device(a) for a in (x, gm, bt, g)]
        _, mean, rstd = C.layer_norm_stats(t[0], t[1], t[2], EPS)
        want = [bits(o.numpy()) for o in C.layer_norm_adjoint(t[0], t[1], mean, rstd, t[3])]
        out = [C.empty((rows, n), t[0].dtype), C.empty((n,), t[1].dtype), C.empty((n,), t[1].dtype)]
        C.synchronize()
        graph = Captured(lambda: C.layer_norm_adjoint(t[0], t[1], mean, rstd, t[3], *out))
        calls.append((t, mean, rstd, want, out, graph))
    for _ in range(3):
        for t, mean, rstd, want, out, graph in calls:
            graph.launch()
        for t, mean, rstd, want, out, graph in calls:
            eager = C.layer_norm_adjoint(t[0], t[1], mean, rstd, t[3])
            C.synchronize()
            for o, e, w in zip(out, eager, want):
                assert np.array_equal(bits(o.numpy()), w) and np.array_equal(bits(e.numpy()), w)


def test_a_call_captured_before_any_other():
    """The scratch of a size no call asked for before is allocated while the
    stream is being captured, and stays with the graph: eager calls of that
    size between the replays take other storage."""
    rows, n = 1111, 11111
    (x, _), (gm, _), (_, _), (g, _) = operands("f32", "f32", rows, n, 3)
    t = [C.to_device(a) for a in (x, gm, g)]
    mean, rstd = C.to_device(x.mean(1)), C.to_device(1 / x.std(1))
    out = [C.empty((rows, n), np.float32), C.empty((n,), np.float32), C.empty((n,), np.float32)]
    C.synchronize()
    graph = Captured(lambda: C.layer_norm_adjoint(t[0], t[1], mean, rstd, t[2], *out))
    want = [bits(o.numpy()) for o in C.layer_norm_adjoint(t[0], t[1], mean, rstd, t[2])]
    other = C.to_device(2 * g)
    for _ in range(3):
        graph.launch()
        C.layer_norm_adjoint(t[0], t[1], mean, rstd, other)
        C.synchronize()
        for o, w in zip(out, want):
            assert np.array_equal(bits(o.numpy()), w)
