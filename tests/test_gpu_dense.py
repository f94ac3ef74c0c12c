"""The 16-bit product with its epilogue and its gradients against binary64: every
activation, both orders of the weights, sizes off every tile and vector, from one
row to launches of the largest tiles and of K slices, strides, aliasing, special
values, graph replays."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import NP, Captured, check, decode, draw, encode
from training_reference import act, dense, dense_adjoint

pytestmark = pytest.mark.gpu
ACTS = [None, "relu", "gelu", "silu"]
# (rows, k, n)
SIZES = [(1, 1, 1), (1, 8, 8), (2, 3, 5), (5, 16, 9), (1, 300, 264), (17, 33, 65), (32, 256, 32), (33, 257, 40), (64, 64, 64),
         (130, 70, 129), (250, 1000, 77), (257, 520, 264), (1000, 65, 33), (300, 129, 1001)]


def bits(a):
    return np.ascontiguousarray(a).view(np.uint8)


class Case:
    def __init__(self, kind, rows, k, n, order, seed, bias=None, lead=()):
        rng = np.random.default_rng(seed)
        self.kind, self.rows, self.k, self.n, self.order = kind, rows, k, n, order
        self.bias_kind = bias or kind
        self.x, self.xv = draw(kind, rng, (rows, k))
        w, wv = draw(kind, rng, (k, n), k ** -0.5)
        self.wv = wv
        self.w = w if order == "kn" else np.ascontiguousarray(w.T)
        self.bias, self.bv = draw(self.bias_kind, rng, n, 0.3)
        self.res, self.rv = draw(kind, rng, (rows, n), 1.5)
        self.g, self.gv = draw(kind, rng, (rows, n), 0.1)
        self.z, self.zv = draw(kind, rng, (rows, n), 1.5)
        self.dev = {name: C.to_device(getattr(self, name)) for name in ("x", "bias", "res", "g", "z")}
        self.dev["w"] = self.matrix(C.to_device(self.w))

    def matrix(self, t):
        return t if self.order == "kn" else t.view((self.k, self.n), (1, self.k))

    def forward(self, name, bias=True, residual=True, z=True, **to):
        d = self.dev
        return C.dense(d["x"], d["w"], d["bias"] if bias else None, name, d["res"] if residual else None, z=z, **to)

    def want(self, name, bias=True, residual=True):
        return dense(self.kind, self.xv, self.wv, self.bv if bias else None, name, self.rv if residual else None)


def check_case(c, name, grads="same"):
    y, z = c.forward(name)
    wy, wz = c.want(name)
    check(decode(c.kind, y.numpy()), *wy, "y")
    check(decode(c.kind, z.numpy()), *wz, "z")
    out_kind = c.kind if grads == "same" else "f32"
    dw = c.matrix(C.empty(c.w.shape, NP[out_kind]))
    got = C.dense_adjoint(c.dev["x"], c.dev["w"], c.dev["g"], c.dev["z"] if name else None, name, dw=dw,
                          dbias=C.empty((c.n,), NP[out_kind]))
    want = dense_adjoint(c.kind, out_kind, c.xv, c.wv, c.zv if name else None, name, c.gv)
    for what, t, kind, w in zip(("dx", "dw", "dbias"), got, (c.kind, out_kind, out_kind), want):
        check(decode(kind, t.numpy()), *w, what)
    return y, z, got


@pytest.mark.parametrize("rows,k,n", SIZES)
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("order", ["kn", "nk"])
def test_forward_and_gradients(kind, order, rows, k, n):
    for i, name in enumerate(ACTS):
        c = Case(kind, rows, k, n, order, rows * 7 + k + n + i, "f32" if i % 2 else None)
        y, z, got = check_case(c, name, "f32" if i % 2 else "same")
        # without z, bias or residual; some gradients alone, and again: the same bits
        assert np.array_equal(bits(c.forward(name, z=False).numpy()), bits(y.numpy()))
        for bias, residual in ((False, True), (True, False), (False, False)):
            wy, _ = c.want(name, bias, residual)
            check(decode(kind, c.forward(name, bias, residual, z=False).numpy()), *wy, f"y {bias} {residual}")
        for j in range(3):
            ask = {f"want_{part}": j == m for m, part in enumerate(("dx", "dw", "dbias"))}
            given = [None, c.matrix(C.empty(c.w.shape, got[1].dtype)), C.empty((n,), got[2].dtype)]
            alone = C.dense_adjoint(c.dev["x"], c.dev["w"], c.dev["g"], c.dev["z"] if name else None, name, *given, **ask)
            assert [a is not None for a in alone] == [j == m for m in range(3)]
            assert np.array_equal(bits(alone[j].numpy()), bits(got[j].numpy()))


# sizes whose products run in the largest tiles, in several K slices and in the shapes
# between
@pytest.mark.parametrize("kind,rows,k,n,order", [("bf16", 4096, 72, 4096, "nk"), ("f16", 2050, 264, 4104, "kn"),
                                                 ("bf16", 33, 8200, 64, "kn"), ("f16", 8200, 40, 96, "nk"),
                                                 ("bf16", 2000, 520, 1003, "kn"), ("bf16", 12000, 64, 200, "kn")])
def test_large_products(kind, rows, k, n, order):
    check_case(Case(kind, rows, k, n, order, k), "gelu" if order == "kn" else None)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows,k,n", [(1, 1024, 520), (1, 4100, 33), (2, 2048, 40), (3, 1031, 8), (4, 4096, 72), (5, 1025, 37),
                                      (7, 4099, 5), (8, 2500, 1001)])
def test_a_few_rows(kind, rows, k, n):
    for order in ("kn", "nk"):
        c = Case(kind, rows, k, n, order, k + rows)
        for name in ("gelu", None):
            y, z = c.forward(name)
            wy, wz = c.want(name)
            check(decode(kind, y.numpy()), *wy, "y")
            check(decode(kind, z.numpy()), *wz, "z")


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_no_contraction_and_no_rows(kind):
    c = Case(kind, 5, 4, 9, "kn", 1)
    x, w = C.empty((5, 0), NP[kind]), C.empty((0, 9), NP[kind])
    y, z = C.dense(x, w, c.dev["bias"], "gelu", c.dev["res"], z=True)
    wy, wz = dense(kind, np.zeros((5, 0)), np.zeros((0, 9)), c.bv, "gelu", c.rv)
    check(decode(kind, y.numpy()), *wy, "y")
    check(decode(kind, z.numpy()), *wz, "z")
    dx, dw, db = C.dense_adjoint(x, w, c.dev["g"], c.dev["z"], "silu")
    check(decode(kind, db.numpy()), *dense_adjoint(kind, kind, np.zeros((5, 0)), np.zeros((0, 9)), c.zv, "silu", c.gv)[2], "dbias")
    assert dx.shape == (5, 0) and dw.shape == (0, 9)
    none = C.empty((0, 9), NP[kind])
    assert C.dense(C.empty((0, 4), NP[kind]), c.dev["w"], None, "relu").shape == (0, 9)
    ones = lambda *s: C.to_device(encode(kind, np.ones(s)))
    dx, dw, db = C.dense_adjoint(C.empty((0, 4), NP[kind]), c.dev["w"], none, none, "relu", dw=ones(4, 9), dbias=ones(9))
    assert dx.shape == (0, 4) and not dw.numpy().any() and not db.numpy().any()
    assert C.dense(c.dev["x"], C.empty((4, 0), NP[kind])).shape == (5, 0)
    dx, _, _ = C.dense_adjoint(c.dev["x"], C.empty((4, 0), NP[kind]), C.empty((5, 0), NP[kind]), dx=ones(5, 4))
    assert not dx.numpy().any()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("k,n,ld,off", [(64, 72, 96, 8), (64, 72, 91, 0), (61, 70, 96, 3)])
def test_strided_operands_keep_what_lies_between(kind, k, n, ld, off):
    """Rows ld apart from an element off on, three leading axes; the results'
    gaps stay, those of the operands hold NaN."""
    a, b = 6, 7
    c = Case(kind, a * b, k, n, "kn", 3)
    nan = encode(kind, np.full(a * b * ld + off, np.nan))

    def strided(values, width):
        back = nan.copy()
        back[off:].reshape(a * b, ld)[:, :width] = values
        t = C.to_device(back)
        return t, t.view((a, b, width), (b * ld, ld, 1), off)

    d = {m: strided(getattr(c, m), k if m == "x" else n) for m in ("x", "res", "g", "z")}
    wide = encode(kind, np.full((k, ld), np.nan))
    wide[:, :n] = c.w
    w = C.to_device(wide).view((k, n), (ld, 1))
    to = {m: strided(nan[:a * b * (k if m == "dx" else n)].reshape(a * b, -1), k if m == "dx" else n) for m in ("y", "z2", "dx")}
    dw = C.to_device(encode(kind, np.full((k, ld), np.nan)))
    C.dense(d["x"][1], w, c.dev["bias"], "gelu", d["res"][1], to["y"][1], to["z2"][1])
    wy, wz = c.want("gelu")
    check(decode(kind, to["y"][1].numpy()).reshape(a * b, n), *wy, "y")
    check(decode(kind, to["z2"][1].numpy()).reshape(a * b, n), *wz, "z")
    C.dense_adjoint(d["x"][1], w, d["g"][1], d["z"][1], "gelu", to["dx"][1], dw.view((k, n), (ld, 1)))
    want = dense_adjoint(kind, kind, c.xv, c.wv, c.zv, "gelu", c.gv)
    check(decode(kind, to["dx"][1].numpy()).reshape(a * b, k), *want[0], "dx")
    check(decode(kind, dw.numpy())[:, :n], *want[1], "dw")
    for m, width in (("y", n), ("z2", n), ("dx", k)):
        now = to[m][0].numpy()
        gap = lambda v: bits(v[off:].reshape(a * b, ld)[:, width:])
        assert np.array_equal(gap(now), gap(nan)) and np.array_equal(bits(now[:off]), bits(nan[:off]))
    assert np.isnan(decode(kind, dw.numpy())[:, n:]).all()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows,k,n", [(3, 40, 24), (70, 33, 129), (600, 256, 512)])
def test_result_over_the_residual(kind, rows, k, n):
    c = Case(kind, rows, k, n, "nk", 5)
    y = c.forward("silu", z=False)
    over = C.dense(c.dev["x"], c.dev["w"], c.dev["bias"], "silu", c.dev["res"], c.dev["res"])
    assert np.array_equal(bits(over.numpy()), bits(y.numpy()))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("k", [40, 41])
def test_special_values_stay_in_their_rows_and_columns(kind, k):
    rows, n = 70, 67
    c = Case(kind, rows, k, n, "kn", 6)
    plain = decode(kind, c.forward("gelu", z=False).numpy())
    x = c.xv.copy()
    x[11, k - 1], x[12, 0] = np.nan, np.inf
    c.dev["x"] = C.to_device(encode(kind, x))
    got = decode(kind, c.forward("gelu", z=False).numpy())
    keep = [i for i in range(rows) if i not in (11, 12)]
    assert np.array_equal(got[keep], plain[keep])
    assert np.isnan(got[11]).all()
    # the infinite row: +inf stays, gelu(-inf) is 0 beside the residual
    with np.errstate(invalid="ignore"):
        sign = np.sign(c.wv[0])
    assert (got[12][sign > 0] == np.inf).all() and np.array_equal(got[12][sign < 0], c.rv[12][sign < 0])
    g = c.gv.copy()
    g[3, 5] = np.nan
    dx, dw, db = C.dense_adjoint(C.to_device(c.x), c.dev["w"], C.to_device(encode(kind, g)), c.dev["z"], "silu")
    rx, rw, rb = C.dense_adjoint(C.to_device(c.x), c.dev["w"], c.dev["g"], c.dev["z"], "silu")
    rest = [i for i in range(rows) if i != 3]
    cols = [j for j in range(n) if j != 5]
    assert np.array_equal(bits(dx.numpy()[rest]), bits(rx.numpy()[rest])) and np.isnan(decode(kind, dx.numpy())[3]).all()
    assert np.array_equal(bits(dw.numpy()[:, cols]), bits(rw.numpy()[:, cols])) and np.isnan(decode(kind, dw.numpy())[:, 5]).all()
    assert np.array_equal(bits(db.numpy()[cols]), bits(rb.numpy()[cols])) and np.isnan(decode(kind, db.numpy())[5])


@pytest.mark.parametrize("kind,quiet", [("bf16", 0x7FC0), ("f16", 0x7E00)])
def test_nan_is_the_canonical_one(kind, quiet):
    x = C.to_device(encode(kind, np.full((4, 16), np.nan)))
    w = C.to_device(encode(kind, np.ones((16, 24))))
    for name in ACTS:
        y, z = C.dense(x, w, act=name, z=True)
        assert (y.numpy().view(np.uint16) == quiet).all() and (z.numpy().view(np.uint16) == quiet).all()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("name", ["gelu", "silu", "relu"])
def test_activations_and_slopes_over_their_range(kind, name):
    """Through the identity: z = x exactly, y = act(x), and dw = dz; the slope
    also against differences of the plain activation (h = 1e-4: off by h^2)."""
    n = 512
    v = np.concatenate([np.linspace(-14, 14, 8 * n - 24), [0.0, -0.0, np.inf, -np.inf, 1e4, -1e4, 65504.0, -65504.0],
                        2.0 ** -np.arange(0, 16)])
    x = encode(kind, v.reshape(8, n))
    xv = decode(kind, x)
    eye = C.to_device(encode(kind, np.eye(n)))
    finite = np.isfinite(xv)
    rows = np.where(finite, xv, 0.0)
    got, _ = C.dense(C.to_device(encode(kind, rows)), eye, act=name, z=True)
    y, ey = act(name, rows)
    check(decode(kind, got.numpy()), y, ey + 2.0**-8 * np.abs(y) if kind == "bf16" else ey + 2.0**-11 * np.abs(y) + 2.0**-25, name)
    ident = C.to_device(encode(kind, np.eye(8)))
    g = C.to_device(encode(kind, np.ones((8, n))))
    _, dw, _ = C.dense_adjoint(ident, C.to_device(encode(kind, np.zeros((8, n)))), g, C.to_device(x), name)
    slopes = decode(kind, dw.numpy())
    h, u = 1e-4, 2.0**-8 if kind == "bf16" else 2.0**-11
    with np.errstate(invalid="ignore"):
        want = (act(name, xv + h)[0] - act(name, xv - h)[0]) / (2 * h)
    smooth = finite & (np.abs(xv) < 20) & ((np.abs(xv) > 2 * h) | (name != "relu"))
    bound = u * np.abs(want) + 2.0**-16 + h * h
    assert (np.abs(slopes - want) <= bound)[smooth].all()
    assert (slopes[xv > 1e3] == 1).all() and (slopes[xv < -1e3] == 0).all()
    if name == "relu":
        assert (slopes[xv == 0] == 0).all()


@pytest.mark.parametrize("kind,rows,k,n,order", [("bf16", 64, 256, 512, "kn"), ("f16", 300, 1000, 77, "nk"), ("bf16", 33, 8200, 64, "kn")])
def test_captured_calls_replay(kind, rows, k, n, order):
    """Two captured steps replayed in turn, with eager calls of the same sizes
    (which take cached scratch) between them."""
    calls = []
    for seed in (1, 2):
        c = Case(kind, rows, k, n, order, seed)
        d = c.dev
        y, z = c.forward("gelu")
        want = [bits(t.numpy()) for t in (y, z, *C.dense_adjoint(d["x"], d["w"], d["g"], z, "gelu",
                                                                 dw=c.matrix(C.empty(c.w.shape, NP[kind]))))]
        out = [C.empty(y.shape, y.dtype), C.empty(y.shape, y.dtype), C.empty((rows, k), NP[kind]),
               c.matrix(C.empty(c.w.shape, NP[kind])), C.empty((n,), NP[kind])]

        def step(d=d, out=out):
            C.dense(d["x"], d["w"], d["bias"], "gelu", d["res"], out[0], out[1])
            C.dense_adjoint(d["x"], d["w"], d["g"], out[1], "gelu", *out[2:])

        C.synchronize()
        calls.append((c, z, out, want, Captured(step)))
    for _ in range(3):
        for *_, graph in calls:
            graph.launch()
        for c, z, out, want, graph in calls:
            c.forward("gelu")
            C.dense_adjoint(c.dev["x"], c.dev["w"], c.dev["g"], z, "gelu")
            C.synchronize()
            assert all(np.array_equal(bits(o.numpy()), w) for o, w in zip(out, want))
