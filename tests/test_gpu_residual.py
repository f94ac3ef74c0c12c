"""The residual stream between two blocks (norm, gate, scale, sum, norm) and its
gradients against the plain binary64 form: lengths from one element to rows past
the register capacity, every dtype, each part absent, gates for runs of rows,
strides, aliasing, special rows, graph replays, differences."""
import itertools

import numpy as np
import pytest

import chelis_amd as C
from block_reference import NP, Captured, check, decode, draw, encode
from training_reference import residual_norm, residual_norm_adjoint

pytestmark = pytest.mark.gpu
EPS, SCALE = 1e-5, 0.7
TYPES = [("f32", "f32"), ("f64", "f64"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")]
# (groups, rows, n): every launch shape of each width, vectors moved back at a row's end, long rows
SHAPES = [(1, 1, 1), (2, 3, 7), (1, 5, 8), (3, 4, 33), (1, 130, 128), (2, 37, 129), (1, 70, 500), (5, 13, 512),
          (1, 9, 1000), (2, 515, 1024), (1, 3, 2049), (40, 1, 264), (3, 2, 4104), (1, 5, 8200), (1, 2, 16384), (2, 3, 16389)]
PARTS = [("layer", "layer", True), ("rms", "rms", True), ("none", "layer", False), ("layer", "none", True),
         ("rms", "layer", False), ("none", "none", True), ("none", "rms", True)]


def bits(a):
    return np.ascontiguousarray(a).view(np.uint8)


class Case:
    def __init__(self, kind, weights, groups, rows, n, post, pre, gate, seed):
        rng = np.random.default_rng(seed)
        self.kind, self.weights, self.shape, self.n = kind, weights, (groups, rows, n), n
        self.host, self.val = {}, {}

        def add(name, t, shape, scale, mean=0.0):
            self.host[name], self.val[name] = draw(t, rng, shape, scale, mean)

        add("x", kind, self.shape, 1.5, 0.25)
        add("b", kind, self.shape, 0.8, 0.1)
        add("du", kind, self.shape, 0.01)
        add("dh", kind, self.shape, 0.01)
        for side, how in (("post", post), ("pre", pre)):
            if how != "none":
                add(side + "_gamma", weights, n, 0.1, 1.0)
            if how == "layer":
                add(side + "_beta", weights, n, 0.1)
        if gate:
            add("gate", weights, (groups, n) if groups > 1 else (n,), 0.3, 0.5)
        self.dev = {k: C.to_device(v) for k, v in self.host.items()}
        self.how = {"post": post, "pre": pre}
        gv = self.val.get("gate")
        self.gate = None if gv is None else gv[:, None] if groups > 1 else gv

    def norm(self, side, mean=None, rstd=None):
        if self.how[side] == "none":
            return None
        return C.Norm(self.how[side], self.dev[side + "_gamma"], self.dev.get(side + "_beta"), mean, rstd)

    def plain(self, side, norm=None):
        if self.how[side] == "none":
            return None
        out = (self.how[side], self.val[side + "_gamma"], self.val.get(side + "_beta"))
        if norm is not None:
            out += (None if norm.mean is None else norm.mean.numpy().astype(np.float64), norm.rstd.numpy().astype(np.float64))
        return out


def forward(c, **to):
    post, pre = c.norm("post"), c.norm("pre")
    u, h = C.residual_norm(c.dev["x"], c.dev["b"], post, c.dev.get("gate"), SCALE, pre, EPS, **to)
    return u, h, post, pre


def check_forward(c, u, h, post, pre):
    want = residual_norm(c.kind, c.val["x"], c.val["b"], c.plain("post"), c.gate, SCALE, c.plain("pre"), EPS)
    check(decode(c.kind, u.numpy()), *want["u"], "u")
    if pre:
        check(decode(c.kind, h.numpy()), *want["h"], "h")
    for name, norm in (("post", post), ("pre", pre)):
        if norm:
            check(norm.rstd.numpy().astype(np.float64), *want[name + "_rstd"], name + " rstd")
            if norm.kind == "layer":
                check(norm.mean.numpy().astype(np.float64), *want[name + "_mean"], name + " mean")


def check_adjoint(c, got, u, post, pre):
    dx, db, dgate, dpost, dpre = got
    want = residual_norm_adjoint(c.kind, c.weights, decode(c.kind, u.numpy()), c.val["b"], c.plain("post", post), c.gate, SCALE,
                                 c.plain("pre", pre), c.val["du"], c.val["dh"] if pre else None)
    check(decode(c.kind, dx.numpy()), *want["dx"], "dx")
    check(decode(c.kind, db.numpy()), *want["db"], "db")
    if dgate is not None:
        shape = dgate.shape
        check(decode(c.weights, dgate.numpy()), want["dgate"][0].reshape(-1, c.n).sum(0) if len(shape) == 1 else want["dgate"][0],
              want["dgate"][1].reshape(-1, c.n).sum(0) if len(shape) == 1 else want["dgate"][1], "dgate")
    for name, pair in (("post", dpost), ("pre", dpre)):
        for part, t in zip(("_dgamma", "_dbeta"), pair):
            if t is not None:
                check(decode(c.weights, t.numpy()), *want[name + part], name + part)


def adjoint(c, u, post, pre, **to):
    return C.residual_norm_adjoint(u, c.dev["b"], post, c.dev.get("gate"), SCALE, pre, c.dev["du"], c.dev["dh"] if pre else None, **to)


@pytest.mark.parametrize("groups,rows,n", SHAPES)
@pytest.mark.parametrize("kind,weights", TYPES)
def test_forward_and_gradients(kind, weights, groups, rows, n):
    for i, (post, pre, gate) in enumerate(PARTS if n < 4000 else PARTS[:2]):
        c = Case(kind, weights, groups, rows, n, post, pre, gate, rows * 31 + n + i)
        u, h, po, pr = forward(c)
        check_forward(c, u, h, po, pr)
        got = adjoint(c, u, po, pr)
        check_adjoint(c, got, u, po, pr)
        # some gradients alone, and again: the same bits
        again = C.residual_norm_adjoint(u, c.dev["b"], po, c.dev.get("gate"), SCALE, pr, c.dev["du"], c.dev["dh"] if pr else None,
                                        want_weights=False)
        assert all(np.array_equal(bits(a.numpy()), bits(b.numpy())) for a, b in zip(again[:2], got[:2]))
        assert again[2] is None and again[3] == (None, None) and again[4] == (None, None)


@pytest.mark.parametrize("kind,weights,n", [("f32", "f32", 40001), ("bf16", "f32", 33000), ("f64", "f64", 9000), ("f16", "f16", 8193)])
def test_rows_past_the_register_capacity(kind, weights, n):
    for post, pre, gate in PARTS:
        c = Case(kind, weights, 2, 3, n, post, pre, gate, n)
        u, h, po, pr = forward(c)
        check_forward(c, u, h, po, pr)
        check_adjoint(c, adjoint(c, u, po, pr), u, po, pr)


@pytest.mark.parametrize("kind,weights", TYPES)
@pytest.mark.parametrize("n", [65, 1000, 17000])
def test_results_over_inputs(kind, weights, n):
    c = Case(kind, weights, 2, 5, n, "layer", "rms", True, 4)
    u, h, po, pr = forward(c)
    got = adjoint(c, u, po, pr)
    for to in ({"u": "x", "h": "b"}, {"u": "b", "h": "x"}):
        t = Case(kind, weights, 2, 5, n, "layer", "rms", True, 4)
        uu, hh, _, _ = forward(t, **{k: t.dev[v] for k, v in to.items()})
        assert np.array_equal(bits(uu.numpy()), bits(u.numpy())) and np.array_equal(bits(hh.numpy()), bits(h.numpy()))
    for dx, db in itertools.permutations(("du", "dh", "b", "u"), 2):
        t = Case(kind, weights, 2, 5, n, "layer", "rms", True, 4)
        t.dev["u"] = C.clone(u)
        t.dev.update(dx=t.dev[dx], db=t.dev[db])
        over = C.residual_norm_adjoint(t.dev["u"], t.dev["b"], po, t.dev["gate"], SCALE, pr, t.dev["du"], t.dev["dh"],
                                       dx=t.dev["dx"], db=t.dev["db"])
        flat = lambda r: [r[0], r[1], r[2], *r[3], *r[4]]
        assert all(a is None or np.array_equal(bits(a.numpy()), bits(b.numpy())) for a, b in zip(flat(over), flat(got)))


@pytest.mark.parametrize("kind", ["f32", "f64", "bf16", "f16"])
@pytest.mark.parametrize("how", ["layer", "rms"])
@pytest.mark.parametrize("n", [5, 264, 1000, 9000])
def test_a_norm_alone(kind, how, n):
    """Without a block's result: h = pre(x), and its gradient beside what
    arrives at x from elsewhere, or alone."""
    c = Case(kind, kind, 1, 6, n, "none", how, False, 9)
    pre = c.norm("pre")
    none, h = C.residual_norm(c.dev["x"], pre=pre, eps=EPS)
    assert none is None
    want = residual_norm(kind, c.val["x"], None, None, None, 1.0, c.plain("pre"), EPS)
    check(decode(kind, h.numpy()), *want["h"], "h")
    for du in (None, "du"):
        dx, db, dgate, _, dpre = C.residual_norm_adjoint(c.dev["x"], pre=pre, du=c.dev.get(du), dh=c.dev["dh"])
        assert db is None and dgate is None
        want = residual_norm_adjoint(kind, kind, c.val["x"], None, None, None, 1.0, c.plain("pre", pre),
                                     c.val["du"] if du else None, c.val["dh"])
        check(decode(kind, dx.numpy()), *want["dx"], "dx")
        check(decode(kind, dpre[0].numpy()), *want["pre_dgamma"], "dgamma")


def test_a_norm_without_weights():
    c = Case("bf16", "bf16", 1, 7, 520, "rms", "rms", False, 2)
    for side in ("post", "pre"):
        c.val[side + "_gamma"] = None
    post, pre = C.Norm("rms"), C.Norm("rms")
    u, h = C.residual_norm(c.dev["x"], c.dev["b"], post, None, SCALE, pre, EPS)
    check_forward(c, u, h, post, pre)
    check_adjoint(c, adjoint(c, u, post, pre), u, post, pre)


@pytest.mark.parametrize("kind,weights", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
def test_strided_rows_keep_what_lies_between(kind, weights):
    groups, rows, n, ld, off = 2, 3, 203, 260, 3
    c = Case(kind, weights, groups, rows, n, "layer", "layer", True, 8)
    rng = np.random.default_rng(9)

    def strided(a):
        back = draw(kind, rng, groups * rows * ld + off)[0]
        back[off:].reshape(groups, rows, ld)[:, :, :n] = a
        t = C.to_device(back)
        return t, back, t.view((groups, rows, n), (rows * ld, ld, 1), off)

    kept = {k: strided(c.host[k]) for k in ("x", "b", "du", "dh")}
    results = {k: strided(c.host["x"]) for k in ("u", "h", "dx", "db")}
    for k, (_, _, view) in kept.items():
        c.dev[k] = view
    u, h, po, pr = forward(c, u=results["u"][2], h=results["h"][2])
    check_forward(c, u, h, po, pr)
    check_adjoint(c, adjoint(c, u, po, pr, dx=results["dx"][2], db=results["db"][2]), u, po, pr)
    for t, back, _ in results.values():
        now = t.numpy()
        assert np.array_equal(bits(now[:off]), bits(back[:off]))
        gap = lambda a: bits(a[off:].reshape(groups, rows, ld)[:, :, n:])
        assert np.array_equal(gap(now), gap(back))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [100, 1000, 17000])
def test_special_rows_stay_in_their_rows(kind, n):
    for value in (np.nan, np.inf):
        c = Case(kind, kind, 1, 8, n, "layer", "rms", True, n)
        plain = forward(c)
        v = c.val["b"].copy()
        v[0, 3, n // 2] = value
        c.dev["b"] = C.to_device(encode(kind, v))
        u, h, po, pr = forward(c)
        keep = [i for i in range(8) if i != 3]
        for a, b in zip((u, h), plain):
            assert np.array_equal(bits(a.numpy()[0, keep]), bits(b.numpy()[0, keep]))
            assert np.isnan(decode(kind, a.numpy())[0, 3]).all()
        dx, db, *_ = adjoint(c, u, po, pr)
        wx, wb, *_ = adjoint(c, plain[0], plain[2], plain[3])
        assert np.array_equal(bits(dx.numpy()[0, keep]), bits(wx.numpy()[0, keep]))
        c.dev["b"] = C.to_device(c.host["b"])
        wx, wb, *_ = adjoint(c, plain[0], plain[2], plain[3])
        assert np.array_equal(bits(db.numpy()[0, keep]), bits(wb.numpy()[0, keep]))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [24, 9000])
def test_no_rows_give_zero_weight_gradients(kind, n):
    for shape, gate in (((0, n), (n,)), ((2, 0, n), (2, n)), ((0, 5, n), (0, n))):
        x, g = C.empty(shape, NP[kind]), C.to_device(encode(kind, np.ones(gate)))
        w = lambda: C.to_device(encode(kind, np.ones(n)))
        post, pre = C.Norm("layer", w(), w()), C.Norm("rms", w())
        C.residual_norm(x, C.empty(shape, NP[kind]), post, g, SCALE, pre, EPS)
        dpost, dpre, dgate = (w(), w()), (w(), None), C.to_device(encode(kind, np.ones(gate)))
        C.residual_norm_adjoint(x, C.empty(shape, NP[kind]), post, g, SCALE, pre, x, x, dgate=dgate, dpost=dpost, dpre=dpre)
        for t in (*dpost, dpre[0], dgate):
            assert not t.numpy().any()


def test_gradients_against_differences():
    """Central differences of the binary64 forward: for h = 1e-5 their own
    error is below 1e-8 of the gradient's scale at these sizes."""
    rng = np.random.default_rng(3)
    groups, rows, n, h = 2, 3, 37, 1e-5
    for how in ("layer", "rms"):
        v = {"x": rng.standard_normal((groups, rows, n)), "b": rng.standard_normal((groups, rows, n)),
             "gate": rng.standard_normal((groups, n)), "post_gamma": rng.standard_normal(n), "post_beta": rng.standard_normal(n),
             "pre_gamma": rng.standard_normal(n), "pre_beta": rng.standard_normal(n)}
        du, dh = rng.standard_normal((2, groups, rows, n))

        def run(a):
            d = {k: C.to_device(t) for k, t in a.items()}
            post, pre = C.Norm(how, d["post_gamma"], d["post_beta"]), C.Norm(how, d["pre_gamma"], d["pre_beta"])
            u, hh = C.residual_norm(d["x"], d["b"], post, d["gate"], SCALE, pre, EPS)
            return d, post, pre, u, (u.numpy() * du).sum() + (hh.numpy() * dh).sum()

        d, post, pre, u, _ = run(v)
        dx, db, dgate, dpost, dpre = C.residual_norm_adjoint(u, d["b"], post, d["gate"], SCALE, pre, C.to_device(du), C.to_device(dh))
        for name, grad in zip(("x", "b", "gate", "post_gamma", "post_beta", "pre_gamma", "pre_beta"), (dx, db, dgate, *dpost, *dpre)):
            way = rng.standard_normal(v[name].shape)
            want = (run({**v, name: v[name] + h * way})[-1] - run({**v, name: v[name] - h * way})[-1]) / (2 * h)
            assert abs((grad.numpy() * way).sum() - want) < 1e-6 * np.abs(grad.numpy() * way).sum(), name


@pytest.mark.parametrize("kind,weights,shape", [("f32", "f32", (2, 150, 500)), ("bf16", "f32", (1, 40, 3000)),
                                                ("bf16", "bf16", (3, 11, 17000))])
def test_captured_calls_replay(kind, weights, shape):
    """Two captured steps replayed in turn, with eager calls of the same sizes
    (which take cached scratch) between them."""
    calls = []
    for seed in (1, 2):
        c = Case(kind, weights, *shape, "layer", "rms", True, seed)
        u, h, po, pr = forward(c)
        flat = lambda r: [r[0], r[1], r[2], *r[3], r[4][0]]
        want = [bits(t.numpy()) for t in (u, h, *flat(adjoint(c, u, po, pr)))]
        out = [C.empty(t.shape, t.dtype) for t in (u, h, *flat(adjoint(c, u, po, pr)))]

        def step(c=c, out=out, po=po, pr=pr):
            C.residual_norm(c.dev["x"], c.dev["b"], po, c.dev["gate"], SCALE, pr, EPS, u=out[0], h=out[1])
            C.residual_norm_adjoint(out[0], c.dev["b"], po, c.dev["gate"], SCALE, pr, c.dev["du"], c.dev["dh"], dx=out[2], db=out[3],
                                    dgate=out[4], dpost=(out[5], out[6]), dpre=(out[7], None))

        C.synchronize()
        calls.append((c, u, po, pr, out, want, Captured(step)))
    for _ in range(3):
        for *_, graph in calls:
            graph.launch()
        for c, u, po, pr, out, want, graph in calls:
            adjoint(c, u, po, pr)
            C.synchronize()
            assert all(np.array_equal(bits(o.numpy()), w) for o, w in zip(out, want))
