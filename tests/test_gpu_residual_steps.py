"""The residual stream's gradients where a workgroup takes several steps through its
rows, the last one ragged: the column sums carried over the steps, rows requested one
ahead, results over inputs whose next rows are already under way, rows of a later
step that are not there; and long rows in several partial sums a gate.

The sums over rows are held to the chain that forms them, not to the number of rows:
a lane adds a row of each step, at most 32 rows join in the workgroup, at most 32
partial sums a thread and 32 threads join in the second launch, and the gates'
sums: under 160 additions for these sizes, each 2^-24 (2^-53) of the sum of
magnitudes. A row that is missing or counted twice is far outside that."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import TINY, check, decode, draw, encode, half_step, width_of
from training_reference import residual_norm_adjoint

pytestmark = pytest.mark.gpu
EPS, SCALE, CHAIN = 1e-5, 0.7, 160

# (groups, rows, n): three steps or more in every launch form (16 lanes a row, one wave,
# two, four and eight) on 256 compute units, the last one short
WIDE = [(1, 6149, 1000), (3, 2051, 264), (1, 2600, 2049), (2, 9001, 50), (1, 601, 4500), (2, 1301, 1500), (2, 150, 8192), (1, 6149, 512)]
F64 = [(1, 6149, 500), (3, 2051, 133), (2, 4500, 25), (1, 2600, 1000), (1, 1301, 2000), (1, 601, 3500)]
CASES = [("f32", "f32", s) for s in WIDE] + [(k, "f32", s) for k in ("bf16", "f16") for s in WIDE + [(2, 9001, 100)]] + \
    [("f64", "f64", s) for s in F64] + [("bf16", "bf16", (1, 6149, 1000)), ("f16", "f16", (2, 9001, 100))]
LONG = [("f32", "f32", (2, 41, 8200)), ("bf16", "f32", (1, 83, 9000)), ("f16", "f32", (3, 40, 8193)), ("f64", "f64", (1, 70, 4100)),
        ("bf16", "bf16", (2, 41, 16390))]


def bits(a):
    return np.ascontiguousarray(a).view(np.uint8)


class Case:
    def __init__(self, kind, weights, shape, post, pre, seed):
        rng = np.random.default_rng(seed)
        groups, rows, n = shape
        self.kind, self.weights, self.shape, self.n = kind, weights, shape, n
        host = {"u": draw(kind, rng, shape, 1.5, 0.25), "b": draw(kind, rng, shape, 0.8, 0.1), "du": draw(kind, rng, shape, 0.01),
                "dh": draw(kind, rng, shape, 0.01), "gate": draw(weights, rng, (groups, n), 0.3, 0.5)}
        self.how = {"post": post, "pre": pre}
        for side in ("post", "pre"):
            if self.how[side] != "none":
                host[side + "_gamma"] = draw(weights, rng, n, 0.1, 1.0)
            if self.how[side] == "layer":
                host[side + "_beta"] = draw(weights, rng, n, 0.1)
        self.host, self.val = {k: s for k, (s, _) in host.items()}, {k: v for k, (_, v) in host.items()}
        stat = np.float64 if kind == "f64" else np.float32
        self.stat = {}
        for side, rowsv in (("post", "b"), ("pre", "u")):
            if self.how[side] == "none":
                continue
            x = self.val[rowsv]
            mean = x.mean(-1) if self.how[side] == "layer" else 0 * x[..., 0]
            c = x - mean[..., None]
            self.stat[side] = [mean.astype(stat), (1 / np.sqrt((c * c).mean(-1) + EPS)).astype(stat)]

    def device(self):
        return {k: C.to_device(v) for k, v in self.host.items()}

    def norm(self, d, side):
        if self.how[side] == "none":
            return None
        mean, rstd = self.stat[side]
        return C.Norm(self.how[side], d[side + "_gamma"], d.get(side + "_beta"),
                      C.to_device(mean) if self.how[side] == "layer" else None, C.to_device(rstd))

    def run(self, d, **to):
        return C.residual_norm_adjoint(d["u"], d["b"], self.norm(d, "post"), d["gate"], SCALE, self.norm(d, "pre"), d["du"],
                                       d["dh"] if self.how["pre"] != "none" else None, **to)

    def want(self):
        """The plain form's values, its bounds for rows, and for sums over rows those
        of the chain."""
        v, e = self.val, width_of(self.kind)

        def plain(side):
            if self.how[side] == "none":
                return None
            mean, rstd = (s.astype(np.float64) for s in self.stat[side])
            return (self.how[side], v[side + "_gamma"], v.get(side + "_beta"), mean, rstd)

        post, pre = plain("post"), plain("pre")
        gate = v["gate"][:, None]
        w = residual_norm_adjoint(self.kind, self.weights, v["u"], v["b"], post, gate, SCALE, pre, v["du"], v["dh"] if pre else None)
        u, tiny = half_step(self.kind), TINY[self.kind]
        bound = w["dx"][1]
        t = w["dx"][0]
        et = (bound - tiny - u * np.abs(t)) / (1 + u)  # t before its rounding

        def unit(x, side):
            if side is None:
                return x, 0 * x
            k = (x - (side[3][..., None] if side[0] == "layer" else 0.0)) * side[4][..., None]
            return k, 3 * e * np.abs(k)

        def total(a, ea, axes):
            return a.sum(axes), ea.sum(axes) + CHAIN * e * np.abs(a).sum(axes)

        def put(name, s, es):
            uw = half_step(self.weights)
            assert np.allclose(s, w[name][0], rtol=1e-9, atol=1e-12)
            w[name] = (s, es + uw * (np.abs(s) + es) + TINY[self.weights])

        k, ek = unit(v["b"], post)
        s1, e1 = total(t, et, 1)
        s2, e2 = total(t * k, et * np.abs(k) + np.abs(t) * ek + e * np.abs(t * k), 1)
        gamma = 1.0 if post is None else post[1]
        beta = 0.0 if post is None or post[2] is None else post[2]
        g, eg = gamma * s2 + beta * s1, np.abs(gamma) * e2 + np.abs(beta) * e1 + 4 * e * (np.abs(gamma * s2) + np.abs(beta * s1))
        put("dgate", SCALE * g, SCALE * (eg + e * np.abs(g)))
        if post:
            f = SCALE * v["gate"]
            for name, s, es in (("post_dgamma", s2, e2), ("post_dbeta", s1, e1)):
                if name in w:
                    put(name, (f * s).sum(0), (np.abs(f) * es + 4 * e * np.abs(f * s)).sum(0))
        if pre:
            m, em = unit(v["u"], pre)
            put("pre_dgamma", *total(v["dh"] * m, np.abs(v["dh"]) * em + e * np.abs(v["dh"] * m), (0, 1)))
            put("pre_dbeta", *total(v["dh"], 0 * m, (0, 1)))
        return w


def flat(got):
    dx, db, dgate, dpost, dpre = got
    return {"dx": dx, "db": db, "dgate": dgate, "post_dgamma": dpost[0], "post_dbeta": dpost[1], "pre_dgamma": dpre[0],
            "pre_dbeta": dpre[1]}


def check_all(c, got, want):
    for name, t in flat(got).items():
        if t is None:
            continue
        value, bound = want[name]
        kind = c.kind if name in ("dx", "db") else c.weights
        check(decode(kind, t.numpy()).reshape(value.shape), value, bound, name)


@pytest.mark.parametrize("kind,weights,shape", CASES + LONG)
@pytest.mark.parametrize("post,pre", [("layer", "layer"), ("rms", "none")])
def test_sums_over_several_steps(kind, weights, shape, post, pre):
    c = Case(kind, weights, shape, post, pre, sum(shape))
    check_all(c, c.run(c.device()), c.want())


@pytest.mark.parametrize("kind,weights,shape", [("f32", "f32", (1, 6149, 1000)), ("bf16", "f32", (1, 6149, 1000)), ("bf16", "f32", (2, 9001, 100)),
                                                ("f16", "f32", (1, 2600, 2049)), ("f16", "f16", (3, 2051, 264)), ("f64", "f64", (1, 2600, 1000)),
                                                ("f32", "f32", (2, 41, 8200)), ("bf16", "f32", (1, 601, 4500))])
@pytest.mark.parametrize("dx,db", [("u", "b"), ("b", "u"), ("du", "dh"), ("dh", "du"), ("du", "b"), ("u", "dh")])
def test_results_over_inputs(kind, weights, shape, dx, db):
    c = Case(kind, weights, shape, "rms", "layer", 5)
    want = flat(c.run(c.device()))
    d = c.device()
    got = flat(c.run(d, dx=d[dx], db=d[db]))
    for name, t in want.items():
        assert t is None or np.array_equal(bits(t.numpy()), bits(got[name].numpy())), name


@pytest.mark.parametrize("kind,weights,shape", [("f32", "f32", (1, 6149, 1000)), ("bf16", "f32", (1, 6149, 1000)), ("f16", "f32", (2, 9001, 100))])
def test_a_special_row_of_a_later_step_stays_alone(kind, weights, shape):
    """A NaN in a row of the last, ragged step: the other rows keep their bits, and
    only its column sums turn NaN (dbeta's in its own column alone)."""
    c = Case(kind, weights, shape, "rms", "layer", 6)
    plain = flat(c.run(c.device()))
    at = (shape[0] - 1, shape[1] - 2, 7)
    held = decode(kind, c.host["dh"]).copy()
    held[at] = np.nan
    c.host["dh"] = encode(kind, held)
    got = flat(c.run(c.device()))
    for name in ("dx", "db"):
        a, b = decode(kind, got[name].numpy()), decode(kind, plain[name].numpy())
        assert np.isnan(a[at[0], at[1]]).all()
        a[at[0], at[1]] = b[at[0], at[1]] = 0
        assert np.array_equal(a, b)
    a, b = decode(weights, got["pre_dbeta"].numpy()), decode(weights, plain["pre_dbeta"].numpy())
    assert np.isnan(a[7]) and np.array_equal(np.delete(a, 7), np.delete(b, 7))
