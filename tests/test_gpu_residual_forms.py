"""The residual stream in forms beside the usual batch of rows: a norm that stands for
none, one row without leading axes."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import check, decode, draw
from training_reference import residual_norm, residual_norm_adjoint

pytestmark = pytest.mark.gpu
EPS, SCALE = 1e-5, 0.7


def bits(a):
    return np.ascontiguousarray(a).view(np.uint8)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("post,pre", [("none", "rms"), ("layer", "none"), ("none", "none")])
def test_kind_none_is_no_norm(kind, post, pre):
    rng = np.random.default_rng(1)
    x, b, du, dh, gate = (C.to_device(draw(kind, rng, s)[0]) for s in (*[(2, 7, 65)] * 4, (65,)))
    make = lambda how, absent: None if how == "none" and absent else C.Norm(how)
    runs = []
    for absent in (False, True):
        po, pr = make(post, absent), make(pre, absent)
        u, h = C.residual_norm(x, b, po, gate, SCALE, pr, EPS)
        assert (h is None) == (pre == "none")
        dx, db, dgate, dpost, dpre = C.residual_norm_adjoint(u, b, po, gate, SCALE, pr, du, None if h is None else dh)
        assert dpost == dpre == (None, None)
        runs.append([t.numpy() for t in (u, h, dx, db, dgate) if t is not None])
    assert all(np.array_equal(bits(a), bits(c)) for a, c in zip(*runs))


@pytest.mark.parametrize("kind", ["f32", "f64", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 9, 1000, 9001])
def test_one_row_without_leading_axes(kind, n):
    rng = np.random.default_rng(n)
    host = {k: draw(kind, rng, n, *how) for k, how in
            {"x": (1.5, 0.25), "b": (0.8,), "du": (0.01,), "dh": (0.01,), "gate": (0.3, 0.5), "g1": (0.1, 1.0), "g2": (0.1, 1.0)}.items()}
    d, v = {k: C.to_device(s) for k, (s, _) in host.items()}, {k: a for k, (_, a) in host.items()}
    post, pre = C.Norm("rms", d["g1"]), C.Norm("layer", d["g2"])
    u, h = C.residual_norm(d["x"], d["b"], post, d["gate"], SCALE, pre, EPS)
    assert u.shape == h.shape == (n,)
    want = residual_norm(kind, v["x"], v["b"], ("rms", v["g1"], None), v["gate"], SCALE, ("layer", v["g2"], None), EPS)
    check(decode(kind, u.numpy()), *want["u"], "u")
    check(decode(kind, h.numpy()), *want["h"], "h")
    got = C.residual_norm_adjoint(u, d["b"], post, d["gate"], SCALE, pre, d["du"], d["dh"])
    one = lambda t: t.numpy().astype(np.float64).reshape(1, 1)
    row = lambda a: a.reshape(1, 1, n)
    want = residual_norm_adjoint(kind, kind, row(decode(kind, u.numpy())), row(v["b"]), ("rms", v["g1"], None, None, one(post.rstd)),
                                 v["gate"], SCALE, ("layer", v["g2"], None, one(pre.mean), one(pre.rstd)), row(v["du"]), row(v["dh"]))
    for name, t in (("dx", got[0]), ("db", got[1]), ("dgate", got[2]), ("post_dgamma", got[3][0]), ("pre_dgamma", got[4][0])):
        check(decode(kind, t.numpy()).reshape(n), *(a.reshape(n) for a in want[name]), name)

