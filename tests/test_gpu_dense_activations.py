"""The dense operators' activations and slopes at every finite 16-bit value, with the
bound of the arithmetic that they use, also where a residual cancels the value.

GELU's tail Phi(-a) = q(t) exp(-a^2/2), t = 1/(1 + a/K): the polynomial is within
6.4e-8 (its generator's figure, checked here without a device). Beside it, in steps E =
2^-24: t carries a/K's two roundings, the sum's and the reciprocal's last place (6),
through a polynomial whose relative slope stays under 2; its eight fused steps with
coefficients whose magnitudes sum to under 2.5 q (20); the exponential's argument a^2
0.72 rounded twice and its constant once (3 a^2/2), and its last place (2); the
products with a (3). Rounded up: (38 + 1.5 a^2) E. Results under 2^-118 may go to 0:
the hardware's exponential and reciprocal end at 2^-126 and are multiplied by at most
100."""
import os
import sys

import numpy as np
import pytest

import chelis_amd as C
from block_reference import TINY, check, decode, encode, half_step
from training_reference import E, LOG2E, erfc
from training_reference import act as plain_act

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
POLY, FLOOR = 6.4e-8, 2.0**-118


def every(kind):
    """All finite values of the type: [1, count] stored, and in binary64."""
    b = np.arange(1 << 16, dtype=np.uint16)
    b = b if kind == "bf16" else b.view(np.float16)
    b = b[np.isfinite(decode(kind, b))]
    return b[None], decode(kind, b)


def tail(x):
    a = np.minimum(np.abs(x), 40.0)
    return 0.5 * erfc(a / np.sqrt(2)), np.exp(-0.5 * a * a) / np.sqrt(2 * np.pi), POLY + (38 + 1.5 * a * a) * E


def sigmoid(x):
    s = 1 / (1 + np.exp(-np.clip(x, -200, 200)))
    return s, ((np.minimum(np.abs(x), 200) * LOG2E + 4) * E) * (1 - s) + 6 * E


def act(name, x):
    if name == "gelu":
        t, _, rel = tail(x)
        a = np.minimum(np.abs(x), 40.0)
        y = np.where(x >= 0, x - a * t, -a * t)
        return y, rel * a * t + E * np.abs(y) + FLOOR
    if name == "silu":
        s, rel = sigmoid(x)
        return x * s, (rel + E) * np.abs(x * s) + FLOOR
    return np.maximum(x, 0), 0 * x


def slope(name, x):
    if name == "gelu":
        t, density, rel = tail(x)
        a = np.minimum(np.abs(x), 40.0)
        below = t - a * density  # q e - a e / sqrt(2 pi), one fused step and a product
        eb = rel * t + (4 + 1.5 * a * a) * E * a * density + 2 * E * (t + a * density)
        return np.where(x < 0, below, 1 - below), eb + E + FLOOR
    if name == "silu":
        s, rel = sigmoid(x)
        c = np.minimum(np.abs(x), 200) * np.sign(x)
        d = s * (1 + c * (1 - s))
        # 1 - s is off by s's error and a rounding
        return d, rel * np.abs(d) + s * np.abs(c) * (rel * s + E) + 4 * E * (s + s * np.abs(c) * (1 - s)) + FLOOR
    return (x > 0) * 1.0, 0 * x


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("name", ["gelu", "silu", "relu"])
def test_activations(kind, name):
    """Through x = 1 by one row of weights: z is the value itself."""
    w, v = every(kind)
    one = C.to_device(encode(kind, np.ones((1, 1))))
    y, z = C.dense(one, C.to_device(w), act=name, z=True)
    assert np.array_equal(decode(kind, z.numpy())[0], v)
    want, bound = act(name, v)
    check(decode(kind, y.numpy())[0], want, bound + half_step(kind) * (np.abs(want) + bound) + TINY[kind], name)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("name", ["gelu", "silu", "relu"])
def test_slopes(kind, name):
    """dbias of one row with g = 1, in f32: the slope as it is formed."""
    z, v = every(kind)
    n = len(v)
    one = C.to_device(encode(kind, np.ones((1, 1))))
    _, _, db = C.dense_adjoint(one, C.to_device(encode(kind, np.ones((1, n)))), C.to_device(encode(kind, np.ones((1, n)))),
                               C.to_device(z), name, dbias=C.empty((n,), np.float32), want_dx=False, want_dw=False)
    want, bound = slope(name, v)
    check(db.numpy().astype(np.float64), want, bound, name)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("name", ["gelu", "silu", "relu"])
def test_values_that_the_residual_cancels(kind, name):
    """y = act(z) + r with r the value's negative rounded to 16 bits: what is left is
    of the size of a rounding, and stored to 16 bits of its own. The sum is one more
    rounding in binary32, and the plain form's bound holds as well."""
    w, v = every(kind)
    want, bound = act(name, v)
    r = encode(kind, -want)
    left = want + decode(kind, r)
    ok = np.isfinite(left)
    one = C.to_device(encode(kind, np.ones((1, 1))))
    y = decode(kind, C.dense(one, C.to_device(w), None, name, C.to_device(r[None])).numpy())[0]
    for b in (bound, plain_act(name, np.clip(v, -60, 60))[1] + bound * (np.abs(v) >= 60)):
        b = b + 2 * E * (np.abs(left) + np.abs(want))
        check(y[ok], left[ok], (b + half_step(kind) * (np.abs(left) + b) + TINY[kind])[ok], name)


def test_the_polynomial_is_as_good_as_its_header_says():
    """The coefficients that the kernels hold, in binary64."""
    sys.path.insert(0, os.path.join(ROOT, "chelis_amd", "csrc"))
    try:
        import gen_gelu16_poly as gen
    finally:
        sys.path.pop(0)
    text = open(os.path.join(ROOT, "chelis_amd", "csrc", "gelu16_poly.h")).read()
    held = [float.fromhex(t.strip().rstrip("f")) for t in text[text.rindex("{") + 1:text.rindex("}")].replace("\\", "").split(",")]
    assert len(held) == gen.DEG + 1
    a = np.linspace(0.0, gen.AMAX, 200001)
    err = np.abs(np.polyval(held[::-1], gen.K / (a + gen.K)) / (0.5 * gen.erfcx(a / np.sqrt(2.0))) - 1).max()
    assert err < POLY
