"""The norm of f64 gradients over binary64's whole range, where their squares leave
it, against sums in extended precision (its exponents reach 2^16383), alone and
beside the other types; and their clipping by it."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import draw

pytestmark = pytest.mark.gpu
WIDE = np.longdouble
# At most 2^14 terms: a thread's and the join's sums are under 2^7 additions long, 2^-53
# each of the sum of squares; half of that in its root, three more roundings behind it.
REL = 2.0**-46


def exact(*values, scale=1.0):
    return float(WIDE(scale) * np.sqrt(sum((v.astype(WIDE) ** 2).sum() for v in values)))


def norm_of(tensors, scale=1.0, wide=np.float64):
    return float(C.gradient_norm(tensors, scale, C.empty((), wide)).numpy())


@pytest.mark.parametrize("power", [-1074, -1060, -1022, -700, -540, -481, -480, -479, 0, 479, 480, 481, 511, 512, 600, 1017])
def test_powers_of_two(power):
    """4096 equal elements: the norm is 2^(power + 6), every sum exact."""
    t = C.to_device(np.full(4096, np.ldexp(1.0, power)))
    assert norm_of([t]) == np.ldexp(1.0, power + 6)


@pytest.mark.parametrize("low,high", [(-1070, 1015), (-1070, -400), (-500, -460), (-200, -100), (460, 500), (400, 1015)])
@pytest.mark.parametrize("count", [1, 3, 777, 16384])
def test_mixed_magnitudes(low, high, count):
    rng = np.random.default_rng(count)
    v = rng.choice([-1, 1], count) * rng.uniform(1, 2, count) * np.exp2(rng.uniform(low, high, count))
    want = exact(v)
    assert abs(norm_of([C.to_device(v)]) - want) <= REL * want + 2.0**-1074


@pytest.mark.parametrize("v", [[1e200, 3.0, 1e-200], [1e-170, 1e-165], [1e-160, 3e-162, 1e-150], [2.0**480, np.nextafter(2.0**480, 0)],
                               [2.0**-480, np.nextafter(2.0**-480, 0)], [2.0**-100, 2.0**-490], [0.0, 5e-324], [0.0, 0.0]])
def test_a_few_elements(v):
    v = np.array(v)
    want = exact(v)
    assert abs(norm_of([C.to_device(v)]) - want) <= REL * want


def test_the_scale_brings_the_norm_back():
    big = np.full(16, 1.5e308)  # 6e308, past the largest
    assert norm_of([C.to_device(big)]) == np.inf
    for scale in (0.125, 2.0**-70, 2.0**-1000):
        want = exact(big, scale=scale)
        assert abs(norm_of([C.to_device(big)], scale) - want) <= REL * want
    small = np.full(16, 2.0**-1073)
    assert norm_of([C.to_device(small)], 2.0**900) == 2.0**-171
    assert norm_of([C.to_device(small)], 2.0**-2) == 2.0**-1073


def test_beside_other_types_and_in_rows():
    rng = np.random.default_rng(1)
    kinds = [(k, *draw(k, rng, (301,), 0.3)) for k in ("f32", "bf16", "f16")]
    others, values = [C.to_device(s) for _, s, _ in kinds], [v for _, _, v in kinds]
    for size in (1e-250, 1e-3, 1e250):
        wide = rng.standard_normal((70, 40)) * size
        rows = [C.to_device(wide).view((33,), (1,), 40 * i) for i in range(3)]
        strided = C.to_device(wide).view((70, 33), (40, 1), 0)
        want = exact(*values, *[wide[i, :33] for i in range(3)], wide[:, :33])
        got = norm_of([others[0], *rows, strided, *others[1:]])
        assert abs(got - want) <= REL * want
        held = norm_of([others[0], *rows, strided, *others[1:]], wide=np.float32)
        assert held == (np.inf if size > 1e200 else np.float32(got))
    # without f64 elements among them
    empty = C.empty((0, 4), np.float64)
    assert norm_of([*others, empty]) == norm_of(others)


@pytest.mark.parametrize("special", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("beside", [1e-300, 1.0, 1e300])
def test_what_is_not_finite(special, beside):
    v = np.full(500, beside)
    v[77] = special
    got = norm_of([C.to_device(v)])
    assert np.isnan(got) if np.isnan(special) else got == np.inf


@pytest.mark.parametrize("size", [1e-280, 1e-170, 1e160, 1e300])
def test_clipping_far_out(size):
    """The clipped gradients are the gradients times the factor of the norm held,
    in binary64: not zero where the norm was taken for infinite, not as they were
    where it was taken for 0."""
    rng = np.random.default_rng(2)
    v = rng.standard_normal((50, 60)) * size
    t = C.to_device(v)
    norm = C.gradient_norm([t], 1.0, C.empty((), np.float64))
    held, most = float(norm.numpy()), 0.25 * size
    (out,) = C.clip_gradients([t], norm, most, 1.0, [C.empty(v.shape, np.float64)])
    assert np.array_equal(out.numpy(), v * (most / held))
    after = exact(out.numpy())
    assert abs(after - most) <= 2.0**-40 * most


def test_a_captured_call_replays():
    from block_reference import Captured

    t, norm = C.to_device(np.full((64, 64), 1e200)), C.empty((), np.float64)
    other = C.to_device(np.full(5000, 1e-200))
    graph = Captured(lambda: C.gradient_norm([t, other], 0.5, norm))
    for _ in range(3):
        graph.launch()
        assert norm_of([other]) < 1e-190
        C.synchronize()
        assert float(norm.numpy()) == 0.5 * 64e200
