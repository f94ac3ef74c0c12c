"""The tables that a clipping call's tensors travel in, at their ends: 160 dense
tensors to a launch, 64 of rows a step apart, both in one call, cut into several
pieces and into one."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import NP, draw
from test_gpu_clip import norm_of, scaled

pytestmark = pytest.mark.gpu
KINDS = ["f32", "bf16", "f16", "f64"]


def bits(a):
    return np.ascontiguousarray(a).view(np.uint8)


class Dense:
    def __init__(self, rng, kind):
        self.kind = kind
        self.stored, self.value = draw(kind, rng, (int(rng.integers(1, 3000)),), 0.3)
        self.grad = C.to_device(self.stored)
        self.out = C.empty(self.stored.shape, NP[kind])

    def check(self, norm, most, scale):
        assert np.array_equal(self.out.numpy(), scaled(self.kind, self.stored, self.value, norm, most, scale))
        assert np.array_equal(bits(self.grad.numpy()), bits(self.stored))


class Rows:
    """Rows of n in one of ld from an element off on, result rows elsewhere in
    another step; what lies between stays."""

    def __init__(self, rng, kind, rows=None, n=None):
        self.kind = kind
        rows, n = rows or int(rng.integers(2, 9)), n or int(rng.integers(1, 700))
        ld, ldo, off = n + int(rng.integers(1, 9)), n + int(rng.integers(0, 9)), int(rng.integers(0, 5))
        self.back, values = draw(kind, rng, off + rows * ld, 0.3)
        cut = lambda a, step: a[off:].reshape(rows, step)[:, :n]
        self.stored, self.value = cut(self.back, ld), cut(values, ld)
        self.base = C.to_device(self.back)
        self.grad = self.base.view((rows, n), (ld, 1), off)
        self.room = draw(kind, rng, off + rows * ldo, 0.3)[0]
        self.into = C.to_device(self.room)
        self.out = self.into.view((rows, n), (ldo, 1), off)
        self.cut_out = lambda a: cut(a, ldo)

    def check(self, norm, most, scale):
        want = self.room.copy()
        self.cut_out(want)[:] = scaled(self.kind, self.stored, self.value, norm, most, scale)
        assert np.array_equal(bits(self.into.numpy()), bits(want))
        assert np.array_equal(bits(self.base.numpy()), bits(self.back))


def run(items, scale=0.5):
    grads = C.tensor_list([t.grad for t in items])
    norm = C.gradient_norm(grads, scale, C.empty((), np.float64))
    want = norm_of([(t.kind, t.stored, t.value) for t in items], scale)
    # binary64 sums of under 2^20 terms
    assert abs(float(norm.numpy()) - want) <= 2.0**-30 * want
    held = float(norm.numpy())
    again = C.gradient_norm(grads, scale, C.empty((), np.float64))
    assert float(again.numpy()) == held
    C.clip_gradients(grads, norm, 0.25 * held, scale, [t.out for t in items])
    for t in items:
        t.check(held, 0.25 * held, scale)
    # in place: the same elements
    C.clip_gradients(grads, norm, 0.25 * held, scale)
    for t in items:
        assert np.array_equal(bits(t.grad.numpy()), bits(t.out.numpy()))


@pytest.mark.parametrize("count", [159, 160, 161, 320, 321])
def test_dense_tensors(count):
    rng = np.random.default_rng(count)
    run([Dense(rng, KINDS[i % 4]) for i in range(count)])


@pytest.mark.parametrize("dense", [0, 1, 161])
@pytest.mark.parametrize("count", [1, 63, 64, 65, 128, 130])
def test_rows_a_step_apart(count, dense):
    rng = np.random.default_rng(count + dense)
    items = [Rows(rng, KINDS[i % 4]) for i in range(count)] + [Dense(rng, KINDS[i % 4]) for i in range(dense)]
    rng.shuffle(items)
    run(items)


@pytest.mark.parametrize("kinds", [["f32"], ["bf16", "f16"], KINDS])
def test_pieces(kinds):
    """Rows of several pieces beside short ones, and more rows than a piece has
    threads."""
    rng = np.random.default_rng(9)
    sizes = [(3, 8191), (2, 8192), (3, 8193), (2, 30000), (700, 3), (5, 1), (2, 16385)]
    run([Rows(rng, kinds[i % len(kinds)], *sizes[i % 7]) for i in range(70)] + [Dense(rng, kinds[0]) for _ in range(3)])
