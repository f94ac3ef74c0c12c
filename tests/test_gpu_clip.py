"""The norm of many gradients together and their clipping against binary64:
every dtype in one call, more tensors than a launch's table, empty and
one-element tensors, layouts, in place and into a flat buffer, limits, graph
replays."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import NP, Captured, decode, draw, encode

pytestmark = pytest.mark.gpu
KINDS = ["f32", "bf16", "f16", "f64"]
SHAPES = [(1,), (3,), (0, 5), (7, 9), (256,), (8191,), (64, 1024), (16385, 3), (), (5, 1, 4099), (300000,)]


def gradients(seed, shapes=SHAPES, kinds=KINDS, scale=0.3):
    rng = np.random.default_rng(seed)
    out = []
    for i, shape in enumerate(shapes):
        kind = kinds[i % len(kinds)]
        out.append((kind, *draw(kind, rng, shape, scale)))
    return out


def norm_of(gs, scale=1.0):
    return scale * np.sqrt(sum((v * v).sum() for _, _, v in gs))


def scaled(kind, stored, value, norm, most, scale):
    """The kernel's own arithmetic: the factor in binary64; a wide product
    rounded once, a 16-bit one formed in binary32."""
    factor = scale * (most / norm) if norm > most else scale
    with np.errstate(invalid="ignore", over="ignore"):
        if kind in ("f32", "f64"):
            return (value * factor).astype(NP[kind])
        return encode(kind, (value.astype(np.float32) * np.float32(factor)).astype(np.float64))


@pytest.mark.parametrize("scale", [1.0, 1 / 1024])
@pytest.mark.parametrize("most", [0.125, 5.0, 1e6])
@pytest.mark.parametrize("wide", [np.float32, np.float64])
def test_norm_and_clipping(scale, most, wide):
    gs = gradients(3)
    dev = [C.to_device(s) for _, s, _ in gs]
    norm = C.gradient_norm(dev, scale, C.empty((), wide))
    want = norm_of(gs, scale)
    # binary64 sums of under 2^20 terms, then the one rounding of the result
    assert abs(float(norm.numpy()) - want) <= (2.0**-30 + (2.0**-24 if wide == np.float32 else 0)) * want
    held = float(norm.numpy())
    out = C.clip_gradients(dev, norm, most, scale, [C.empty(t.shape, t.dtype) for t in dev])
    for (kind, s, v), o, d in zip(gs, out, dev):
        assert np.array_equal(o.numpy().ravel(), scaled(kind, s, v, held, most, scale).ravel()), kind
        assert np.array_equal(d.numpy().ravel(), s.ravel())  # a () array travels as (1,)
    C.clip_gradients(dev, norm, most, scale)
    for d, o in zip(dev, out):
        assert np.array_equal(d.numpy(), o.numpy())


@pytest.mark.parametrize("count", [0, 1, 63, 64, 65, 131, 700])
def test_many_tensors(count):
    rng = np.random.default_rng(count)
    gs = gradients(count, [(int(n),) for n in rng.integers(0, 3000, count)])
    dev = C.tensor_list([C.to_device(s) for _, s, _ in gs])
    norm = C.gradient_norm(dev, 1.0)
    want = norm_of(gs)
    assert abs(float(norm.numpy()) - want) <= (2.0**-24 + 2.0**-30) * want
    held = float(norm.numpy())
    C.clip_gradients(dev, norm, 0.5 * held + 1e-9)
    for (kind, s, v), d in zip(gs, dev):
        assert np.array_equal(d.numpy(), scaled(kind, s, v, held, 0.5 * held + 1e-9, 1.0))


def test_layouts_and_a_flat_buffer():
    """Transposed, row-strided and permuted gradients; results in the same order
    of axes as views of one buffer from odd elements on, whose other elements
    stay."""
    rng = np.random.default_rng(1)
    base, val = draw("bf16", rng, (40, 50, 60))
    t = C.to_device(base)
    views = [(t.view((60, 50), (1, 60), 0), val[0].T), (t.view((30, 17), (60, 1), 3 * 3000 + 5), val[3][:30, 5:22]),
             (t.view((50, 4, 60), (60, 3000, 1), 10 * 3000), val[10:14].transpose(1, 0, 2)),
             (t.view((25, 8), (120, 1), 20 * 3000), val[20].reshape(25, 120)[:, :8])]
    grads = [v for v, _ in views]
    want = np.sqrt(sum((v * v).sum() for _, v in views))
    norm = C.gradient_norm(grads)
    held = float(norm.numpy())
    assert abs(held - want) <= (2.0**-24 + 2.0**-30) * want
    back, _ = draw("bf16", rng, 20001)
    flat = C.to_device(back)
    at, outs = 7, []
    expect = back.copy()
    for v, values in views:
        order = sorted(range(len(v.shape)), key=lambda a: -v.strides[a])
        strides = [0] * len(order)
        for i, a in enumerate(order):
            strides[a] = int(np.prod([v.shape[b] for b in order[i + 1:]]))
        outs.append(flat.view(v.shape, strides, at))
        expect[at:at + values.size] = scaled("bf16", None, values.transpose(order), held, 1.0, 1.0).ravel()
        at += values.size + 3
    C.clip_gradients(grads, norm, 1.0, 1.0, outs)
    assert np.array_equal(flat.numpy(), expect)
    assert np.array_equal(t.numpy(), base)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_special_values(kind, value):
    """An infinite norm makes the factor 0 (and 0 times the infinity a NaN), a
    NaN norm leaves the scale."""
    v = np.linspace(-1, 1, 1000)
    v[17] = value
    s = encode(kind, v)
    t = C.to_device(s)
    norm = C.gradient_norm([t])
    got = float(norm.numpy())
    assert np.isnan(got) if np.isnan(value) else got == np.inf
    out = list(C.clip_gradients([t], norm, 1.0, 0.5, [C.empty(t.shape, t.dtype)]))[0]
    out = decode(kind, out.numpy())
    with np.errstate(invalid="ignore"):
        want = decode(kind, s) * (0.5 if np.isnan(value) else 0.0)
    assert np.array_equal(np.isnan(out), np.isnan(want))
    ok = ~np.isnan(want)
    assert (np.abs(out[ok] - want[ok]) <= 2.0**-8 * np.abs(want[ok])).all()


def test_large_values_do_not_overflow():
    """Gradients whose squares pass binary32: 2^100 each."""
    t = C.to_device(np.full(4096, 2.0**100, np.float32))
    assert float(C.gradient_norm([t]).numpy()) == 2.0**106
    small = C.to_device(np.full(4096, 2.0**-140, np.float32))
    assert float(C.gradient_norm([small]).numpy()) == np.float32(2.0**-134)


def test_the_same_gradient_twice_counts_twice():
    s = np.full(100, 3.0, np.float32)
    t = C.to_device(s)
    assert float(C.gradient_norm([t, t]).numpy()) == np.float32(np.sqrt(1800.0))


def test_captured_steps_replay():
    """Two captured norm-and-clip steps replayed in turn with eager ones of the
    same size between them."""
    calls = []
    for seed in (1, 2):
        gs = gradients(seed)
        dev = C.tensor_list([C.to_device(s) for _, s, _ in gs])
        norm, out = C.empty((), np.float32), C.tensor_list([C.empty(t.shape, t.dtype) for t in dev])

        def step(dev=dev, norm=norm, out=out):
            C.gradient_norm(dev, 0.5, norm)
            C.clip_gradients(dev, norm, 0.25, 0.5, out)

        step()
        want = [t.numpy().copy() for t in (norm, *out)]
        C.synchronize()
        calls.append((step, dev, norm, out, want, Captured(step)))
    for _ in range(3):
        for *_, graph in calls:
            graph.launch()
        for step, dev, norm, out, want, graph in calls:
            C.gradient_norm(dev)
            C.synchronize()
            assert all(np.array_equal(t.numpy(), w, equal_nan=True) for t, w in zip((norm, *out), want))


@pytest.mark.parametrize("kind,value,norm,most,scale", [
    ("bf16", 2.0**126, 2.0**127, 1e-7, 1.0),     # factor 5.9e-46, under binary32's smallest
    ("bf16", 1.5 * 2.0**120, 1e38, 1e-6, 1.0),   # factor 1e-44, a subnormal of three bits
    ("f16", 2.0**15, 1e45, 3e4, 0.75),           # the result underflows to 0
    ("bf16", 2.0**-120, 1.0, 2.0, 2.0**140),     # factor above binary32's largest
])
def test_factors_outside_binary32(kind, value, norm, most, scale):
    """A 16-bit gradient times a factor that no normal binary32 number holds: the
    binary64 product rounded to binary32 and to the type, 2^-24 + 2^-8 (bf16)
    relative and half the type's smallest number."""
    s = encode(kind, value * np.linspace(-1, 1, 1001))
    t = C.to_device(s)
    at = C.to_device(np.full((), norm, np.float64))
    out = decode(kind, list(C.clip_gradients([t], at, most, scale, [C.empty(t.shape, t.dtype)]))[0].numpy())
    want = decode(kind, s) * (scale * (most / norm) if norm > most else scale)
    assert (np.abs(out - want) <= (2.0**-8 + 2.0**-23) * np.abs(want) + (2.0**-134 if kind == "bf16" else 2.0**-25)).all()
