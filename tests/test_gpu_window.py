"""Attention with a sliding window and sinks, and its gradients, against the
plain binary64 form (block_reference): one token to long sequences, grouped
heads, cached and padded batches, rows that see nothing, hidden garbage,
strides, extreme scores, repeated and captured calls."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import (NP, Captured, check, decode, draw, encode, spans, visible, window_adjoint,
                             window_forward)

pytestmark = pytest.mark.gpu
KINDS = ["f32", "bf16", "f16"]


def bits(a):
    return np.ascontiguousarray(a).view(np.uint8)


def index(v, dtype=np.int32):
    return None if v is None else C.to_device(np.asarray(v, dtype))


def stored(kind, values):
    a = encode(kind, values)
    return a, decode(kind, a)


def run_both(kind, q, k, v, g, window, sinks, scale, lengths=None, starts=None, hidden=None):
    """Forward and gradients of stored arrays, checked. `hidden` (a pair of
    arrays k, v) takes the place of k and v on the device."""
    qv, kv, vv, gv = (decode(kind, x) for x in (q, k, v, g))
    dk_, dv_ = hidden or (k, v)
    t = [C.to_device(x) for x in (q, dk_, dv_, g)]
    where = dict(lengths=index(lengths), starts=index(starts, np.int64))
    o, lse = C.window_attention(t[0], t[1], t[2], window, sinks, scale, lse=True, **where)
    (wo, bo), (wl, bl) = window_forward(kind, qv, kv, vv, window, sinks, scale, lengths, starts)
    check(decode(kind, o.numpy()), wo, bo, "o")
    check(lse.numpy().astype(np.float64), wl, bl, "lse")
    grads = C.window_attention_adjoint(t[0], t[1], t[2], o, lse, t[3], window, sinks, scale, **where)
    ov, lv = decode(kind, o.numpy()), lse.numpy().astype(np.float64)
    want = window_adjoint(kind, qv, kv, vv, ov, lv, gv, window, sinks, scale, lengths, starts)
    for name, got, (w, bound) in zip(("dq", "dk", "dv"), grads, want):
        check(decode(kind, got.numpy()), w, bound, name)
    again = C.window_attention_adjoint(t[0], t[1], t[2], o, lse, t[3], window, sinks, scale, **where)
    for a, b in zip(grads, again):
        assert np.array_equal(bits(a.numpy()), bits(b.numpy()))
    return o, lse, grads


def operands(kind, B, H, KV, S, N, W, seed, scale=1.0):
    rng = np.random.default_rng(seed)
    return (draw(kind, rng, (B, H, S, W), scale)[0], draw(kind, rng, (B, KV, N, W))[0],
            draw(kind, rng, (B, KV, N, W))[0], draw(kind, rng, (B, H, S, W), 0.01)[0])


# batch, heads, kv heads, rows, keys, width, window, sinks, lengths, starts
CASES = [
    (1, 1, 1, 1, 1, 8, 1, 0, None, None),
    (2, 2, 1, 1, 9, 64, 4, 2, [9, 0], None),
    (1, 4, 2, 5, 5, 40, 2, 1, None, None),
    (2, 3, 3, 33, 33, 64, 1, 0, None, None),
    (1, 2, 1, 64, 64, 64, 1000, 0, None, None),
    (1, 4, 4, 127, 127, 72, 40, 3, None, None),
    (2, 4, 1, 129, 129, 128, 64, 64, None, None),
    (1, 2, 2, 200, 333, 96, 100, 5, None, None),
    (3, 6, 3, 150, 150, 96, 30, 70, [150, 97, 1], [0, 0, 0]),
    (2, 2, 1, 70, 300, 64, 128, 4, [300, 71], None),
    (2, 2, 2, 50, 40, 64, 16, 2, None, None),
    (3, 2, 1, 40, 200, 128, 33, 1, [200, 10, 130], [-5, 8, 120]),
    (1, 8, 2, 513, 513, 128, 200, 4, None, None),
    (1, 1, 1, 700, 700, 64, 65, 130, None, None),
    (4, 8, 8, 1, 700, 128, 256, 16, [700, 1, 300, 257], None),
    (2, 8, 1, 4, 1000, 96, 5000, 0, [1000, 513], None),
    (2, 16, 2, 1, 2500, 128, 600, 33, [2500, 634], None),
    (1, 2, 1, 17, 3001, 64, 900, 40, None, None),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:8])))
@pytest.mark.parametrize("kind", KINDS)
def test_forward_and_gradients(kind, case):
    B, H, KV, S, N, W, window, sinks, lengths, starts = case
    run_both(kind, *operands(kind, B, H, KV, S, N, W, S * 1000 + N), window, sinks, W ** -0.5, lengths, starts)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_any_finite_scale(kind, scale):
    run_both(kind, *operands(kind, 1, 2, 1, 70, 70, 64, 11), 20, 3, scale)


@pytest.mark.parametrize("kind", KINDS)
def test_what_lies_past_a_length_is_never_read(kind):
    """NaN in the cache past each sequence's keys, and in the rows and
    cotangents of a padded batch behind its end."""
    B, H, KV, S, N, W = 3, 4, 2, 90, 90, 64
    q, k, v, g = operands(kind, B, H, KV, S, N, W, 12)
    lengths = [90, 40, 0]
    past = np.arange(N)[None, :] >= np.array(lengths)[:, None]
    bad = encode(kind, np.full(1, np.nan))[0]
    kh, vh, qh, gh = k.copy(), v.copy(), q.copy(), g.copy()
    kh.transpose(0, 2, 1, 3)[past] = bad
    vh.transpose(0, 2, 1, 3)[past] = bad
    qh.transpose(0, 2, 1, 3)[past] = bad
    gh.transpose(0, 2, 1, 3)[past] = bad
    t = [C.to_device(x) for x in (qh, kh, vh, gh)]
    clean = run_both(kind, q, k, v, g, 30, 5, W ** -0.5, lengths, [0] * B, hidden=(kh, vh))
    where = dict(lengths=index(lengths), starts=index([0] * B))
    o, lse = C.window_attention(t[0], t[1], t[2], 30, 5, W ** -0.5, lse=True, **where)
    assert np.array_equal(bits(o.numpy()), bits(clean[0].numpy()))
    assert np.array_equal(bits(lse.numpy()), bits(clean[1].numpy()))
    for a, b in zip(C.window_attention_adjoint(t[0], t[1], t[2], o, lse, t[3], 30, 5, W ** -0.5, **where), clean[2]):
        assert np.array_equal(decode(kind, a.numpy()), decode(kind, b.numpy()))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("S,at,window,sinks", [(100, 50, 20, 3), (100, 99, 20, 3), (100, 1, 20, 0), (1, 60, 20, 3),
                                               (4, 40, 64, 1)])
def test_a_hidden_key_adds_nothing(kind, value, S, at, window, sinks):
    """One key's v is not finite: rows that do not see it are what they are
    without it, rows that do get the value's effect; the gradients of rows and
    keys that no such pair touches stay."""
    B, H, KV, N, W = 1, 2, 1, 100, 64
    q, k, v, g = operands(kind, B, H, KV, S, N, W, 13)
    vh = v.copy()
    vh[0, 0, at, 5] = encode(kind, np.full(1, value))[0]
    vis = visible(S, N, N, N - S, window, sinks)
    sees = vis[:, at]
    t = [C.to_device(x) for x in (q, k, v, vh, g)]
    o, lse = C.window_attention(t[0], t[1], t[2], window, sinks, 0.125, lse=True)
    oh, lh = C.window_attention(t[0], t[1], t[3], window, sinks, 0.125, lse=True)
    assert np.array_equal(bits(lse.numpy()), bits(lh.numpy()))
    a, b = decode(kind, o.numpy()), decode(kind, oh.numpy())
    assert np.array_equal(a[0][:, ~sees], b[0][:, ~sees])
    other = np.arange(W) != 5
    assert np.array_equal(a[..., other], b[..., other])
    hit = b[0][:, sees, 5]
    assert np.isnan(hit).all() if np.isnan(value) else (hit == value).all()
    # gradients: rows that see the key lose their dq; keys no such row sees keep dk
    g1 = C.window_attention_adjoint(t[0], t[1], t[2], o, lse, t[4], window, sinks, 0.125)
    g2 = C.window_attention_adjoint(t[0], t[1], t[3], o, lse, t[4], window, sinks, 0.125)
    (dq1, dk1, dv1), (dq2, dk2, dv2) = ([decode(kind, x.numpy()) for x in gs] for gs in (g1, g2))
    assert np.array_equal(dq1[0][:, ~sees], dq2[0][:, ~sees])
    apart = np.arange(N) != at
    assert np.array_equal(dk1[0][:, apart], dk2[0][:, apart])
    assert np.array_equal(dv1, dv2)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("which", ["k", "q", "g"])
def test_a_nan_reaches_only_its_pairs(kind, which):
    """A NaN key, query row or cotangent row: rows and keys of no pair with it
    keep their gradients."""
    B, H, KV, S, W, window, sinks, at = 1, 2, 2, 100, 64, 20, 2, 50
    q, k, v, g = operands(kind, B, H, KV, S, S, W, 14)
    bad = encode(kind, np.full(1, np.nan))[0]
    x = {"q": q.copy(), "k": k.copy(), "g": g.copy()}
    x[which][0, 0, at, 3] = bad
    t = [C.to_device(a) for a in (q, k, v, g)]
    u = [C.to_device(x["q"]), C.to_device(x["k"]), t[2], C.to_device(x["g"])]
    vis = visible(S, S, S, 0, window, sinks)
    o, lse = C.window_attention(*t[:3], window, sinks, 0.125, lse=True)
    oh, _ = C.window_attention(*u[:3], window, sinks, 0.125, lse=True)
    rows = vis[:, at] if which == "k" else np.arange(S) == at
    if which != "g":
        a, b = decode(kind, o.numpy()), decode(kind, oh.numpy())
        assert np.array_equal(a[0, 1], b[0, 1]) and np.array_equal(a[0, 0, ~rows], b[0, 0, ~rows])
        assert np.isnan(b[0, 0, rows]).all()
    keys = (vis[rows].any(0) if which == "k" else vis[at])
    g1 = C.window_attention_adjoint(*t[:3], o, lse, t[3], window, sinks, 0.125)
    g2 = C.window_attention_adjoint(*u[:3], o, lse, u[3], window, sinks, 0.125)
    for n, (a, b) in enumerate(zip(g1, g2)):
        a, b = decode(kind, a.numpy()), decode(kind, b.numpy())
        hit = rows if n == 0 else keys
        assert np.array_equal(a[0, 1], b[0, 1]), n
        assert np.array_equal(a[0, 0, ~hit], b[0, 0, ~hit]), n
    assert np.isnan(decode(kind, g2[0].numpy())[0, 0, rows]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_scores_far_apart(kind):
    """Scores of several hundred, a window whose first tiles hold far smaller
    ones than its last, and rows whose scores are all equal."""
    B, H, S, W = 1, 1, 300, 64
    q, k, v, g = operands(kind, B, H, 1, S, S, W, 15, 4.0)
    kv = decode(kind, k)
    kv[0, 0] *= np.linspace(0.01, 8, S)[:, None]
    k = encode(kind, kv)
    run_both(kind, q, k, v, g, 250, 2, 1.0)
    q[...] = encode(kind, np.zeros(1))[0]
    run_both(kind, q, k, v, g, 250, 2, 1.0)


@pytest.mark.parametrize("kind", KINDS)
def test_infinite_scores(kind):
    """A key of -inf scores weighs nothing beside finite ones; a row that sees
    only such keys, or one of +inf, is NaN as its formula is."""
    S, W = 40, 64
    q, k, v, _ = operands(kind, 1, 1, 1, S, S, W, 16)
    one = encode(kind, np.ones(1))[0]
    q[0, 0, :, 0] = one
    for value in (-np.inf, np.inf):
        kh = k.copy()
        kh[0, 0, 10, 0] = encode(kind, np.full(1, value))[0]
        o = decode(kind, C.window_attention(*(C.to_device(x) for x in (q, kh, v)), 5, 0, 0.125).numpy())[0, 0]
        (want, bound), _ = window_forward(kind, *(decode(kind, x) for x in (q, k, v)), 5, 0, 0.125)
        far = np.ones(S, bool)
        far[10:15] = False
        check(o[far], want[0, 0][far], bound[0, 0][far])
        if value > 0:
            assert np.isnan(o[10:15]).all()
        else:
            assert np.isfinite(o).all()
    alone = k.copy()
    alone[0, 0, :, 0] = encode(kind, np.full(1, -np.inf))[0]
    o = decode(kind, C.window_attention(*(C.to_device(x) for x in (q, alone, v)), 5, 0, 0.125).numpy())
    assert np.isnan(o).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [1e-7, 1.0, 3000.0])
def test_gradients_of_any_size(kind, size):
    """f16 cotangents near its least and its largest values keep their bits in
    dS; 1e-7 itself is a subnormal of two bits there, so the test scales v."""
    q, k, v, g = operands(kind, 2, 4, 2, 130, 130, 96, 17)
    v = encode(kind, decode(kind, v) * (size if size > 1 else 1))
    g = encode(kind, decode(kind, g) * (1 if size > 1 else max(size, 2e-3 if kind == "f16" else size) * 100))
    run_both(kind, q, k, v, g, 64, 4, 96 ** -0.5)


@pytest.mark.parametrize("kind", KINDS)
def test_views_of_packed_projections(kind):
    """q, k and v as views of one [batch, seq, heads + 2 kv, width] tensor from
    an odd element on, their gradients written into another, the result into
    a third; what lies between stays."""
    B, S, H, KV, W, off = 2, 75, 4, 2, 72, 3
    rng = np.random.default_rng(18)
    row = (H + 2 * KV) * W
    back, values = draw(kind, rng, off + B * S * row)
    x = values[off:].reshape(B, S, H + 2 * KV, W)
    parts = [x[:, :, a:b].transpose(0, 2, 1, 3) for a, b in ((0, H), (H, H + KV), (H + KV, H + 2 * KV))]
    t, d = C.to_device(back), C.to_device(back)

    def views(base):
        return [base.view((B, n, S, W), (S * row, W, row, 1), off + at * W)
                for at, n in ((0, H), (H, KV), (H + KV, KV))]

    guard = encode(kind, np.full(5 + B * S * H * W + 7, 9.0))
    out = C.to_device(guard)
    o = out.view((B, H, S, W), (S * H * W, W, H * W, 1), 5)
    lse = C.empty((B, H, S), np.float32)
    q, k, v = views(t)
    C.window_attention(q, k, v, 30, 2, 0.1, o, lse)
    (wo, bo), (wl, bl) = window_forward(kind, *parts, 30, 2, 0.1)
    check(decode(kind, o.numpy()), wo, bo, "o")
    check(lse.numpy().astype(np.float64), wl, bl, "lse")
    now = out.numpy()
    assert np.array_equal(bits(now[:5]), bits(guard[:5])) and np.array_equal(bits(now[-7:]), bits(guard[-7:]))
    g, gv = draw(kind, rng, (B, H, S, W), 0.01)
    dq, dk, dv = views(d)
    C.window_attention_adjoint(q, k, v, o, lse, C.to_device(g), 30, 2, 0.1, dq, dk, dv)
    want = window_adjoint(kind, *parts, decode(kind, o.numpy()), lse.numpy().astype(np.float64), gv, 30, 2, 0.1)
    for name, got, (w, bound) in zip(("dq", "dk", "dv"), (dq, dk, dv), want):
        check(decode(kind, got.numpy()), w, bound, name)
    assert np.array_equal(bits(d.numpy()[:off]), bits(back[:off]))


@pytest.mark.parametrize("kind", KINDS)
def test_keys_shared_by_the_batch(kind):
    """k and v with stride 0 over the batch (one prompt for every sequence)."""
    B, H, S, W = 3, 2, 20, 64
    q, k, v, _ = operands(kind, B, H, 1, S, S, W, 19)
    t, u = C.to_device(k[:1]), C.to_device(v[:1])
    o = C.window_attention(C.to_device(q), t.view((B, 1, S, W), (0, 0, W, 1)), u.view((B, 1, S, W), (0, 0, W, 1)), 7, 1, 0.125)
    (want, bound), _ = window_forward(kind, decode(kind, q), *(np.repeat(decode(kind, x[:1]), B, 0) for x in (k, v)), 7, 1, 0.125)
    check(decode(kind, o.numpy()), want, bound)


@pytest.mark.parametrize("dtype", [np.int32, np.int64])
def test_lengths_out_of_the_extent_are_taken_into_it(dtype):
    q, k, v, _ = operands("f32", 3, 2, 1, 1, 50, 64, 20)
    t = [C.to_device(x) for x in (q, k, v)]
    far = np.array([-3, 51, 2**31 - 1], np.int64).astype(dtype)
    got = C.window_attention(*t, 20, 1, 0.125, lengths=C.to_device(far)).numpy()
    want = C.window_attention(*t, 20, 1, 0.125, lengths=index([0, 50, 50])).numpy()
    assert np.array_equal(got, want) and not got[0].any()
    # every second of a longer list
    pairs = C.to_device(np.array([10, -1, 20, -1, 30, -1], dtype)).view((3,), (2,))
    got = C.window_attention(*t, 20, 1, 0.125, lengths=pairs).numpy()
    assert np.array_equal(got, C.window_attention(*t, 20, 1, 0.125, lengths=index([10, 20, 30])).numpy())


@pytest.mark.parametrize("shape", [(0, 2, 1, 5, 5), (2, 2, 1, 0, 5), (2, 2, 1, 5, 0), (2, 0, 0, 5, 5)])
def test_empty_extents(shape):
    B, H, KV, S, N = shape
    q, k = C.to_device(np.ones((B, H, S, 64), np.float32)), C.empty((B, KV, N, 64), np.float32)
    o, lse = C.window_attention(q, k, k, 3, 1, 0.125, lse=True)
    assert not o.numpy().any() and (lse.numpy() == -np.inf).all()
    mark = [C.to_device(np.full(x.shape, 7, np.float32)) for x in (q, k, k)]
    C.window_attention_adjoint(q, k, k, o, lse, q, 3, 1, 0.125, *mark)
    assert not any(m.numpy().any() for m in mark)


def test_a_chunk_and_single_tokens_are_the_prompts_rows():
    """A prompt at once, in two chunks over a cache and token by token: each
    row within both bounds of the same formula."""
    kind, H, KV, S, W, window, sinks = "bf16", 8, 2, 150, 128, 60, 4
    q, k, v, _ = operands(kind, 1, H, KV, S, S, W, 21)
    tk, tv = C.to_device(k), C.to_device(v)
    (want, bound), _ = window_forward(kind, *(decode(kind, x) for x in (q, k, v)), window, sinks, 0.09)
    for step in (S, 83, 1):
        for at in range(0, S, step):
            n = min(step, S - at)
            part = C.to_device(np.ascontiguousarray(q[:, :, at:at + n]))
            o = C.window_attention(part, tk, tv, window, sinks, 0.09, lengths=index([at + n]))
            check(decode(kind, o.numpy()), want[:, :, at:at + n], bound[:, :, at:at + n], (step, at))


def test_gradients_against_differences():
    """Directional central differences of the binary64 formula (h = 1e-5: their
    own error is far below the binary32 bound that is allowed beside it)."""
    kind, B, H, KV, S, W, window, sinks, scale = "f32", 1, 2, 1, 45, 64, 12, 3, 0.2
    arrays = operands(kind, B, H, KV, S, S, W, 22)
    q, k, v, g = (a.astype(np.float64) for a in arrays)
    t = [C.to_device(a) for a in arrays]
    o, lse = C.window_attention(*t[:3], window, sinks, scale, lse=True)
    grads = C.window_attention_adjoint(*t[:3], o, lse, t[3], window, sinks, scale)
    want = window_adjoint(kind, q, k, v, o.numpy().astype(np.float64), lse.numpy().astype(np.float64), g, window, sinks, scale)
    rng = np.random.default_rng(23)
    for n in range(3):
        way = rng.standard_normal((q, k, v)[n].shape)

        def loss(h):
            x = [q, k, v]
            x[n] = x[n] + h * way
            return (window_forward(kind, *x, window, sinks, scale)[0][0] * g).sum()

        diff = (loss(1e-5) - loss(-1e-5)) / 2e-5
        got = (grads[n].numpy().astype(np.float64) * way).sum()
        # o and lse are the rounded ones: their effect on dS counts beside the bound
        slack = (want[n][1] * np.abs(way)).sum() + 64 * 2.0**-24 * (np.abs(want[n][0]) * np.abs(way)).sum()
        assert abs(got - diff) <= slack + 1e-8, (n, got, diff, slack)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("S,N", [(1, 2000), (200, 200)])
def test_captured_calls_replay(kind, S, N):
    """Two captured calls replayed in turn, eager calls between the replays."""
    B, H, KV, W, window, sinks = 2, 8, 2, 128, 500, 4
    calls = []
    for seed in (24, 25):
        t = [C.to_device(x) for x in operands(kind, B, H, KV, S, N, W, seed)]
        o, lse = C.window_attention(*t[:3], window, sinks, 0.09, lse=True)
        want = [bits(x.numpy()) for x in (o, lse, *C.window_attention_adjoint(*t[:3], o, lse, t[3], window, sinks, 0.09))]
        out = [C.empty(x.shape, x.dtype) for x in (o, lse, t[0], t[1], t[1])]
        C.synchronize()

        def both():
            C.window_attention(*t[:3], window, sinks, 0.09, out[0], out[1])
            C.window_attention_adjoint(*t[:3], out[0], out[1], t[3], window, sinks, 0.09, *out[2:])

        calls.append((t, want, out, Captured(both)))
    for _ in range(3):
        for t, want, out, graph in calls:
            graph.launch()
        for t, want, out, graph in calls:
            o, lse = C.window_attention(*t[:3], window, sinks, 0.09, lse=True)
            eager = [o, lse, *C.window_attention_adjoint(*t[:3], o, lse, t[3], window, sinks, 0.09)]
            C.synchronize()
            for a, b, w in zip(out, eager, want):
                assert np.array_equal(bits(a.numpy()), w) and np.array_equal(bits(b.numpy()), w)


@pytest.mark.parametrize("kind", KINDS)
def test_numbers_at_their_limits(kind):
    """A window and sinks past every key, and first positions past both ends
    of any sequence."""
    q, k, v, g = operands(kind, 2, 2, 1, 20, 20, 64, 26)
    t = [C.to_device(x) for x in (q, k, v, g)]
    plain = C.window_attention(*t[:3], 20, 0, 0.125).numpy()
    for window, sinks in ((2**62, 0), (1, 2**40), (2**62, 2**62)):
        assert np.array_equal(bits(C.window_attention(*t[:3], window, sinks, 0.125).numpy()), bits(plain))
    far = index([-2**62, 2**62], np.int64)
    o, lse = C.window_attention(*t[:3], 5, 1, 0.125, lse=True, starts=far)
    assert not decode(kind, o.numpy()).any() and (lse.numpy() == -np.inf).all()
    for d in C.window_attention_adjoint(*t[:3], o, lse, t[3], 5, 1, 0.125, starts=far):
        assert not decode(kind, d.numpy()).any()


@pytest.mark.parametrize("S,N", [(1, 3), (3, 3)])
def test_rows_four_gigabytes_apart(S, N):
    """Keys, values and gradients whose rows lie 2^31 elements apart (offsets
    past 32 bits), in one storage: results are those of dense operands. Rotary
    positions of 0 (a turn by nothing) write the rows where they lie."""
    kind, W, far = "bf16", 64, 2**31
    q, k, v, g = operands(kind, 1, 1, 1, S, N, W, 27)
    base = C.empty((2 * far + 4 * W,), np.uint16)
    ks, vs, dk, dv = (base.view((1, 1, N, W), (3 * far, 3 * far, far, 1), at * W) for at in range(4))
    none, freqs = C.to_device(np.zeros((1, 1, N), np.int32)), C.to_device(np.ones(W // 2))
    for x, to in ((k, ks), (v, vs)):
        C.rotary(C.to_device(x), none, freqs, [W // 2], out=to)
        assert np.array_equal(to.numpy(), x)
    t = [C.to_device(x) for x in (q, k, v, g)]
    o, lse = C.window_attention(*t[:3], 2, 1, 0.125, lse=True)
    of, lf = C.window_attention(t[0], ks, vs, 2, 1, 0.125, lse=True)
    assert np.array_equal(of.numpy(), o.numpy()) and np.array_equal(lf.numpy(), lse.numpy())
    want = C.window_attention_adjoint(*t[:3], o, lse, t[3], 2, 1, 0.125)
    got = C.window_attention_adjoint(t[0], ks, vs, o, lse, t[3], 2, 1, 0.125, None, dk, dv)
    for a, b in zip(got, want):
        assert np.array_equal(a.numpy(), b.numpy())
    # the same rows through the norm, in place
    one, zero = C.to_device(encode(kind, np.ones(W))), C.to_device(encode(kind, np.zeros(W)))
    rows, dense = base.view((N, W), (far, 1)), C.to_device(k.reshape(N, W))
    y, mean, rstd = C.layer_norm_stats(dense, one, zero, 1e-5)
    grad = C.layer_norm_adjoint(dense, one, mean, rstd, dense)[0].numpy()
    C.layer_norm_adjoint(rows, one, mean, rstd, rows, dx=base.view((N, W), (far, 1), 2 * W), want_weights=False)
    assert np.array_equal(base.view((N, W), (far, 1), 2 * W).numpy(), grad)
    C.layer_norm_stats(rows, one, zero, 1e-5, y=rows)
    assert np.array_equal(rows.numpy(), y.numpy())


def test_more_rows_than_a_launch_has_workgroups():
    # 2^24 rows of narrow heads over few keys, nearly all of them ahead of the sequence
    H, S, N, W = 16, 1 << 20, 64, 8
    q, k, v, _ = operands("f32", 1, H, H, N, N, W, 31)
    device = C.empty((1, H, S, W), np.float32)
    last = device.view((1, H, N, W), (H * S * W, S * W, W, 1), (S - N) * W)
    none, freqs = C.to_device(np.zeros((1, 1, N), np.int32)), C.to_device(np.ones(W // 2))
    C.rotary(C.to_device(q), none, freqs, [W // 2], out=last)
    ks, vs = C.to_device(k), C.to_device(v)
    o = C.window_attention(device, ks, vs, N, 0, 0.5)
    want, bound = window_forward("f32", q.astype(np.float64), k.astype(np.float64), v.astype(np.float64), N, 0, 0.5)[0]
    check(o.view((1, H, N, W), (H * S * W, S * W, W, 1), (S - N) * W).numpy().astype(np.float64), want, bound, "o")
    assert not o.view((1, H, N, W), (H * S * W, S * W, W, 1), (S - 2 * N) * W).numpy().any()
