"""The block operators at sizes that take the launch shapes of large calls:
prompts whose rows go whole, in every type and held width, with window edges,
sinks and padding; heads dealt in chunks over the XCDs; rotary threads that
turn several heads; tokens over more splits than the join reads at once; float16
gradients that need the power of two they are held under."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import check, decode, draw, encode, rotary, visible, window_adjoint, window_forward

pytestmark = pytest.mark.gpu
KINDS = ["f32", "bf16", "f16"]


def operands(kind, B, H, KV, S, N, W, seed, scale=1.0):
    rng = np.random.default_rng(seed)
    return (draw(kind, rng, (B, H, S, W), scale)[0], draw(kind, rng, (B, KV, N, W))[0],
            draw(kind, rng, (B, KV, N, W))[0], draw(kind, rng, (B, H, S, W), 0.01)[0])


def index(v):
    return None if v is None else C.to_device(np.asarray(v, np.int64))


def attended(kind, arrays, window, sinks, scale, lengths=None, starts=None, some=None, gradients=False):
    """Forward (and gradients), checked over the sequences `some`."""
    q, k, v, g = arrays
    t = [C.to_device(x) for x in arrays]
    where = dict(lengths=index(lengths), starts=index(starts))
    o, lse = C.window_attention(*t[:3], window, sinks, scale, lse=True, **where)
    on, ln = o.numpy(), lse.numpy()
    some = range(q.shape[0]) if some is None else some
    for b in some:
        part = [decode(kind, x[b:b + 1]) for x in (q, k, v)]
        place = [None if x is None else x[b:b + 1] for x in (lengths, starts)]
        (wo, bo), (wl, bl) = window_forward(kind, *part, window, sinks, scale, *place)
        check(decode(kind, on[b:b + 1]), wo, bo, ("o", b))
        check(ln[b:b + 1].astype(np.float64), wl, bl, ("lse", b))
    if not gradients:
        return
    got = [x.numpy() for x in C.window_attention_adjoint(*t[:3], o, lse, t[3], window, sinks, scale, **where)]
    for b in some:
        part = [decode(kind, x[b:b + 1]) for x in (q, k, v, on, g)]
        place = [None if x is None else x[b:b + 1] for x in (lengths, starts)]
        want = window_adjoint(kind, *part[:4], ln[b:b + 1].astype(np.float64), part[4], window, sinks, scale, *place)
        for name, a, (w, bound) in zip(("dq", "dk", "dv"), got, want):
            check(decode(kind, a[b:b + 1]), w, bound, (name, b))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("W", [64, 72, 96, 128])
@pytest.mark.parametrize("window,sinks,padded", [(90, 5, False), (33, 70, True), (300, 0, True), (1, 0, False)])
def test_prompts_whose_rows_go_whole(kind, W, window, sinks, padded):
    """128 heads in all: no launch of these rows splits their keys, binary32
    neither, whose halves of a tile that a wave does not see are left out."""
    B, H, KV, S = 8, 16, 8, 300
    lengths = [300, 299, 257, 130, 65, 64, 1, 0] if padded else None
    attended(kind, operands(kind, B, H, KV, S, S, W, W + window), window, sinks, W ** -0.5, lengths,
             [0] * B if padded else None, some=range(0, B, 3) if not padded else (0, 2, 3, 5, 6, 7))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sign", [1, -1])
def test_a_maximum_that_moves_far(kind, sign):
    """Rows that go whole over keys whose scores grow (and fall) from tile to
    tile by far more than the slack within which results are not rescaled."""
    B, H, S, W = 8, 16, 320, 64
    q, k, v, g = operands(kind, B, H, 8, S, S, W, 41)
    qv, kv = decode(kind, q), decode(kind, k)
    qv[..., 0], kv[..., 0] = 4.0, np.linspace(-20, 20, S) * sign
    attended(kind, (encode(kind, qv), encode(kind, kv), v, g), 250, 3, 1.0, some=(0, 5))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_hidden_values_of_rows_that_go_whole(kind, value):
    """One key's v is not finite: rows that do not see it keep every bit."""
    B, H, KV, S, W, window, sinks = 8, 16, 8, 300, 64, 40, 3
    q, k, v, _ = operands(kind, B, H, KV, S, S, W, 42)
    t = [C.to_device(x) for x in (q, k, v)]
    plain = C.window_attention(*t, window, sinks, 0.125).numpy()
    vh = v.copy()
    for at in (100, 290):
        vh[:, ::2, at, 9] = encode(kind, np.full(1, value))[0]
    o = C.window_attention(t[0], t[1], C.to_device(vh), window, sinks, 0.125).numpy()
    vis = visible(S, S, S, 0, window, sinks)
    sees = vis[:, 100] | vis[:, 290]
    assert np.array_equal(o[:, :, ~sees], plain[:, :, ~sees])
    other = np.arange(W) != 9
    assert np.array_equal(o[..., other], plain[..., other])
    hit = decode(kind, np.ascontiguousarray(o[:, :, sees, 9])).reshape(B, KV, H // KV, -1)
    assert (np.isnan(hit[:, ::2]) if np.isnan(value) else hit[:, ::2] == value).all()
    assert np.isfinite(hit[:, 1::2]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_chunks_of_tiles_and_several_heads(kind):
    """Eight row tiles of eight key heads, two neighbouring tiles to a chunk,
    four query heads dealt with each; the last tile is not whole."""
    attended(kind, operands(kind, 2, 16, 4, 1000, 1000, 64, 43), 300, 4, 0.125, some=(1,), gradients=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,KV,N,W,window", [(16, 4, 4096, 128, 4096), (2, 1, 16384, 64, 16384), (4, 1, 16000, 40, 9000)])
def test_one_token_over_many_splits(kind, H, KV, N, W, window):
    """128, 512 and about 280 splits: more than a thread's first parts, and more
    statistics than the join has threads."""
    attended(kind, operands(kind, 1, H, KV, 1, N, W, 44), window, 4, W ** -0.5)


@pytest.mark.parametrize("kind", ["f32", "f64", "bf16", "f16"])
@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
@pytest.mark.parametrize("inside", [False, True], ids=["heads-apart", "heads-inside"])
@pytest.mark.parametrize("heads,kv", [(16, 4), (13, 5)])
def test_rotary_threads_that_turn_several_heads(kind, pairing, inside, heads, kv):
    """8192 tokens: a thread keeps its angles for up to eight heads (of four
    neighbours each where they lie inside the sequence axis), four loaded at a
    time. Every result in place too."""
    B, S, W, sections = 2, 4096, 64, [12, 16]
    rng = np.random.default_rng(45)
    pos, freqs = rng.integers(0, 100000, (2, B, S)).astype(np.int32), 10000.0 ** (-np.arange(28) / 28)
    dp, df = C.to_device(pos), C.to_device(freqs)
    arrays = [draw(kind, rng, (B, S, h, W) if inside else (B, h, S, W)) for h in (heads, kv)]
    t, out = [C.to_device(a) for a, _ in arrays], [C.empty(a.shape, a.dtype) for a, _ in arrays]

    def by_head(x, h):
        return x.view((B, h, S, W), (S * h * W, W, h * W, 1)) if inside else x

    xs, ys = ([by_head(x, h) for x, h in zip(p, (heads, kv))] for p in (t, out))
    C.rotary(xs, dp, df, sections, pairing, out=ys)
    for (_, x), y in zip(arrays, out):
        x = x.transpose(0, 2, 1, 3) if inside else x
        got = decode(kind, y.numpy()).transpose(0, 2, 1, 3) if inside else decode(kind, y.numpy())
        check(got[:, :, ::5], *(r[:, :, ::5] for r in rotary(kind, x, pos, freqs, sections, pairing)), "turned")
    want = [y.numpy() for y in out]
    C.rotary(xs, dp, df, sections, pairing, out=xs)
    for x, w in zip(t, want):
        assert np.array_equal(x.numpy().view(np.uint8), w.view(np.uint8))


@pytest.mark.parametrize("which", ["large", "small-dq", "small-dk"])
def test_float16_score_gradients_past_the_type(which):
    """dS past 65504, and below half of float16's least subnormal, where dq and
    dk themselves are ordinary numbers: rounded to float16 as they are, they
    would miss the bound (asserted here), so the scale has to work."""
    B, H, KV, S, W, window, sinks = 1, 2, 1, 150, 64, 40, 3
    rng = np.random.default_rng(46)
    sizes = {"large": (1e-3, 1e-3, 5000.0, 100.0), "small-dq": (1e-4, 5000.0, 1e-2, 2e-6),
             "small-dk": (5000.0, 1e-4, 1e-2, 2e-6)}[which]
    q, k, v, g = (draw("f16", rng, (B, h, S, W), s)[0] for h, s in zip((H, KV, KV, H), sizes))
    scale = 0.5
    Q, K, V, G = (decode("f16", x) for x in (q, k, v, g))
    (o, _), (lse, _) = window_forward("f16", Q, K, V, window, sinks, scale)
    # what rounding dS as it stands would leave of the first head's gradients
    vis = visible(S, S, S, 0, window, sinks)
    p = np.where(vis, np.exp(np.where(vis, Q[0, 0] @ K[0, 0].T * scale - lse[0, 0][:, None], 0)), 0)
    ds = p * (G[0, 0] @ V[0, 0].T - (G[0, 0] * o[0, 0]).sum(1, keepdims=True))
    with np.errstate(over="ignore", invalid="ignore"):
        rough = ds.astype(np.float16).astype(np.float64)
        (dq, bq), (dk, bk), _ = window_adjoint("f16", Q[:, :1], K, V, o[:, :1], lse[:, :1], G[:, :1], window, sinks, scale)
        of_q, of_k = scale * rough @ K[0, 0] - dq[0, 0], scale * rough.T @ Q[0, 0] - dk[0, 0]
        if which == "large":
            assert np.abs(ds).max() > 65504 and np.isinf(rough).any()
            assert not (np.abs(of_q) <= bq[0, 0]).all() and not (np.abs(of_k) <= bk[0, 0]).all()
        else:
            assert np.median(np.abs(ds[vis])) < 2.0**-25
            assert not (np.abs(of_q if which == "small-dq" else of_k) <= (bq if which == "small-dq" else bk)[0, 0]).all()
    result = dq if which != "small-dk" else dk
    assert 2.0**-14 < np.abs(result).max() < 60000 and np.abs(dk).max() < 60000 and np.abs(dq).max() < 60000
    attended("f16", (q, k, v, g), window, sinks, scale, gradients=True)


def test_log_sums_not_asked_for():
    t = [C.to_device(x) for x in operands("f32", 1, 2, 1, 3, 9, 16, 47)[:3]]
    want = C.window_attention(*t, 4, 1, 0.25).numpy()
    assert np.array_equal(C.window_attention(*t, 4, 1, 0.25, lse=False).numpy(), want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("score", [60.0, np.inf])
@pytest.mark.parametrize("shape", [(8, 16, 8, 300), (1, 2, 1, 40)], ids=["whole", "split"])
def test_no_bit_of_a_row_depends_on_scores_it_does_not_have(kind, score, shape):
    """One key scores far above all others: rows that do not see it, beside
    rows that do, keep every bit they have without it."""
    B, H, KV, S = shape
    W, window, sinks, at = 64, 100, 2, S - 20
    q, k, v, _ = operands(kind, B, H, KV, S, S, W, 48)
    q[..., 0] = encode(kind, np.ones(1))[0]
    far = k.copy()
    far[:, :, at, 0] = encode(kind, np.full(1, score / 0.125))[0]
    sees = visible(S, S, S, 0, window, sinks)[:, at]
    t = [C.to_device(x) for x in (q, k, v)]
    o, lse = (x.numpy() for x in C.window_attention(*t, window, sinks, 0.125, lse=True))
    p, lsf = (x.numpy() for x in C.window_attention(t[0], C.to_device(far), t[2], window, sinks, 0.125, lse=True))
    assert np.array_equal(o[:, :, ~sees], p[:, :, ~sees]) and np.array_equal(lse[:, :, ~sees], lsf[:, :, ~sees])
    assert not np.array_equal(o[:, :, sees], p[:, :, sees])
