"""Norm, positions and windowed attention together, as a block's attention
half uses them: layer norm, one packed q/k/v product, rotary positions in
place, attention with a window and sinks over views of the packed result, and
all of it backwards, against binary64; and the same block serving, a prompt and
then token by token over a cache."""
import numpy as np
import pytest

import chelis_amd as C
from block_reference import decode, draw, encode, rotary, visible

pytestmark = pytest.mark.gpu
EPS = 1e-5


def _forward(x, gamma, w, pos, freqs, sections, B, S, H, KV, W, window, sinks, scale):
    mean = x.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + EPS)
    hat = (x - mean) * rstd
    y = hat * gamma[0] + gamma[1]
    qkv = (y @ w).reshape(B, S, H + 2 * KV, W).transpose(0, 2, 1, 3)
    q, _ = rotary("f64", qkv[:, :H], pos, freqs, sections, "halves")
    k, _ = rotary("f64", qkv[:, H:H + KV], pos, freqs, sections, "halves")
    v = qkv[:, H + KV:]
    vis = visible(S, S, S, 0, window, sinks)
    s = np.where(vis, (q @ np.repeat(k, H // KV, 1).swapaxes(2, 3)) * scale, -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return hat, rstd, y, q, k, v, p, p @ np.repeat(v, H // KV, 1)


def _backward(g, hat, rstd, y, q, k, v, p, o, gamma, w, pos, freqs, sections, H, KV, W, scale):
    B, _, S, _ = q.shape
    G = H // KV
    kk, vv = np.repeat(k, G, 1), np.repeat(v, G, 1)
    ds = p * (g @ vv.swapaxes(2, 3) - (g * o).sum(-1, keepdims=True)) * scale
    dq, dk, dv = ds @ kk, ds.swapaxes(2, 3) @ q, p.swapaxes(2, 3) @ g
    dk, dv = (t.reshape(B, KV, G, S, W).sum(2) for t in (dk, dv))
    dq, _ = rotary("f64", dq, pos, freqs, sections, "halves", -1.0)
    dk, _ = rotary("f64", dk, pos, freqs, sections, "halves", -1.0)
    dqkv = np.concatenate([dq, dk, dv], 1).transpose(0, 2, 1, 3).reshape(B * S, -1)
    dw, dy = y.reshape(B * S, -1).T @ dqkv, (dqkv @ w.T).reshape(y.shape)
    gg = dy * gamma[0]
    dx = rstd * (gg - gg.mean(-1, keepdims=True) - hat * (gg * hat).mean(-1, keepdims=True))
    return dx, (dy * hat).sum((0, 1)), dy.sum((0, 1)), dw


@pytest.mark.parametrize("B,S,M,H,KV,W,window,sinks", [(2, 75, 96, 4, 2, 64, 20, 3), (1, 200, 128, 2, 1, 72, 64, 1)])
def test_forward_and_backward(B, S, M, H, KV, W, window, sinks):
    """Binary32 throughout. The longest chain of sums here is a few hundred
    terms deep at every one of six stages, each a relative half step of its
    magnitudes; a mistake in a formula is of the results' own size. Bar: 2^-24
    times 4096 of each result's largest value."""
    kind, N = "f32", (H + 2 * KV) * W
    rng = np.random.default_rng(S)
    x, w = draw(kind, rng, (B, S, M))[0], draw(kind, rng, (M, N), M ** -0.5)[0]
    gamma, beta, g = draw(kind, rng, M, 0.1, 1.0)[0], draw(kind, rng, M, 0.1)[0], draw(kind, rng, (B, H, S, W), 0.1)[0]
    sections = [W // 4, W // 2 - W // 4]
    pos, freqs = rng.integers(0, 1000, (2, B, S)).astype(np.int32), 10000.0 ** (-np.arange(W // 2) / (W // 2))
    scale = W ** -0.5
    dx, dw_, dgm, dbt, dg, dp, df = (C.to_device(t) for t in (x, w, gamma, beta, g, pos, freqs))

    y, mean, rstd = C.layer_norm_stats(dx, dgm, dbt, EPS)
    y2 = y.view((B * S, M), (M, 1))
    qkv = C.matmul(y2, dw_)

    def parts(t):
        return [t.view((B, n, S, W), (S * N, W, N, 1), at * W) for at, n in ((0, H), (H, KV), (H + KV, KV))]

    q, k, v = parts(qkv)
    C.rotary([q, k], dp, df, sections, "halves", out=[q, k])
    o, lse = C.window_attention(q, k, v, window, sinks, scale, lse=True)
    dqkv = C.empty((B * S, N), np.float32)
    gq, gk, gv = parts(dqkv)
    C.window_attention_adjoint(q, k, v, o, lse, dg, window, sinks, scale, gq, gk, gv)
    C.rotary_adjoint([gq, gk], dp, df, sections, "halves", out=[gq, gk])
    dW = C.matmul(y2.base.view((M, B * S), (1, M)), dqkv)
    dy = C.matmul(dqkv, dw_.view((N, M), (1, N)))
    got = C.layer_norm_adjoint(dx, dgm, mean, rstd, dy.view((B, S, M), (S * M, M, 1)))

    r = [t.astype(np.float64) for t in (x, w, gamma, beta, g)]
    f = _forward(r[0], (r[2], r[3]), r[1], pos, freqs, sections, B, S, H, KV, W, window, sinks, scale)
    want = _backward(r[4], *f, (r[2], r[3]), r[1], pos, freqs, sections, H, KV, W, scale)
    for name, a, b in [("o", o.numpy(), f[-1])] + list(zip(("dx", "dgamma", "dbeta", "dw"), [t.numpy() for t in (*got, dW)], want)):
        assert np.abs(a - b).max() <= 2.0**-12 * np.abs(b).max(), (name, np.abs(a - b).max(), np.abs(b).max())


def test_serving_a_prompt_and_then_tokens():
    """bf16: a prompt fills the cache (keys turned to their positions), then
    each token is turned, written behind it and attends over it. Every result
    is that of the whole sequence at once: either one is off by at most a
    rounding of each weight and one of the result (the binary32 terms are far
    below), so the two differ by at most four half steps of the largest value."""
    kind, H, KV, W, P, S, CAP, window, sinks = "bf16", 8, 2, 128, 60, 70, 96, 32, 4
    rng = np.random.default_rng(5)
    q, k, v = (draw(kind, rng, (1, n, S, W))[0] for n in (H, KV, KV))
    freqs = C.to_device(10000.0 ** (-np.arange(W // 2) / (W // 2)))
    pos = np.arange(S, dtype=np.int64).reshape(1, 1, S)

    def turned(a, at, n):
        t = C.to_device(np.ascontiguousarray(a[:, :, at:at + n]))
        return C.rotary(t, C.to_device(np.ascontiguousarray(pos[:, :, at:at + n])), freqs, [W // 2], "halves", out=t)

    whole = C.window_attention(turned(q, 0, S), turned(k, 0, S), C.to_device(v), window, sinks, W ** -0.5).numpy()
    junk = encode(kind, np.full((1, KV, CAP, W), np.nan))
    tk, tv = turned(k, 0, S).numpy(), v
    for at, n in [(0, P)] + [(i, 1) for i in range(P, S)]:
        ck, cv = junk.copy(), junk.copy()  # the cache holds garbage past the sequence
        ck[:, :, :at + n], cv[:, :, :at + n] = tk[:, :, :at + n], tv[:, :, :at + n]
        o = C.window_attention(turned(q, at, n), C.to_device(ck), C.to_device(cv), window, sinks, W ** -0.5,
                               lengths=C.to_device(np.array([at + n], np.int32))).numpy()
        a, b = decode(kind, o), decode(kind, whole[:, :, at:at + n])
        assert np.abs(a - b).max() <= 4 * 2.0**-8 * np.abs(decode(kind, v)).max()
