"""Plain binary64 forms of layer norm with its gradients, rotary positions and
windowed attention with its gradients, with bounds on what the kernels'
roundings can add, and the carriers the tests move 16-bit arrays in.

A bound follows the kernels' arithmetic: u is half a step of the stored type
(one rounding of the result, and of every weight that is rounded to the type
for a product), e half a step of the width sums run at, and a sum of n terms
is off by at most n e times the sum of their magnitudes. Matrix-core sums may
round between products as well as between sums: they count twice."""
import ctypes

import numpy as np

U = {"f64": 2.0**-53, "f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11}
TINY = {"f64": 2.0**-1075, "f32": 2.0**-150, "bf16": 2.0**-134, "f16": 2.0**-25}  # half the least subnormal
NP = {"f64": np.float64, "f32": np.float32, "bf16": np.uint16, "f16": np.float16}


def half_step(kind):
    return U[kind]


def encode(kind, x):
    """The array the device tensor of this dtype is made from."""
    x = np.asarray(x, np.float64)
    if kind != "bf16":
        return x.astype(NP[kind])
    b = x.astype(np.float32).view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> np.uint64(16)) & np.uint64(1))) >> np.uint64(16)).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def decode(kind, a):
    a = np.ascontiguousarray(a)
    if kind != "bf16":
        return a.astype(np.float64)
    return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def draw(kind, rng, shape, scale=1.0, mean=0.0):
    """(stored array, its values in binary64)"""
    a = encode(kind, rng.standard_normal(shape) * scale + mean)
    return a, decode(kind, a)


def check(got, want, bound, what=""):
    """|got - want| <= bound; NaN and infinities where want has them."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    same = got == want
    with np.errstate(invalid="ignore"):
        bad = np.where(fin, ~(np.abs(got - want) <= bound), ~(same | np.isnan(want)))
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4],
                           np.broadcast_to(bound, want.shape)[bad][:4])


class Captured:
    """What `enqueue` launches on the library stream, as a graph."""

    def __init__(self, enqueue):
        import chelis_amd as C
        from chelis_amd import hiprt
        self.hip, self.stream = hiprt.hip(), ctypes.c_void_p(C.lib().chelis_hip_stream())
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 0) == 0
        try:
            enqueue()
        finally:
            end = self.hip.hipStreamEndCapture(self.stream, ctypes.byref(graph))
        assert end == 0
        assert self.hip.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0)) == 0

    def launch(self):
        assert self.hip.hipGraphLaunch(self.exec, self.stream) == 0


# ---- layer norm ----
def width_of(kind):
    return 2.0**-53 if kind == "f64" else 2.0**-24


def norm(kind, x, gamma, beta, eps):
    """y, mean, rstd and their bounds."""
    e, u, n = width_of(kind), half_step(kind), x.shape[-1]
    depth = 40  # roundings along a row sum: 16 in a lane, 6 across lanes, 16 across waves
    mean = x.mean(-1, keepdims=True)
    d = x - mean
    var = (d * d).mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    mean_err = (depth + max(0, n / 16384)) * e * np.abs(x).mean(-1, keepdims=True)
    d_err = e * np.abs(d) + mean_err
    var_err = (depth + 4 + max(0, n / 16384)) * e * var + 2 * (d_err * np.abs(d)).mean(-1, keepdims=True) \
        + (d_err**2).mean(-1, keepdims=True)
    r_rel = 0.5 * var_err / (var + eps) + 4 * e
    y = d * rstd * gamma + beta
    err = np.abs(gamma) * rstd * (d_err + np.abs(d) * (r_rel + 4 * e)) + e * np.abs(y)
    return (y, err + u * np.abs(y) + TINY[kind]), (mean[..., 0], mean_err[..., 0] + e * np.abs(mean[..., 0])), \
        (rstd[..., 0], rstd[..., 0] * r_rel[..., 0])


def norm_adjoint(kind, weights, x, gamma, mean, rstd, g):
    """dx, dgamma, dbeta and their bounds, for the given statistics."""
    e, u, uw = width_of(kind), half_step(kind), half_step(weights)
    n, rows = x.shape[-1], int(np.prod(x.shape[:-1]))
    m, r = mean[..., None], rstd[..., None]
    h = (x - m) * r
    w = g * gamma
    c1, c2 = w.mean(-1, keepdims=True), (w * h).mean(-1, keepdims=True)
    depth = 46 + n / 8192
    dx = r * (w - c1 - h * c2)
    e1, e2 = depth * e * np.abs(w).mean(-1, keepdims=True), (depth + 4) * e * np.abs(w * h).mean(-1, keepdims=True)
    err = np.abs(r) * (e1 + np.abs(h) * e2 + 5 * e * (np.abs(w) + np.abs(c1) + np.abs(h * c2)))
    terms = 160 + rows / 64
    lead = tuple(range(x.ndim - 1))
    dg, db = (g * h).sum(lead), g.sum(lead)
    return (dx, err + u * np.abs(dx) + TINY[kind]), \
        (dg, terms * e * np.abs(g * h).sum(lead) + uw * np.abs(dg) + TINY[weights]), \
        (db, terms * e * np.abs(g).sum(lead) + uw * np.abs(db) + TINY[weights])


# ---- rotary positions ----
def rotary(kind, x, positions, freqs, sections, pairing, sign=1.0):
    """The turned x [batch, heads, seq, width] and its bound: the sine and
    cosine are off by 4 half steps of the arithmetic width (the polynomials,
    the angle's rounding after reduction, their own rounding)."""
    e, u, pairs = width_of(kind), half_step(kind), len(freqs)
    axis = np.repeat(np.arange(len(sections)), sections)
    angle = np.moveaxis(positions.astype(np.float64)[axis], 0, -1) * freqs * sign  # [batch, seq, pairs]
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    i = np.arange(pairs)
    iu, iv = (i, pairs + i) if pairing == "halves" else (2 * i, 2 * i + 1)
    y, bound = x.copy(), np.zeros_like(x)
    a, b = x[..., iu], x[..., iv]
    y[..., iu], y[..., iv] = a * c - b * s, a * s + b * c
    turn = 4 if kind != "f64" else 8  # the reference's own angle and sines round at the same width
    for k in (iu, iv):
        bound[..., k] = (np.abs(a) + np.abs(b)) * (turn + 2) * e + u * np.abs(y[..., k]) + TINY[kind]
    return y, bound


# ---- windowed attention ----
def visible(sq, sk, n, start, window, sinks):
    p = start + np.arange(sq)[:, None]
    j = np.arange(sk)[None, :]
    return (j <= p) & (p < n) & ((p - j < window) | (j < sinks))


def spans(batch, sq, sk, lengths, starts):
    lengths = [sk] * batch if lengths is None else [min(max(int(v), 0), sk) for v in lengths]
    starts = [n - sq for n in lengths] if starts is None else [int(v) for v in starts]
    return lengths, starts


# The exponential instruction returns 0 below the least normal binary32 number,
# and products and sums below it may be flushed on the matrix cores: each
# weight, product and partial sum is off by at most this much more.
FLUSH = 2.0**-126


def _scores(kind, q, k, scale):
    s = (q @ k.T) * scale
    terms = 2 * q.shape[-1] + 2
    err = terms * 2.0**-24 * abs(scale) * (np.abs(q) @ np.abs(k).T)
    return s, err


def window_forward(kind, q, k, v, window, sinks, scale, lengths=None, starts=None):
    """(o, bound), (lse, bound); hidden values of k and v must be finite here."""
    (B, H, S, D), (KV, N), e, u = q.shape, k.shape[1:3], 2.0**-24, half_step(kind)
    o, bo = np.zeros(q.shape), np.zeros(q.shape)
    lse, bl = np.full(q.shape[:3], -np.inf), np.zeros(q.shape[:3])
    for b, (n, start) in enumerate(zip(*spans(B, S, N, lengths, starts))):
        vis = visible(S, N, n, start, window, sinks)
        some = vis.any(1)
        for h in range(H):
            kk, vv = k[b, h * KV // H], v[b, h * KV // H]
            s, err = _scores(kind, q[b, h], kk, scale)
            s = np.where(vis, s, -np.inf)
            m = np.where(some, s.max(1), 0.0)
            w = np.exp(s - m[:, None])
            total = np.where(some, w.sum(1), 1.0)
            p = w / total[:, None]
            o[b, h] = p @ vv
            lse[b, h] = np.where(some, m + np.log(total), -np.inf)
            # every weight: its score, the exponent's roundings, the exponential
            worst = np.where(vis, err + 8 * e * (np.abs(np.where(vis, s, 0)) + np.abs(m)[:, None]), 0).max(1) + 4 * e
            count = vis.sum(1)
            a = p @ np.abs(vv)
            bo[b, h] = a * (2 * worst + (2 * count + 16) * e + u)[:, None] + u * np.abs(o[b, h]) + TINY[kind]
            bo[b, h] += FLUSH * (vis @ (2 + np.abs(vv)))
            if kind == "f16":  # weights below 2^-10 times f16's least subnormal
                bo[b, h] += 2.0**-35 * (vis @ np.abs(vv))
            bl[b, h] = worst + (count + 10) * e + 8 * e * (np.abs(np.where(some, lse[b, h], 0)) + np.abs(m) + 16)
    return (o, bo), (lse, bl)


def window_adjoint(kind, q, k, v, o, lse, g, window, sinks, scale, lengths=None, starts=None):
    """(dq, bound), (dk, bound), (dv, bound) for the given o and lse."""
    (B, H, S, D), (KV, N), e, u = q.shape, k.shape[1:3], 2.0**-24, half_step(kind)
    dq, bq = np.zeros(q.shape), np.zeros(q.shape)
    dk, bk, dv, bv = (np.zeros(k.shape) for _ in range(4))
    # f16's least subnormal under the scale that brings 2 max|g| max|v| width to at least 2^14
    least = 2.0**-25 * 2 * np.abs(g).max(initial=0) * np.abs(v).max(initial=0) * D / 2.0**13 if kind == "f16" else 0.0
    for b, (n, start) in enumerate(zip(*spans(B, S, N, lengths, starts))):
        vis = visible(S, N, n, start, window, sinks)
        some = vis.any(1)
        for h in range(H):
            c = h * KV // H
            Q, K, V, G, O = q[b, h], k[b, c], v[b, c], g[b, h], o[b, h]
            s, err = _scores(kind, Q, K, scale)
            L = np.where(some, lse[b, h], 0.0)[:, None]
            p = np.where(vis, np.exp(np.where(vis, s - L, 0)), 0.0)
            rel = np.where(vis, err + 8 * e * (np.abs(s) + np.abs(L)), 0) + 4 * e
            dot = (G * O).sum(1, keepdims=True)
            dp = G @ V.T
            ds = p * (dp - dot)
            dp_err = (2 * D + 2) * e * (np.abs(G) @ np.abs(V).T + (np.abs(G) * np.abs(O)).sum(1, keepdims=True))
            ds_err = p * dp_err + np.abs(ds) * (rel + 4 * e + u) + np.where(vis, least, 0)
            p_err = p * (rel + u) + np.where(vis, 2.0**-35 if kind == "f16" else 0, 0)
            ds_err, p_err = ds_err + vis * FLUSH * (2 + np.abs(dp) + np.abs(dot)), p_err + vis * FLUSH
            terms, rows = 2 * vis.sum(1, keepdims=True) + 4, 2 * H // KV * vis.sum(0)[:, None] + 4
            dq[b, h] = scale * ds @ K
            bq[b, h] = abs(scale) * ((ds_err + terms * e * np.abs(ds)) @ np.abs(K) + terms * FLUSH)
            dk[b, c] += scale * ds.T @ Q
            bk[b, c] += abs(scale) * (ds_err.T @ np.abs(Q) + rows * (e * (np.abs(ds).T @ np.abs(Q)) + FLUSH))
            dv[b, c] += p.T @ G
            bv[b, c] += p_err.T @ np.abs(G) + rows * (e * (p.T @ np.abs(G)) + FLUSH)
    done = []
    for x, bound in ((dq, bq), (dk, bk), (dv, bv)):
        done.append((x, bound * (1 + u) + u * np.abs(x) + TINY[kind]))
    return done
