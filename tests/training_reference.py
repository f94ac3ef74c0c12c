"""Plain binary64 forms of the dense products, the residual stream between
blocks and gradient clipping, with bounds on what the kernels' roundings can
add. As in block_reference: u is half a step of the stored type, e half a step
of the width sums run at, a sum of chain length n is off by at most n e times
the sum of its magnitudes, matrix-core sums count twice."""
import math

import numpy as np

from block_reference import TINY, half_step, width_of

E = 2.0**-24
LOG2E = 1.4426950408889634
erfc = np.vectorize(math.erfc, otypes=[np.float64])


# ---- activations: value, bound of the binary32 evaluation, Lipschitz constant ----
def phi_tail(x):
    """Phi(-|x|) and the density, with their relative bound: 7.1e-8 of the
    polynomial, and the exponential's argument (two roundings of up to
    0.72 x^2) with four more roundings."""
    a = np.abs(x)
    return 0.5 * erfc(a / math.sqrt(2)), np.exp(-0.5 * a * a) / math.sqrt(2 * math.pi), 8e-8 + (0.5 * a * a * 2 + 12) * E


def act(name, x):
    if name == "gelu":
        tail, _, rel = phi_tail(x)
        y = np.where(x >= 0, x - x * tail, x * tail)
        return y, rel * np.abs(x) * tail + E * np.abs(y) + 2.0**-118
    if name == "silu":
        with np.errstate(over="ignore"):
            s = 1 / (1 + np.exp(-x))
        rel = ((np.abs(x) * LOG2E + 4) * E) * (1 - s) + 6 * E
        return x * s, rel * np.abs(x * s) + 2.0**-118
    if name == "relu":
        return np.maximum(x, 0), 0 * x
    return x, 0 * x


LIPSCHITZ = {None: 1.0, "relu": 1.0, "gelu": 1.13, "silu": 1.1}


def slope(name, x):
    if name == "gelu":
        tail, density, rel = phi_tail(x)
        d = np.where(x >= 0, 1 - tail, tail) + x * density
        return d, rel * (tail + np.abs(x) * density) + 4 * E * ((x >= 0) + np.abs(d)) + 2.0**-118
    if name == "silu":
        with np.errstate(over="ignore"):
            s = 1 / (1 + np.exp(-x))
        es = s * (((np.abs(x) * LOG2E + 4) * E) * (1 - s) + 6 * E)
        d = s * (1 + x * (1 - s))
        return d, es * (1 + np.abs(x) * (1 - s)) + s * (np.abs(x) * (es + E) + 2 * E * (1 + np.abs(x) * (1 - s))) + 2.0**-118
    if name == "relu":
        return (x > 0) * 1.0, 0 * x
    return np.ones_like(x), 0 * x


# ---- dense ----
def dense(kind, x, w, bias, name, residual):
    """(y, bound), (z, bound)"""
    u, k = half_step(kind), x.shape[-1]
    mag = np.abs(x) @ np.abs(w)
    z, ez = x @ w, 2 * (k + 4) * E * mag
    if bias is not None:
        z = z + bias
        ez = ez + 2 * E * (np.abs(z) + np.abs(bias) + mag)
    y, ey = act(name, z)
    ey = ey + LIPSCHITZ[name] * ez
    if residual is not None:
        y = y + residual
        ey = ey + 2 * E * (np.abs(y) + np.abs(residual))
    rounded = lambda v, ev: ev + u * (np.abs(v) + ev) + TINY[kind]
    return (y, rounded(y, ey)), (z, rounded(z, ez))


def dense_adjoint(kind, out_kind, x, w, z, name, g):
    """(dx, bound), (dw, bound), (dbias, bound): dz is rounded once for the
    products and summed as it is for dbias."""
    u, uo = half_step(kind), half_step(out_kind)
    s, es = slope(name, z if z is not None else g)
    dz, edz = g * s, np.abs(g) * es + E * np.abs(g * s)
    stored = edz + (u * (np.abs(dz) + edz) + TINY[kind] if name else 0)
    rounded = lambda v, ev, uu, tiny: ev + uu * (np.abs(v) + ev) + tiny
    ax, aw, ad = np.abs(x), np.abs(w), np.abs(dz) + stored
    dx, dw, db = dz @ w.T, x.T @ dz, dz.sum(0)
    rows, n = dz.shape
    return (dx, rounded(dx, stored @ aw.T + 2 * (n + 4) * E * (ad @ aw.T), u, TINY[kind])), \
        (dw, rounded(dw, ax.T @ stored + 2 * (rows + 4) * E * (ax.T @ ad), uo, TINY[out_kind])), \
        (db, rounded(db, edz.sum(0) + (rows + 8) * E * ad.sum(0), uo, TINY[out_kind]))


# ---- residual stream ----
def _depth(n):
    return 48 + n / 1024  # 16 in a lane, 6 across lanes, 16 across waves; long rows: n / 1024 in a lane


def unit(x, ex, how, eps, e):
    """The rows at unit size with the statistics, each with its bound, for
    inputs off by ex."""
    avg = lambda v: v.mean(-1, keepdims=True)
    n = x.shape[-1]
    d = _depth(n)
    mean = avg(x) if how == "layer" else np.zeros_like(x[..., :1])
    em = (avg(ex) + d * e * avg(np.abs(x)) + 2 * e * np.abs(mean)) * (how == "layer")
    c = x - mean
    ec = ex + em + e * np.abs(c)
    var = avg(c * c)
    ev = avg(2 * np.abs(c) * ec + ec * ec) + (d + 4) * e * var
    rstd = 1 / np.sqrt(var + eps)
    rel = 0.55 * ev / (var + eps) + 4 * e
    k = c * rstd
    return (k, ec * rstd * (1 + rel) + np.abs(k) * (rel + 2 * e)), (mean[..., 0], em[..., 0] + e * np.abs(mean[..., 0])), \
        (rstd[..., 0], (rstd * (rel + e))[..., 0])


def residual_norm(kind, x, b, post, gate, scale, pre, eps):
    """post, pre: (kind, gamma, beta) or None; gate broadcasts against x.
    Returns {name: (value, bound)}."""
    e, u, out = width_of(kind), half_step(kind), {}
    rounded = lambda v, ev: (v, ev + u * (np.abs(v) + ev) + TINY[kind])

    def weigh(k, ek, side):
        gamma, beta = (1.0 if side[1] is None else side[1]), (0.0 if side[2] is None else side[2])
        y = k * gamma + beta
        return y, ek * np.abs(gamma) + 2 * e * (np.abs(k * gamma) + np.abs(y))

    s, es = x, 0 * x
    if b is not None:
        v, ev = b, 0 * b
        if post:
            (k, ek), out["post_mean"], out["post_rstd"] = unit(b, 0 * b, post[0], eps, e)
            v, ev = weigh(k, ek, post)
        f = scale * (1.0 if gate is None else gate)
        s = x + f * v
        es = np.abs(f) * ev + 4 * e * (np.abs(f * v) + np.abs(s))
        out["u"] = rounded(s, es)
    if pre:
        (k, ek), out["pre_mean"], out["pre_rstd"] = unit(s, es, pre[0], eps, e)
        out["h"] = rounded(*weigh(k, ek, pre))
    return out


def residual_norm_adjoint(kind, weights, u, b, post, gate, scale, pre, du, dh):
    """post, pre: (kind, gamma, beta, mean, rstd) or None; gate [groups, 1, n]
    or [n] over u [groups, rows, n]."""
    e, n = width_of(kind), (u if u is not None else du).shape[-1]
    d, out = _depth(n) + 8, {}
    avg = lambda v: v.mean(-1, keepdims=True)
    lead = (0, 1)
    rows = int(np.prod((u if u is not None else du).shape[:-1]))

    def rounded(v, ev, t):
        return v, ev + half_step(t) * (np.abs(v) + ev) + TINY[t]

    def stored(x, side):
        c = x - (side[3][..., None] if side[0] == "layer" else 0.0)
        return c * side[4][..., None], 3 * e * np.abs(c * side[4][..., None])

    def back(w, ew, k, ek, side):
        r = side[4][..., None]
        c1 = avg(w) if side[0] == "layer" else 0.0
        e1 = (avg(ew) + d * e * avg(np.abs(w))) * (side[0] == "layer")
        c2 = avg(w * k)
        e2 = avg(ew * np.abs(k) + ek * np.abs(w)) + d * e * avg(np.abs(w * k))
        return r * (w - c1 - k * c2), r * (ew + e1 + np.abs(k) * e2 + ek * np.abs(c2)
                                           + 5 * e * (np.abs(w) + np.abs(c1) + np.abs(k * c2)))

    t, et = 0.0, 0.0
    if pre:
        k, ek = stored(u, pre)
        g = 1.0 if pre[1] is None else pre[1]
        t, et = back(dh * g, e * np.abs(dh * g), k, ek, pre)
        out["pre_dgamma"] = rounded((dh * k).sum(lead), (np.abs(dh) * ek).sum(lead) + (rows + 40) * e * np.abs(dh * k).sum(lead), weights)
        out["pre_dbeta"] = rounded(dh.sum(lead), (rows + 40) * e * np.abs(dh).sum(lead), weights)
    if du is not None:
        t = t + du
        et = et + e * np.abs(t)
    out["dx"] = rounded(t, et, kind)
    if b is None:
        return out
    k, ek = stored(b, post) if post else (b, 0 * b)
    gamma = 1.0 if not post or post[1] is None else post[1]
    beta = 0.0 if not post or post[2] is None else post[2]
    gv = 1.0 if gate is None else gate
    f = scale * gv
    terms = (rows + 40) * e
    s1, e1 = t.sum(1, keepdims=True), et.sum(1, keepdims=True) + terms * np.abs(t).sum(1, keepdims=True)
    s2 = (t * k).sum(1, keepdims=True)
    e2 = (et * np.abs(k) + np.abs(t) * ek).sum(1, keepdims=True) + terms * np.abs(t * k).sum(1, keepdims=True)
    if not post:
        gg, bb = 1.0, 0.0
    else:
        gg, bb = gamma, beta
    dg = scale * (gg * s2 + bb * s1)
    out["dgate"] = rounded(dg[:, 0], np.abs(scale) * (np.abs(gg) * e2 + np.abs(bb) * e1 + 6 * e * (np.abs(gg * s2) + np.abs(bb * s1)))[:, 0], weights)
    total = lambda s, es: ((f * s).sum(lead), (np.abs(f) * es).sum(lead) + terms * np.abs(f * s).sum(lead))
    if post:
        out["post_dgamma"] = rounded(*total(s2, e2), weights)
        out["post_dbeta"] = rounded(*total(s1, e1), weights)
        p = f * t * gamma
        v, ev = back(p, np.abs(f * gamma) * et + 4 * e * np.abs(p), k, ek, post)
    else:
        v, ev = f * t, np.abs(f) * et + 3 * e * np.abs(f * t)
    out["db"] = rounded(v, ev, kind)
    return out
