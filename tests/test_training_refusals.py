"""What the dense products, the residual stream between blocks and gradient
clipping refuse: each call is turned down on the host, before any device is
touched, so these run without one. The packets point at host memory that nothing
reads."""
import ctypes

import pytest

import chelis_amd as C
from test_block_refusals import (BF16, EDOMAIN, EUNSUPPORTED, F16, F32, F64, I32, at, ref, refused, tensor)


# ---- dense ----
def rows(n, dtype=BF16):
    return tensor((2, 3, n), dtype)


def dense(x=None, w=None, bias=None, act=0, residual=None, y=None, z=None):
    x = x or rows(16)
    return C.lib().chelis_hip_dense(ref(x), ref(w or tensor((16, 24), x.dtype)), ref(bias), act, ref(residual),
                                    ref(y or rows(24, x.dtype)), ref(z))


@pytest.mark.parametrize("change,text,code", [
    (lambda: dict(x=rows(16, F32)), "x must be bf16 or f16", EDOMAIN),
    (lambda: dict(x=tensor((), BF16)), "x needs a last axis", EDOMAIN),
    (lambda: dict(w=tensor((15, 24), BF16)), "w must be [K, N]", EDOMAIN),
    (lambda: dict(w=tensor((16, 24), F16)), "w must be [K, N]", EDOMAIN),
    (lambda: dict(w=tensor((2, 16, 24), BF16)), "w must be [K, N]", EDOMAIN),
    (lambda: dict(w=tensor((16, 24), BF16, (48, 2))), "one axis must be contiguous", EUNSUPPORTED),
    (lambda: dict(x=tensor((2, 3, 16), BF16, (96, 32, 2))), "x: last axis must be contiguous", EUNSUPPORTED),
    (lambda: dict(x=tensor((2, 3, 16), BF16, (100, 32, 1))), "uniform row stride", EUNSUPPORTED),
    (lambda: dict(y=rows(23)), "y must be [x's leading axes, 24]", EDOMAIN),
    (lambda: dict(y=tensor((6, 24), BF16)), "y must be [x's leading axes, 24]", EDOMAIN),
    (lambda: dict(y=rows(24, F16)), "y must have x's dtype", EDOMAIN),
    (lambda: dict(y=tensor((2, 3, 24), BF16, (24, 8, 1))), "y overlaps itself", EDOMAIN),
    (lambda: dict(bias=tensor((23,), BF16)), "bias must be contiguous [N]", EDOMAIN),
    (lambda: dict(bias=tensor((24,), F16)), "bias must have x's dtype or f32", EDOMAIN),
    (lambda: dict(bias=tensor((24,), F32, (2,))), "bias must be contiguous [N]", EDOMAIN),
    (lambda: dict(residual=rows(16)), "residual must be", EDOMAIN),
    (lambda: dict(z=rows(24, F32)), "z must have x's dtype", EDOMAIN),
    (lambda: dict(act=4), "unknown activation", EDOMAIN),
    (lambda: dict(act=-1), "unknown activation", EDOMAIN),
    (lambda: dict(x=tensor((2, 3, 16), BF16, room=64)), "past byte_capacity", EDOMAIN),
])
def test_dense(change, text, code):
    refused(dense(**change()), text, code)


def test_dense_results_lie_apart():
    x, w = rows(24), tensor((24, 24), BF16)
    refused(dense(x=x, w=w, y=at(x, (2, 3, 24), (72, 24, 1), BF16)), "y and x overlap", EDOMAIN)
    refused(dense(w=w, x=x, y=at(w, (2, 3, 24), (72, 24, 1), BF16)), "y and w overlap", EDOMAIN)
    y = rows(24)
    refused(dense(y=y, z=at(y, (2, 3, 24), (72, 24, 1), BF16)), "z and y overlap", EDOMAIN)
    r = tensor((2, 3, 24), BF16, (90, 30, 1))
    refused(dense(residual=r, y=at(r, (2, 3, 24), (72, 24, 1), BF16)), "y overlaps residual with other strides", EDOMAIN)
    refused(dense(residual=r, z=at(r, (2, 3, 24), (90, 30, 1), BF16)), "z and residual overlap", EDOMAIN)


def test_dense_widths_have_a_limit():
    n = (1 << 20) + 1
    x = tensor((1, n), BF16, room=2 * n)
    refused(dense(x=x, w=tensor((n, 1), BF16, room=2 * n), y=tensor((1, 1), BF16)), "widths past 2^20", EUNSUPPORTED)


def adjoint(x=None, w=None, z=0, act=2, g=None, dx=0, dw=0, dbias=0):
    x = x or rows(16)
    made = lambda t, new: new if t == 0 else t
    return C.lib().chelis_hip_dense_adjoint(
        ref(x), ref(w or tensor((16, 24), x.dtype)), ref(made(z, rows(24, x.dtype))), act, ref(g or rows(24, x.dtype)),
        ref(made(dx, rows(16, x.dtype))), ref(made(dw, tensor((16, 24), x.dtype))), ref(made(dbias, tensor((24,), x.dtype))))


@pytest.mark.parametrize("change,text,code", [
    (lambda: dict(dx=None, dw=None, dbias=None), "no gradient asked for", EDOMAIN),
    (lambda: dict(z=None), "needs z", EDOMAIN),
    (lambda: dict(act=7), "unknown activation", EDOMAIN),
    (lambda: dict(g=rows(25)), "g must be [x's leading axes, 24]", EDOMAIN),
    (lambda: dict(z=rows(16)), "z must be", EDOMAIN),
    (lambda: dict(dx=rows(24)), "dx must be [x's leading axes, 16]", EDOMAIN),
    (lambda: dict(dx=rows(16, F32)), "dx must have x's dtype", EDOMAIN),
    (lambda: dict(dw=tensor((24, 16), BF16)), "dw must be [K, N]", EDOMAIN),
    (lambda: dict(dw=tensor((16, 24), F64)), "dw must have x's dtype or f32", EDOMAIN),
    (lambda: dict(dw=tensor((16, 24), BF16, (0, 1))), "dw overlaps itself", EDOMAIN),
    (lambda: dict(dw=tensor((16, 24), BF16, (48, 2))), "dw: one axis must be contiguous", EUNSUPPORTED),
    (lambda: dict(dbias=tensor((24,), F16)), "dbias must have x's dtype or f32", EDOMAIN),
    (lambda: dict(dbias=tensor((1, 24), BF16)), "dbias must be contiguous [N]", EDOMAIN),
])
def test_dense_adjoint(change, text, code):
    refused(adjoint(**change()), text, code)


def test_dense_gradients_lie_apart():
    g = rows(16)
    refused(adjoint(w=tensor((16, 16), BF16), g=g, z=rows(16), dx=at(g, (2, 3, 16), (48, 16, 1), BF16)), "dx and g overlap", EDOMAIN)
    w = tensor((16, 24), BF16)
    refused(adjoint(w=w, dw=at(w, (16, 24), (24, 1), BF16)), "dw and w overlap", EDOMAIN)
    dw = tensor((16, 24), BF16)
    refused(adjoint(dw=dw, dbias=at(dw, (24,), (1,), BF16)), "dbias and dw overlap", EDOMAIN)


# ---- residual stream ----
def side(kind=1, gamma=0, beta=None, mean=0, rstd=0, dtype=F32, n=16, reserved=0):
    made = lambda t, new: new if t == 0 else t
    p = lambda t: ctypes.pointer(t) if t is not None else None
    mean = tensor((4,)) if mean == 0 and kind == 1 else None if mean == 0 else mean
    return C.NormSide(kind, reserved, p(made(gamma, tensor((n,), dtype))), p(beta), p(mean), p(made(rstd, tensor((4,)))))


def residual(x=None, b=0, post=0, gate=None, scale=1.0, pre=0, eps=1e-5, u=0, h=0):
    x = x or tensor((4, 16))
    made = lambda t, new: new() if t == 0 else t
    like = lambda: tensor((4, 16), x.dtype)
    post, pre = made(post, lambda: side(dtype=x.dtype)), made(pre, lambda: side(2, dtype=x.dtype))
    byref = lambda s: ctypes.byref(s) if s is not None else None
    return C.lib().chelis_hip_residual_norm(ref(x), ref(made(b, like)), byref(post), ref(gate), scale, byref(pre), eps,
                                            ref(made(u, like)), ref(made(h, like)))


@pytest.mark.parametrize("change,text,code", [
    (lambda: dict(x=tensor((4, 16), I32), post=None, pre=side(2)), "x must be f32, f64, bf16 or f16", EDOMAIN),
    (lambda: dict(x=tensor((4, 16), F32, (16, 2))), "last axis must be contiguous", EUNSUPPORTED),
    (lambda: dict(b=None), "post, gate and u come with b", EDOMAIN),
    (lambda: dict(b=None, post=None, u=None, pre=None, h=None), "no result asked for", EDOMAIN),
    (lambda: dict(u=None), "b needs u", EDOMAIN),
    (lambda: dict(h=None), "pre and h come together", EDOMAIN),
    (lambda: dict(pre=None), "pre and h come together", EDOMAIN),
    (lambda: dict(scale=float("nan")), "scale must be finite", EDOMAIN),
    (lambda: dict(eps=-1.0), "epsilon must not be negative", EDOMAIN),
    (lambda: dict(b=tensor((4, 15))), "b must match x", EDOMAIN),
    (lambda: dict(u=tensor((4, 16), F64)), "u must match x", EDOMAIN),
    (lambda: dict(h=tensor((4, 16), F32, (0, 1))), "h overlaps itself", EDOMAIN),
    (lambda: dict(post=side(3)), "unknown norm", EDOMAIN),
    (lambda: dict(post=side(reserved=1)), "reserved field", EDOMAIN),
    (lambda: dict(post=side(0)), "beside no norm", EDOMAIN),
    (lambda: dict(post=side(2, mean=tensor((4,)))), "post mean beside an rms norm", EDOMAIN),
    (lambda: dict(post=side(gamma=tensor((15,)))), "post gamma must be contiguous", EDOMAIN),
    (lambda: dict(pre=side(2, beta=tensor((16,), F64))), "pre beta must have x's dtype", EDOMAIN),
    (lambda: dict(pre=side(rstd=tensor((5,)))), "pre rstd must be contiguous", EDOMAIN),
    (lambda: dict(pre=side(mean=tensor((4,), F64))), "pre mean must be f32", EDOMAIN),
    (lambda: dict(gate=tensor((15,))), "gate must be contiguous", EDOMAIN),
    (lambda: dict(gate=tensor((4, 16))), "gate must be contiguous", EDOMAIN),
    (lambda: dict(gate=tensor((16,), F16)), "gate must have x's dtype", EDOMAIN),
    (lambda: dict(x=tensor((4, 16), BF16), gate=tensor((16,))), "share a dtype", EDOMAIN),
])
def test_residual_norm(change, text, code):
    refused(residual(**change()), text, code)


def test_residual_norm_results_lie_apart():
    x = tensor((4, 16), F32, (20, 1))
    refused(residual(x=x, u=at(x, (4, 16), (16, 1))), "u overlaps an input with other strides", EDOMAIN)
    u = tensor((4, 16))
    refused(residual(u=u, h=at(u, (4, 16), (16, 1))), "h and u overlap", EDOMAIN)
    refused(residual(u=u, post=side(rstd=at(u, (4,), (1,)))), "post rstd and u overlap", EDOMAIN)
    r = tensor((4,))
    refused(residual(post=side(rstd=r), pre=side(2, rstd=at(r, (4,), (1,)))), "pre rstd and post rstd overlap", EDOMAIN)
    gate = tensor((64,))
    refused(residual(gate=at(gate, (16,), (1,)), h=at(gate, (4, 16), (16, 1))), "h and gate overlap", EDOMAIN)


def residual_adjoint(u=0, b=0, post=0, gate=None, scale=1.0, pre=0, du=0, dh=0, dx=0, db=0, dgate=None, grads=(None,) * 4):
    made = lambda t, new: new() if t == 0 else t
    like = lambda: tensor((4, 16))
    post, pre = made(post, side), made(pre, lambda: side(2))
    byref = lambda s: ctypes.byref(s) if s is not None else None
    u, b, du, dh, dx, db = (ref(made(t, like)) for t in (u, b, du, dh, dx, db))
    return C.lib().chelis_hip_residual_norm_adjoint(u, b, byref(post), ref(gate), scale, byref(pre), du, dh, dx, db, ref(dgate),
                                                    *[ref(t) for t in grads])


@pytest.mark.parametrize("change,text,code", [
    (lambda: dict(du=None, dh=None), "no cotangent given", EDOMAIN),
    (lambda: dict(dh=None), "pre and dh come together", EDOMAIN),
    (lambda: dict(dx=None, db=None), "no gradient asked for", EDOMAIN),
    (lambda: dict(b=None), "come with b", EDOMAIN),
    (lambda: dict(dgate=tensor((16,))), "dgate without gate", EDOMAIN),
    (lambda: dict(post=None, grads=(tensor((16,)), None, None, None)), "post gradients without post", EDOMAIN),
    (lambda: dict(pre=None, dh=None, grads=(None, None, tensor((16,)), None)), "pre gradients without pre", EDOMAIN),
    (lambda: dict(post=side(rstd=None)), "post rstd (and post mean for layer) must be given", EDOMAIN),
    (lambda: dict(post=side(mean=None)), "must be given", EDOMAIN),
    (lambda: dict(du=tensor((4, 8))), "du must match x", EDOMAIN),
    (lambda: dict(db=tensor((4, 16), F64)), "db must match x", EDOMAIN),
    (lambda: dict(dx=tensor((4, 16), F32, (0, 1))), "dx overlaps itself", EDOMAIN),
    (lambda: dict(gate=tensor((16,)), dgate=tensor((16,), F64)), "dgate must have x's dtype", EDOMAIN),
    (lambda: dict(grads=(tensor((16,), F16), None, None, None)), "post dgamma must have x's dtype", EDOMAIN),
    (lambda: dict(grads=(None, None, None, tensor((17,)))), "pre dbeta must be contiguous", EDOMAIN),
    (lambda: dict(scale=float("inf")), "scale must be finite", EDOMAIN),
])
def test_residual_norm_adjoint(change, text, code):
    refused(residual_adjoint(**change()), text, code)


def test_residual_norm_gradients_lie_apart():
    d = tensor((16,))
    refused(residual_adjoint(grads=(d, at(d, (16,), (1,)), None, None)), "post dbeta and post dgamma overlap", EDOMAIN)
    dx = tensor((4, 16))
    refused(residual_adjoint(dx=dx, db=at(dx, (4, 16), (16, 1))), "db and dx overlap", EDOMAIN)
    refused(residual_adjoint(dx=dx, grads=(None, None, at(dx, (16,), (1,)), None)), "pre dgamma and dx overlap", EDOMAIN)
    du = tensor((4, 16), F32, (20, 1))
    refused(residual_adjoint(du=du, dx=at(du, (4, 16), (16, 1))), "dx overlaps an input with other strides", EDOMAIN)


# ---- clipping ----
def packets(ts):
    return (C.P * max(1, len(ts)))(*[ctypes.pointer(t) for t in ts])


def norm_of(gs, norm=None, scale=1.0):
    return C.lib().chelis_hip_gradient_norm(packets(gs), len(gs), scale, ref(norm or tensor(())))


def clip(gs, outs=None, norm=None, most=1.0, scale=1.0):
    return C.lib().chelis_hip_clip_gradients(packets(gs), len(gs), ref(norm or tensor(())), most, scale, packets(outs or gs))


@pytest.mark.parametrize("call", [norm_of, clip])
@pytest.mark.parametrize("gs,more,text,code", [
    (lambda: [tensor((4,), I32)], {}, "must be f32, f64, bf16 or f16", EDOMAIN),
    (lambda: [tensor((4, 4), F32, (0, 1))], {}, "overlaps itself", EDOMAIN),
    (lambda: [tensor((4,)), tensor((4, 4, 4), F32, (100, 10, 1))], {}, "gradient 1 is neither dense nor", EUNSUPPORTED),
    (lambda: [tensor((4, 4), F32, (20, 2))], {}, "gradient 0 is neither dense nor", EUNSUPPORTED),
    (lambda: [tensor((4,))], {"scale": 0.0}, "scale must be positive", EDOMAIN),
    (lambda: [tensor((4,))], {"scale": float("nan")}, "scale must be positive", EDOMAIN),
    (lambda: [tensor((4,))], {"norm": lambda: tensor((2,))}, "norm must be one f32 or f64 element", EDOMAIN),
    (lambda: [tensor((4,))], {"norm": lambda: tensor((1,), BF16)}, "norm must be one f32 or f64 element", EDOMAIN),
    (lambda: [tensor((40,), room=64)], {}, "past byte_capacity", EDOMAIN),
])
def test_gradient_lists(call, gs, more, text, code):
    refused(call(gs(), **{k: v() if callable(v) else v for k, v in more.items()}), text, code)


@pytest.mark.parametrize("most", [0.0, -1.0, float("inf"), float("nan")])
def test_max_norm(most):
    refused(clip([tensor((4,))], most=most), "max_norm must be positive and finite", EDOMAIN)


def test_clipped_gradients_match_and_lie_apart():
    a, b = tensor((8, 8)), tensor((8, 8))
    refused(clip([a], [tensor((8, 8), F64)]), "result 0 must match", EDOMAIN)
    refused(clip([a], [tensor((64,))]), "result 0 must match", EDOMAIN)
    refused(clip([a], [tensor((8, 8), F32, (1, 8))]), "another order of axes", EUNSUPPORTED)
    refused(clip([a, b], [a, at(a, (8, 8), (8, 1))]), "result 0 overlaps result 1", EDOMAIN)
    refused(clip([a, b], [b, tensor((8, 8))]), "result 0 overlaps gradient 1", EDOMAIN)
    refused(clip([a, a]), "overlaps result", EDOMAIN)
    wide = tensor((8, 16))
    left, right = at(wide, (8, 8), (16, 1)), tensor((8, 8))
    refused(clip([left, b], [left, at(wide, (8, 8), (8, 1))]), "overlaps", EDOMAIN)
    norm = at(b, (1,), (1,))
    refused(clip([a], [b], norm=norm), "norm and result 0 overlap", EDOMAIN)
    refused(norm_of([b], norm=norm), "norm and gradient 0 overlap", EDOMAIN)


# ---- calls that no argument check of theirs alone turns down ----
def test_the_gradients_of_a_norm_need_its_rows():
    refused(residual_adjoint(u=None), "pre needs u", EDOMAIN)
