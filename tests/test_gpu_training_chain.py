"""A whole block's training step in 16 bits, as a program runs it: rms norm, one
packed q/k/v product, rotary positions in place, windowed attention, the output
product, the stream with its norms and gate, the two products of the feed-forward
half, the stream again, all of it backwards, and the gradients' norm and clipping;
against the same step in binary64 by automatic differentiation."""
import math

import numpy as np
import pytest
import torch

import chelis_amd as C
from block_reference import NP, decode, draw

pytestmark = pytest.mark.gpu
EPS = 1e-5


def torch_step(p, g, B, S, H, KV, W, window, sinks, freqs, scale):
    """Gradients of sum(out * g) with the tensors of p as leaves, all binary64."""
    leaf = {k: torch.tensor(v, dtype=torch.float64, requires_grad=True) for k, v in p.items()}
    rms = lambda x, w: x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    gelu = lambda z: 0.5 * z * torch.erfc(-z / math.sqrt(2))
    x = leaf["x"]
    qkv = (rms(x, leaf["norm1"]) @ leaf["wqkv"] + leaf["bqkv"]).reshape(B, S, H + 2 * KV, W).transpose(1, 2)
    angle = torch.arange(S, dtype=torch.float64)[:, None] * torch.tensor(freqs)

    def turn(t):
        u, v = t[..., :W // 2], t[..., W // 2:]
        return torch.cat([u * angle.cos() - v * angle.sin(), u * angle.sin() + v * angle.cos()], -1)

    q, k, v = turn(qkv[:, :H]), turn(qkv[:, H:H + KV]), qkv[:, H + KV:]
    k, v = (t.repeat_interleave(H // KV, 1) for t in (k, v))
    i, j = torch.arange(S)[:, None], torch.arange(S)[None]
    hidden = (j > i) | ((i - j >= window) & (j >= sinks))
    o = torch.softmax((q @ k.transpose(2, 3) * scale).masked_fill(hidden, -torch.inf), -1) @ v
    b1 = o.transpose(1, 2).reshape(B, S, H * W) @ leaf["wo"]
    u = x + 0.5 * leaf["gate1"] * rms(b1, leaf["post1"])
    z = rms(u, leaf["norm2"]) @ leaf["w1"] + leaf["b1"]
    out = u + gelu(z) @ leaf["w2"] + leaf["b2"]
    (out * torch.tensor(g)).sum().backward()
    return out.detach().numpy(), {k: t.grad.numpy() for k, t in leaf.items()}


@pytest.mark.parametrize("kind,B,S,M,H,KV,W,F", [("f16", 2, 75, 96, 4, 2, 64, 200), ("bf16", 1, 200, 256, 4, 4, 72, 512),
                                                 ("f16", 3, 33, 130, 2, 1, 64, 333)])
def test_training_step(kind, B, S, M, H, KV, W, F):
    """Each result's distance from binary64 in the Euclidean norm. The longest way
    from an input to a gradient passes 24 stored 16-bit tensors forwards and
    backwards (12 each way: a norm, qkv, the turned heads, o, b1, u, h, z, y, and
    inside the attention and dense gradients the rounded weights and cotangents),
    each off by at most half a step u of its elements, and no stage here makes a
    relative error more than twice as large (norms: 1 + their own average; products
    and sums of independent terms: 1). Bar: 24 * 2 * u, and 2^-10 beside it for the
    smallest binary16 values' absolute rounding."""
    rng = np.random.default_rng(S)
    window, sinks, scale, N = 24, 2, W ** -0.5, (H + 2 * KV) * W
    freqs = 10000.0 ** (-np.arange(W // 2) / (W // 2))
    shapes = {"x": (B, S, M), "norm1": (M,), "wqkv": (M, N), "bqkv": (N,), "wo": (H * W, M), "gate1": (M,), "post1": (M,),
              "norm2": (M,), "w1": (M, F), "b1": (F,), "w2": (F, M), "b2": (M,)}
    host, val = {}, {}
    for name, shape in shapes.items():
        near_one = name.startswith(("norm", "post", "gate"))
        host[name], val[name] = draw(kind, rng, shape, 0.1 if near_one or name[0] == "b" else shape[0] ** -0.5 if name[0] == "w" else 1.0,
                                     1.0 if near_one else 0.0)
    g, gv = draw(kind, rng, (B, S, M), 1.0)
    d = {k: C.to_device(v) for k, v in host.items()}
    dg, pos = C.to_device(g), C.to_device(np.broadcast_to(np.arange(S, dtype=np.int32), (1, B, S)).copy())
    fr = C.to_device(freqs)
    new = lambda *s: C.empty(s, NP[kind])

    def parts(t):
        return [t.view((B, n, S, W), (S * N, W, N, 1), at * W) for at, n in ((0, H), (H, KV), (H + KV, KV))]

    def step():
        norm1, post1, norm2 = C.Norm("rms", d["norm1"]), C.Norm("rms", d["post1"]), C.Norm("rms", d["norm2"])
        _, h1 = C.residual_norm(d["x"], pre=norm1, eps=EPS)
        qkv = C.dense(h1, d["wqkv"], d["bqkv"])
        q, k, v = parts(qkv)
        C.rotary([q, k], pos, fr, [W // 2], "halves", out=[q, k])
        flat = new(B, S, H * W)
        o, lse = C.window_attention(q, k, v, window, sinks, scale, o=flat.view((B, H, S, W), (S * H * W, W, H * W, 1)), lse=True)
        b1 = C.dense(flat, d["wo"])
        u, h2 = C.residual_norm(d["x"], b1, post1, d["gate1"], 0.5, norm2, EPS)
        y, z = C.dense(h2, d["w1"], d["b1"], "gelu", z=True)
        out = C.dense(y, d["w2"], d["b2"], None, u)
        # backwards
        dy, dw2, db2 = C.dense_adjoint(y, d["w2"], dg)
        dh2, dw1, db1 = C.dense_adjoint(h2, d["w1"], dy, z, "gelu")
        dx, dblock, dgate, dpost, dnorm2 = C.residual_norm_adjoint(u, b1, post1, d["gate1"], 0.5, norm2, dg, dh2)
        dflat, dwo, _ = C.dense_adjoint(flat, d["wo"], dblock, want_dbias=False)
        dqkv = new(B, S, N)
        gq, gk, gvv = parts(dqkv)
        C.window_attention_adjoint(q, k, v, o, lse, dflat.view((B, H, S, W), (S * H * W, W, H * W, 1)), window, sinks, scale, gq, gk, gvv)
        C.rotary_adjoint([gq, gk], pos, fr, [W // 2], "halves", out=[gq, gk])
        dh1, dwqkv, dbqkv = C.dense_adjoint(h1, d["wqkv"], dqkv)
        dx0, _, _, _, dnorm1 = C.residual_norm_adjoint(d["x"], pre=norm1, du=dx, dh=dh1)
        grads = {"norm1": dnorm1[0], "wqkv": dwqkv, "bqkv": dbqkv, "wo": dwo, "gate1": dgate, "post1": dpost[0],
                 "norm2": dnorm2[0], "w1": dw1, "b1": db1, "w2": dw2, "b2": db2}
        names = list(grads)
        norm = C.gradient_norm([grads[n] for n in names])
        return {"out": out, "x": dx0, **grads}, norm, names

    got, norm, names = step()
    want_out, want = torch_step(val, gv, B, S, H, KV, W, window, sinks, freqs, scale)
    bar = 24 * 2 * (2.0**-11 if kind == "f16" else 2.0**-8)
    for name, t in got.items():
        a, b = decode(kind, t.numpy()), want_out if name == "out" else want[name]
        assert np.linalg.norm(a - b) <= bar * np.linalg.norm(b) + 2.0**-10, (name, np.linalg.norm(a - b) / np.linalg.norm(b))
    # the norm is that of the stored gradients, and clipping makes it the bound
    stored = math.sqrt(sum((decode(kind, got[n].numpy()) ** 2).sum() for n in names))
    assert abs(float(norm.numpy()) - stored) <= 2.0**-23 * stored
    C.clip_gradients([got[n] for n in names], norm, 0.25 * stored)
    after = float(C.gradient_norm([got[n] for n in names]).numpy())
    u = 2.0**-11 if kind == "f16" else 2.0**-8
    small = math.sqrt(sum(got[n].size for n in names)) * 2.0**-25  # binary16's own least rounding
    assert abs(after - 0.25 * stored) <= u * 0.25 * stored + small
