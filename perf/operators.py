"""The training and serving operators of a transformer block with positions
and a sliding window, as a program that holds its data in torch tensors gives
them to the package: layer norm with its row statistics and its gradients,
rotary positions over several axes and their gradient, and attention with a
sliding window and always-visible first tokens, for prompts, for gradients
and for single tokens over a cache.

Every case is a dict of plain values; "kind" names the call and the other
entries its sizes and options. With `own` false a pass is computed from
elementary torch operations, with `own` true by the package's entry points
over borrowed device tensors that the caller keeps.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16, "f16": torch.float16,
         "i32": torch.int32}
WIDTH = {"f32": 4, "f64": 8, "bf16": 2, "f16": 2}
EPS = 1e-5
BASE = 10000.0   # rotary frequencies BASE^(-p / pairs)
BLOCK = 512      # query rows the plain attention takes at a time


def listed():
    return [
        # a few tokens through one norm of a narrow 16-bit model: launch latency
        {"name": "norm_bf16_64x512", "kind": "norm", "rows": 64, "n": 512, "dtype": "bf16", "weights": "bf16"},
        # a norm's forward in training, rows that are no power of two
        {"name": "norm_f32_20000x1000", "kind": "norm", "rows": 20000, "n": 1000, "dtype": "f32", "weights": "f32"},
        # the gradients of a norm of the transformer block's eight full sequences
        {"name": "norm_adjoint_f32_4096x1024", "kind": "norm_adjoint", "rows": 4096, "n": 1024, "dtype": "f32",
         "weights": "f32"},
        # the same over a large 16-bit batch whose weights are held in 32 bits
        {"name": "norm_adjoint_bf16_65536x1024", "kind": "norm_adjoint", "rows": 65536, "n": 1024, "dtype": "bf16",
         "weights": "f32"},
        # one new token for each of 64 sequences, far into their texts: launch latency
        {"name": "rotary_bf16_64x1", "kind": "rotary", "batch": 64, "seq": 1, "heads": 16, "kv_heads": 4, "dh": 128,
         "sections": "16,24,24", "pairing": "halves", "dtype": "bf16"},
        # the gradient over a video of 8 frames of 32 x 32 patches, time / height / width
        {"name": "rotary_adjoint_f32_2x8192", "kind": "rotary_adjoint", "batch": 2, "seq": 8192, "heads": 16,
         "kv_heads": 16, "dh": 64, "sections": "8,12,12", "pairing": "adjacent", "dtype": "f32"},
        # the prefill of the transformer block with a window
        {"name": "window_f32_8x16x512x64", "kind": "window", "batch": 8, "heads": 16, "kv_heads": 16, "seq": 512,
         "keys": 512, "dh": 64, "window": 128, "sinks": 4, "ragged": False, "dtype": "f32"},
        # a long prompt with grouped heads
        {"name": "window_bf16_2x16x8192x128", "kind": "window", "batch": 2, "heads": 16, "kv_heads": 4, "seq": 8192,
         "keys": 8192, "dh": 128, "window": 1024, "sinks": 4, "ragged": False, "dtype": "bf16"},
        # gradients of a padded batch, head width and lengths off every tile
        {"name": "window_adjoint_f16_3x12x1000x96", "kind": "window_adjoint", "batch": 3, "heads": 12, "kv_heads": 6,
         "seq": 1000, "keys": 1000, "dh": 96, "window": 300, "sinks": 7, "ragged": True, "dtype": "f16"},
        # gradients of a long training sequence
        {"name": "window_adjoint_bf16_1x16x8192x128", "kind": "window_adjoint", "batch": 1, "heads": 16, "kv_heads": 4,
         "seq": 8192, "keys": 8192, "dh": 128, "window": 1024, "sinks": 4, "ragged": False, "dtype": "bf16"},
        # one token of one conversation
        {"name": "token_bf16_1x16x4096x128", "kind": "window", "batch": 1, "heads": 16, "kv_heads": 4, "seq": 1,
         "keys": 4096, "dh": 128, "window": 1024, "sinks": 4, "ragged": True, "dtype": "bf16"},
        # one token for each of 64 conversations of different lengths
        {"name": "token_bf16_64x32x16384x128", "kind": "window", "batch": 64, "heads": 32, "kv_heads": 8, "seq": 1,
         "keys": 16384, "dh": 128, "window": 4096, "sinks": 16, "ragged": True, "dtype": "bf16"},
    ]


def _size(rng, lo, hi, step=8):
    """A size in [lo, hi], spread over its logarithm; half of them whole
    multiples of `step`, the others as they fall."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))
    if rng.random() < 0.5:
        v = (v + step // 2) // step * step
    return max(lo, min(hi, v))


def _drawn(rng):
    kind = rng.choice(["norm", "norm_adjoint", "norm_adjoint", "rotary", "rotary_adjoint", "window", "window",
                       "window_adjoint", "window_adjoint", "token"])
    if kind in ("norm", "norm_adjoint"):
        n = _size(rng, 64, 20000, 64)
        dtype = rng.choice(["f32", "bf16", "bf16", "f16", "f64"])
        return {"kind": kind, "rows": _size(rng, 1, max(2, min(65536, 40000000 // n))), "n": n, "dtype": dtype,
                "weights": rng.choice([dtype, "f32"]) if WIDTH[dtype] == 2 else dtype}
    if kind in ("rotary", "rotary_adjoint"):
        pairs = rng.choice([16, 24, 32, 36, 40, 48, 64])
        axes = rng.choice([1, 2, 3])
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        heads = rng.choice([4, 8, 12, 16])
        return {"kind": kind, "batch": _size(rng, 1, 8, 2), "seq": _size(rng, 1, 8192, 64), "heads": heads,
                "kv_heads": heads // rng.choice([1, 2, 4]), "dh": 2 * pairs + 8 * rng.choice([0, 0, 2, 4]),
                "sections": ",".join(map(str, sections)), "pairing": rng.choice(["halves", "halves", "adjacent"]),
                "dtype": rng.choice(["f32", "bf16", "bf16", "f16"])}
    group = rng.choice([1, 2, 4, 4])
    heads = group * rng.choice([1, 2, 3, 4])
    case = {"kind": kind, "heads": heads, "kv_heads": heads // group, "dh": rng.choice([64, 64, 72, 96, 128, 128]),
            "window": _size(rng, 16, 4096, 64), "sinks": rng.choice([0, 1, 4, 4, 16, 70]),
            "ragged": rng.random() < 0.5, "dtype": rng.choice(["f32", "bf16", "bf16", "f16"])}
    if kind == "token":
        case.update(kind="window", batch=_size(rng, 1, 128, 8), seq=1, keys=_size(rng, 64, 16384, 64),
                    dtype=rng.choice(["f32", "bf16", "bf16", "f16"]))
        return case
    seq = _size(rng, 2, 8192, 64)
    case.update(batch=_size(rng, 1, 8, 2), seq=seq, keys=seq)
    if kind == "window" and rng.random() < 0.4:  # a chunk of new tokens at the end of longer texts
        case["keys"] = min(16384, seq + _size(rng, 1, 4096, 64))
    return case


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / {"f32": 5e13, "f64": 2e13}.get(case["dtype"], 5e14)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _drawn(rng)
        if _cost(case) <= most:
            return case


# ---------------------------------------------------------------- lengths and visible keys
def _lengths(case):
    """Valid keys of each sequence: the whole extent, or from it down to half
    of it (never below a chunk's own rows)."""
    k, b = case["keys"], case["batch"]
    if not case["ragged"]:
        return [k] * b
    least = 1 if case["kind"] == "window_adjoint" else case["seq"]
    return [max(least, k - (2 * i + 1) * k // (4 * b)) for i in range(b)]


def _starts(case):
    """The position of each sequence's first query row: 0 for a training
    batch padded at its end, else the rows are the sequence's last."""
    if case["kind"] == "window_adjoint":
        return [0] * case["batch"]
    return [n - case["seq"] for n in _lengths(case)]


def _pairs(case):
    """Visible (row, key) pairs of one head, summed over the batch."""
    total, w, s = 0, case["window"], case["sinks"]
    for n, first in zip(_lengths(case), _starts(case)):
        p = torch.arange(first, min(first + case["seq"], n), dtype=torch.int64)
        recent = (p + 1).clamp_max(w)
        early = (p + 1 - w).clamp(0, s)
        total += int((recent + early).sum())
    return total


def _read_keys(case):
    """Keys that some row of their sequence sees, summed over the batch."""
    total, w, s = 0, case["window"], case["sinks"]
    for n, first in zip(_lengths(case), _starts(case)):
        lo = max(0, first - w + 1)
        total += n - lo + min(s, lo)
    return total


# ---------------------------------------------------------------- inputs
def _tensors(case, seed):
    """The case's inputs on the GPU, by name, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 29)
    kind, dt = case["kind"], TORCH[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, dtype=dt):
        draws = torch.float64 if dtype == torch.float64 else torch.float32
        return (torch.randn(*shape, generator=g, device="cuda", dtype=draws) * scale + mean).to(dtype)

    if kind in ("norm", "norm_adjoint"):
        n, rows, wt = case["n"], case["rows"], TORCH[case["weights"]]
        t = {"x": normal(rows, n, scale=1.5, mean=0.25), "gamma": normal(n, scale=0.1, mean=1.0, dtype=wt)}
        if kind == "norm":
            t["beta"] = normal(n, scale=0.1, dtype=wt)
            return t
        t["g"] = normal(rows, n, scale=0.01)
        acc = torch.float64 if dt == torch.float64 else torch.float32
        x = t["x"].double()
        mean = x.mean(-1, keepdim=True)
        t["rstd"] = ((x - mean).square_().mean(-1) + EPS).rsqrt_().to(acc)
        t["mean"] = mean.squeeze(-1).to(acc)
        return t
    b, s, d = case["batch"], case["seq"], case["dh"]
    if kind in ("rotary", "rotary_adjoint"):
        sections = [int(v) for v in case["sections"].split(",")]
        axes, pairs = len(sections), sum(sections)
        t = {"q": normal(b, s, case["heads"], d), "k": normal(b, s, case["kv_heads"], d),
             "freqs": BASE ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)}
        i = torch.arange(s, device="cuda")
        side = max(1, int(math.isqrt(max(1, s // 8))))
        grid = [i // (side * side), i // side % side, i % side][:axes] if axes > 1 else [i]
        # each sequence goes on from its own place in a long text
        first = torch.randint(0, 100000, (b,), generator=g, device="cuda")
        t["positions"] = torch.stack([first[:, None] + p[None, :] for p in grid]).int()
        return t
    kv, n = case["kv_heads"], case["keys"]
    t = {"q": normal(b, s, case["heads"], d, scale=1.5)}
    if kind == "window":  # a cache: each head's keys side by side
        t["k"], t["v"] = normal(b, kv, n, d), normal(b, kv, n, d)
    else:
        t["k"], t["v"] = normal(b, n, kv, d), normal(b, n, kv, d)
        t["g"] = normal(b, s, case["heads"], d, scale=0.01)
    if case["ragged"]:
        t["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
    if kind == "window_adjoint":
        t["starts"] = torch.tensor(_starts(case), device="cuda", dtype=torch.int32)
        o, lse = _attend(case, t, torch.float64)
        t["o"], t["lse"] = o.transpose(1, 2).to(dt), lse.float()
    return t


def _heads_first(t, name):
    """[batch, heads, seq, dh] view of an input stored either way."""
    return t[name].transpose(1, 2)


def _kv(case, t):
    return (t["k"], t["v"]) if case["kind"] == "window" else (_heads_first(t, "k"), _heads_first(t, "v"))


# ---------------------------------------------------------------- the plain form
def _blocks(case):
    """For each block of query rows: (i0, i1, idx [batch, L] key indices,
    mask [batch, rows, L] of visible pairs), every visible key once."""
    b, s, n, w, sinks = case["batch"], case["seq"], case["keys"], case["window"], case["sinks"]
    start = torch.tensor(_starts(case), device="cuda")[:, None]
    length = torch.tensor(_lengths(case), device="cuda")[:, None, None]
    for i0 in range(0, s, BLOCK):
        i1 = min(s, i0 + BLOCK)
        p = (start + torch.arange(i0, i1, device="cuda"))[:, :, None]
        span = w + (i1 - i0) - 1
        if span + sinks >= n:
            idx = torch.arange(n, device="cuda").expand(b, n)
            j = idx[:, None, :]
            mask = (j <= p) & (p < length) & ((p - j < w) | (j < sinks))
        else:
            near = start + i1 - span + torch.arange(span, device="cuda")
            early = torch.arange(sinks, device="cuda").expand(b, sinks)
            idx = torch.cat([early, near], 1)
            j = idx[:, None, :]
            seen = (j >= 0) & (j <= p) & (p < length) & ((p - j < w) | (j < sinks))
            once = torch.cat([torch.ones_like(early, dtype=torch.bool), near >= sinks], 1)[:, None, :]
            mask = seen & once
            idx = idx.clamp(0, n - 1)
        yield i0, i1, idx, mask


def _picked(x, idx):
    """x [batch, heads, keys, dh] at the key indices of each sequence."""
    b, h, _, d = x.shape
    return torch.gather(x, 2, idx[:, None, :, None].expand(b, h, idx.shape[1], d))


def _attend(case, t, acc):
    """o [batch, heads, seq, dh] and lse [batch, heads, seq] at `acc`."""
    b, h, kv, s, d = case["batch"], case["heads"], case["kv_heads"], case["seq"], case["dh"]
    k, v = _kv(case, t)
    q = _heads_first(t, "q")
    o = torch.empty(b, h, s, d, device="cuda", dtype=acc)
    lse = torch.empty(b, h, s, device="cuda", dtype=acc)
    for i0, i1, idx, mask in _blocks(case):
        r = i1 - i0
        qb = q[:, :, i0:i1].to(acc).reshape(b, kv, h // kv * r, d)
        kb, vb = _picked(k, idx).to(acc), _picked(v, idx).to(acc)
        x = (qb @ kb.transpose(2, 3).contiguous()).reshape(b, h, r, -1) * d ** -0.5
        x = x.masked_fill(~mask[:, None], -math.inf)
        m = x.amax(-1, keepdim=True)
        e = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
        total = e.sum(-1, keepdim=True)
        y = (e.reshape(b, kv, -1, e.shape[-1]) @ vb).reshape(b, h, r, d)
        o[:, :, i0:i1] = torch.where(total > 0, y / total, torch.zeros_like(y))
        lse[:, :, i0:i1] = (torch.log(total) + m).squeeze(-1)
    return o, lse


def _attend_adjoint(case, t):
    b, h, kv, s, d = case["batch"], case["heads"], case["kv_heads"], case["seq"], case["dh"]
    k, v = _kv(case, t)
    q, o, g = (_heads_first(t, n) for n in ("q", "o", "g"))
    dq = torch.empty(b, h, s, d, device="cuda")
    dk, dv = (torch.zeros(b, kv, case["keys"], d, device="cuda") for _ in range(2))
    for i0, i1, idx, mask in _blocks(case):
        r = i1 - i0
        qb, ob, gb = (x[:, :, i0:i1].float().reshape(b, kv, h // kv * r, d) for x in (q, o, g))
        kb, vb = _picked(k, idx).float(), _picked(v, idx).float()
        x = (qb @ kb.transpose(2, 3).contiguous()).reshape(b, h, r, -1) * d ** -0.5
        p = torch.exp(x - t["lse"][:, :, i0:i1, None]).masked_fill(~mask[:, None], 0.0)
        p = p.reshape(b, kv, h // kv * r, -1)
        ds = p * ((gb @ vb.transpose(2, 3).contiguous()) - (gb * ob).sum(-1, keepdim=True)) * d ** -0.5
        dq[:, :, i0:i1] = (ds @ kb).reshape(b, h, r, d)
        where = idx[:, None, :, None].expand(b, kv, idx.shape[1], d)
        dk.scatter_add_(2, where, ds.transpose(2, 3).contiguous() @ qb)
        dv.scatter_add_(2, where, p.transpose(2, 3).contiguous() @ gb)
    return dq, dk, dv


def _rotate(x, positions, freqs, sections, pairing, sign):
    """x [batch, seq, heads, dh], the first 2 * pairs of dh turned."""
    pairs = freqs.numel()
    axis = torch.repeat_interleave(torch.arange(len(sections), device="cuda"),
                                   torch.tensor(sections, device="cuda"))
    angle = positions.double()[axis].permute(1, 2, 0) * freqs * sign
    c, s = torch.cos(angle).to(x.dtype)[:, :, None], torch.sin(angle).to(x.dtype)[:, :, None]
    y = x.clone()
    if pairing == "halves":
        u, v = x[..., :pairs], x[..., pairs:2 * pairs]
        y[..., :pairs], y[..., pairs:2 * pairs] = u * c - v * s, u * s + v * c
    else:
        u, v = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = u * c - v * s, u * s + v * c
    return y


def _plain(case, t):
    kind, dt = case["kind"], TORCH[case["dtype"]]
    acc = torch.float64 if dt == torch.float64 else torch.float32
    if kind == "norm":
        x = t["x"].to(acc)
        mean = x.mean(-1, keepdim=True)
        c = x - mean
        rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)
        y = c * rstd * t["gamma"].to(acc) + t["beta"].to(acc)
        return {"y": y.to(dt), "mean": mean.squeeze(-1), "rstd": rstd.squeeze(-1)}
    if kind == "norm_adjoint":
        x, g, wt = t["x"].to(acc), t["g"].to(acc), t["gamma"].dtype
        hat = (x - t["mean"][:, None]) * t["rstd"][:, None]
        gg = g * t["gamma"].to(acc)
        dx = t["rstd"][:, None] * (gg - gg.mean(-1, keepdim=True) - hat * (gg * hat).mean(-1, keepdim=True))
        return {"dx": dx.to(dt), "dgamma": (g * hat).sum(0).to(wt), "dbeta": g.sum(0).to(wt)}
    if kind in ("rotary", "rotary_adjoint"):
        sections = [int(v) for v in case["sections"].split(",")]
        sign = 1 if kind == "rotary" else -1
        return {n: _rotate(t[n].to(acc), t["positions"], t["freqs"], sections, case["pairing"], sign).to(dt)
                for n in ("q", "k")}
    if kind == "window":
        o, lse = _attend(case, t, torch.float32)
        return {"o": o.transpose(1, 2).to(dt), "lse": lse}
    dq, dk, dv = _attend_adjoint(case, t)
    return {"dq": dq.transpose(1, 2).to(dt), "dk": dk.transpose(1, 2).to(dt), "dv": dv.transpose(1, 2).to(dt)}


# ---------------------------------------------------------------- the package's calls
def _results(case):
    """name -> (shape, torch dtype) of the case's results."""
    kind, dt = case["kind"], TORCH[case["dtype"]]
    acc = torch.float64 if dt == torch.float64 else torch.float32
    if kind in ("norm", "norm_adjoint"):
        n, rows, wt = case["n"], case["rows"], TORCH[case["weights"]]
        if kind == "norm":
            return {"y": ((rows, n), dt), "mean": ((rows,), acc), "rstd": ((rows,), acc)}
        return {"dx": ((rows, n), dt), "dgamma": ((n,), wt), "dbeta": ((n,), wt)}
    b, s, h, kv, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dh"]
    if kind in ("rotary", "rotary_adjoint"):
        return {"q": ((b, s, h, d), dt), "k": ((b, s, kv, d), dt)}
    if kind == "window":
        return {"o": ((b, s, h, d), dt), "lse": ((b, h, s), torch.float32)}
    return {"dq": ((b, s, h, d), dt), "dk": ((b, case["keys"], kv, d), dt), "dv": ((b, case["keys"], kv, d), dt)}


def _wrap(C, t):
    """A torch tensor's storage as a borrowed device tensor of the library."""
    import numpy as np
    names = {torch.float32: np.float32, torch.float64: np.float64, torch.bfloat16: np.uint16,
             torch.float16: np.float16, torch.int32: np.int32}
    return C.borrow(tuple(t.shape), names[t.dtype], t.data_ptr(), t.numel() * t.element_size())


def _by_head(x):
    """The [batch, heads, seq, dh] view of a wrapped [batch, seq, heads, dh] tensor."""
    b, s, h, d = x.shape
    return x.view((b, h, s, d), (s * h * d, d, h * d, 1))


def prepare(case, seed):
    t = {k: v.contiguous() for k, v in _tensors(case, seed).items()}
    state = {"case": case, "in": t}
    if own:
        import chelis_amd as C
        out = {k: torch.zeros(shape, dtype=dt, device="cuda") for k, (shape, dt) in _results(case).items()}
        i, o = {k: _wrap(C, v) for k, v in t.items()}, {k: _wrap(C, v) for k, v in out.items()}
        # heads lie inside the sequence axis of what the projections write and read
        if case["kind"] not in ("norm", "norm_adjoint"):
            stored = ("q", "k", "v", "o", "g") if case["kind"] == "window_adjoint" else \
                ("q", "k") if case["kind"].startswith("rotary") else ("q",)
            i.update({k: _by_head(i[k]) for k in stored})
            o.update({k: _by_head(o[k]) for k in o if k != "lse"})
        state.update(C=C, wrapped=i, to=o, out=out)
        # the library works on its own stream: what torch has in flight is finished first
        torch.cuda.synchronize()
    return state


def run(state):
    case = state["case"]
    if not own:
        return _plain(case, state["in"])
    C, i, o, kind = state["C"], state["wrapped"], state["to"], case["kind"]
    if kind == "norm":
        C.layer_norm_stats(i["x"], i["gamma"], i["beta"], EPS, o["y"], o["mean"], o["rstd"])
    elif kind == "norm_adjoint":
        C.layer_norm_adjoint(i["x"], i["gamma"], i["mean"], i["rstd"], i["g"], o["dx"], o["dgamma"], o["dbeta"])
    elif kind in ("rotary", "rotary_adjoint"):
        turn = C.rotary if kind == "rotary" else C.rotary_adjoint
        turn([i["q"], i["k"]], i["positions"], i["freqs"], [int(v) for v in case["sections"].split(",")],
             case["pairing"], [o["q"], o["k"]])
    elif kind == "window":
        C.window_attention(i["q"], i["k"], i["v"], case["window"], case["sinks"], case["dh"] ** -0.5, o["o"],
                           o["lse"], lengths=i.get("lengths"))
    else:
        C.window_attention_adjoint(i["q"], i["k"], i["v"], i["o"], i["lse"], i["g"], case["window"], case["sinks"],
                                   case["dh"] ** -0.5, o["dq"], o["dk"], o["dv"], lengths=i.get("lengths"),
                                   starts=i["starts"])
    return state["out"]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, w = case["kind"], WIDTH[case["dtype"]]
    acc = 8 if case["dtype"] == "f64" else 4
    if kind in ("norm", "norm_adjoint"):
        rows, n, ww = case["rows"], case["n"], WIDTH[case["weights"]]
        if kind == "norm":
            return {"bytes": 2 * w * rows * n + 2 * ww * n + 2 * acc * rows, "flops": 8 * rows * n}
        return {"bytes": 3 * w * rows * n + 3 * ww * n + 2 * acc * rows, "flops": 14 * rows * n}
    b, s, h, kv, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dh"]
    if kind in ("rotary", "rotary_adjoint"):
        sections = case["sections"].split(",")
        pairs = sum(int(v) for v in sections)
        return {"bytes": 2 * w * b * s * (h + kv) * d + 4 * len(sections) * b * s + 8 * pairs,
                "flops": 6 * b * s * (h + kv) * pairs}
    per_row, per_key = b * s * h, kv * d * w
    if kind == "window":
        return {"bytes": 2 * w * per_row * d + 4 * per_row + 2 * per_key * _read_keys(case),
                "flops": 4 * d * h * _pairs(case)}
    valid = sum(min(n, s) for n in _lengths(case))
    return {"bytes": w * d * h * (3 * valid + b * s) + 4 * h * valid + per_key * (2 * _read_keys(case) + 2 * b * case["keys"]),
            "flops": 10 * d * h * _pairs(case)}


# ---------------------------------------------------------------- the same in 64 bits
def _exact_attention(case, raw):
    """The definition over whole key rows, one shared head of one sequence at
    a time: forward, or the gradients of the stored o and lse."""
    b, h, kv, s, n, d = (case[k] for k in ("batch", "heads", "kv_heads", "seq", "keys", "dh"))
    forward, scale, group = case["kind"] == "window", case["dh"] ** -0.5, case["heads"] // case["kv_heads"]
    new = lambda *shape: torch.zeros(*shape, device="cuda", dtype=torch.float64)
    if forward:
        out = {"o": new(b, s, h, d), "lse": new(b, h, s)}
    else:
        out = {"dq": new(b, s, h, d), "dk": new(b, n, kv, d), "dv": new(b, n, kv, d)}
    key = torch.arange(n, device="cuda")
    for z, (length, first) in enumerate(zip(_lengths(case), _starts(case))):
        for c in range(kv):
            keys, values = (raw[m][z, c] if forward else raw[m][z, :, c] for m in ("k", "v"))
            keys, values = keys.double(), values.double()
            for i in range(0, s, 1024):
                rows = slice(i, min(s, i + 1024))
                place = first + torch.arange(rows.start, rows.stop, device="cuda")[:, None]
                hidden = (key > place) | (place >= length) | ((place - key >= case["window"]) & (key >= case["sinks"]))
                for head in range(c * group, (c + 1) * group):
                    q = raw["q"][z, rows, head].double()
                    scores = (q @ keys.T * scale).masked_fill(hidden, -math.inf)
                    if forward:
                        lse = torch.logsumexp(scores, 1)
                        weights = torch.exp(scores - lse[:, None]).masked_fill(hidden, 0.0)
                        out["o"][z, rows, head] = weights @ values
                        out["lse"][z, head, rows] = lse
                        continue
                    g = raw["g"][z, rows, head].double()
                    dot = (g * raw["o"][z, rows, head].double()).sum(1, keepdim=True)
                    weights = torch.exp(scores - raw["lse"][z, head, rows, None].double()).masked_fill(hidden, 0.0)
                    ds = weights * (g @ values.T - dot) * scale
                    out["dq"][z, rows, head] = ds @ keys
                    out["dk"][z, :, c] += ds.T @ q
                    out["dv"][z, :, c] += weights.T @ g
    return out


def exact(case, seed):
    kind, raw = case["kind"], _tensors(case, seed)
    if kind in ("window", "window_adjoint"):
        return _exact_attention(case, raw)
    if kind == "norm":
        x = raw["x"].double()
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        rstd = (var + EPS) ** -0.5
        return {"y": (x - mean) * rstd * raw["gamma"].double() + raw["beta"].double(), "mean": mean[:, 0],
                "rstd": rstd[:, 0]}
    if kind == "norm_adjoint":
        r, x, g = raw["rstd"].double()[:, None], raw["x"].double(), raw["g"].double()
        unit = (x - raw["mean"].double()[:, None]) * r
        weighted = g * raw["gamma"].double()
        n = case["n"]
        dx = (weighted - weighted.sum(1, keepdim=True) / n - unit * ((weighted * unit).sum(1, keepdim=True) / n)) * r
        return {"dx": dx, "dgamma": (g * unit).sum(0), "dbeta": g.sum(0)}
    # a pair as a complex number, turned by multiplying with exp(+-i angle)
    sections = [int(v) for v in case["sections"].split(",")]
    pairs, turn, out = sum(sections), 1.0 if kind == "rotary" else -1.0, {}
    place = torch.cat([raw["positions"][a].double()[..., None].expand(-1, -1, c) for a, c in enumerate(sections)], -1)
    unit = torch.polar(torch.ones_like(place), place * raw["freqs"] * turn)[:, :, None]
    for name in ("q", "k"):
        x = raw[name].double()
        y = x.clone()
        if case["pairing"] == "halves":
            z = torch.complex(x[..., :pairs].contiguous(), x[..., pairs:2 * pairs].contiguous()) * unit
            y[..., :2 * pairs] = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.complex(x[..., 0:2 * pairs:2].contiguous(), x[..., 1:2 * pairs:2].contiguous()) * unit
            y[..., :2 * pairs] = torch.stack([z.real, z.imag], -1).flatten(-2)
        out[name] = y
    return out
