"""The training step of a transformer block in 16 bits around its attention,
as a program that holds its data in torch tensors gives it to the package:
matrix products with bias, activation and residual and their gradients, the
residual stream between two blocks (norm of the block's result, gate, scale,
sum, norm before the next block) and its gradients, and the global norm of all
gradients with clipping.

Every case is a dict of plain values; "kind" names the call and the other
entries its sizes and options. With `own` false a pass is computed from
elementary torch operations, with `own` true by the package's entry points
over borrowed device tensors that the caller keeps.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16, "f16": torch.float16}
WIDTH = {"f32": 4, "f64": 8, "bf16": 2, "f16": 2}
EPS = 1e-5


def listed():
    return [
        # one new token through the first product of a block's two
        {"name": "dense_bf16_1x1024x4096", "kind": "dense", "rows": 1, "k": 1024, "n": 4096, "dtype": "bf16",
         "weights": "kn", "act": "gelu", "bias": True, "residual": False, "z": False},
        # the same in training, eight full sequences, what the gradient needs kept
        {"name": "dense_bf16_4096x1024x4096", "kind": "dense", "rows": 4096, "k": 1024, "n": 4096, "dtype": "bf16",
         "weights": "kn", "act": "gelu", "bias": True, "residual": False, "z": True},
        # a padded batch through sizes off every tile and vector, weights stored along k
        {"name": "dense_f16_1499x1001x2003", "kind": "dense", "rows": 1499, "k": 1001, "n": 2003, "dtype": "f16",
         "weights": "nk", "act": "silu", "bias": True, "residual": True, "z": False},
        # the projection back into the residual stream of a wide model, a long batch
        {"name": "dense_bf16_16384x8192x4096", "kind": "dense", "rows": 16384, "k": 8192, "n": 4096, "dtype": "bf16",
         "weights": "nk", "act": "none", "bias": True, "residual": True, "z": False},
        # the hidden layer of the image classifier, a batch off every power of two
        {"name": "dense_adjoint_f16_1000x784x512", "kind": "dense_adjoint", "rows": 1000, "k": 784, "n": 512,
         "dtype": "f16", "weights": "kn", "act": "relu"},
        # the gradients of the block's first product over 16 full sequences
        {"name": "dense_adjoint_bf16_8192x1024x4096", "kind": "dense_adjoint", "rows": 8192, "k": 1024, "n": 4096,
         "dtype": "bf16", "weights": "kn", "act": "gelu"},
        # the stream between two blocks for a few tokens: launch latency
        {"name": "residual_bf16_64x1024", "kind": "residual", "groups": 1, "rows": 64, "n": 1024, "dtype": "bf16",
         "weights": "bf16", "post": "rms", "pre": "rms", "gate": True},
        # a training batch of rows that are no power of two, no norm behind the block
        {"name": "residual_f32_20000x1000", "kind": "residual", "groups": 1, "rows": 20000, "n": 1000, "dtype": "f32",
         "weights": "f32", "post": "none", "pre": "layer", "gate": False},
        # the gradients of the stream, a gate of its own for each of eight sequences
        {"name": "residual_adjoint_f32_8x512x1024", "kind": "residual_adjoint", "groups": 8, "rows": 512, "n": 1024,
         "dtype": "f32", "weights": "f32", "post": "layer", "pre": "layer", "gate": True},
        # the same over a large 16-bit batch with one gate
        {"name": "residual_adjoint_bf16_65536x1024", "kind": "residual_adjoint", "groups": 1, "rows": 65536, "n": 1024,
         "dtype": "bf16", "weights": "f32", "post": "rms", "pre": "rms", "gate": True},
        # the image classifier's four gradients: launch latency
        {"name": "clip_f32_classifier", "kind": "clip", "blocks": 0, "hidden": 512, "inputs": 784, "outputs": 10,
         "dtype": "f32", "vectors": "f32", "loss_scale": 1, "clips": True},
        # the gradients of a stack of twelve blocks with their embedding, vectors in 32 bits
        {"name": "clip_bf16_12_blocks", "kind": "clip", "blocks": 12, "hidden": 1024, "inputs": 32000, "outputs": 0,
         "dtype": "bf16", "vectors": "f32", "loss_scale": 1, "clips": True},
    ]


def _size(rng, lo, hi, step=8):
    """A size in [lo, hi], spread over its logarithm; half of them whole
    multiples of `step`, the others as they fall."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))
    if rng.random() < 0.5:
        v = (v + step // 2) // step * step
    return max(lo, min(hi, v))


def _drawn(rng):
    kind = rng.choice(["dense", "dense", "dense", "dense_adjoint", "dense_adjoint", "residual", "residual_adjoint",
                       "residual_adjoint", "clip"])
    if kind in ("dense", "dense_adjoint"):
        dtype = rng.choice(["bf16", "bf16", "f16"])
        case = {"kind": kind, "rows": _size(rng, 1, 16384, 64), "k": _size(rng, 32, 8192, 64),
                "n": _size(rng, 32, 8192, 64), "dtype": dtype, "weights": rng.choice(["kn", "nk"]),
                "act": rng.choice(["none", "relu", "gelu", "gelu", "silu"])}
        if kind == "dense":
            case.update(bias=rng.random() < 0.8, residual=rng.random() < 0.4, z=rng.random() < 0.5)
        return case
    if kind in ("residual", "residual_adjoint"):
        n, groups = _size(rng, 64, 20000, 64), rng.choice([1, 1, 2, 8, 32])
        dtype = rng.choice(["f32", "bf16", "bf16", "f16", "f64"])
        pre = rng.choice(["layer", "rms", "rms", "none"])
        return {"kind": kind, "groups": groups, "rows": _size(rng, 1, max(2, min(65536, 40000000 // n) // groups)),
                "n": n, "dtype": dtype, "weights": rng.choice([dtype, "f32"]) if WIDTH[dtype] == 2 else dtype,
                "post": rng.choice(["none", "layer", "rms"]), "pre": pre, "gate": pre == "none" or rng.random() < 0.6}
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    return {"kind": kind, "blocks": rng.choice([0, 1, 2, 4, 12, 24]), "hidden": _size(rng, 32, 1400, 64),
            "inputs": _size(rng, 10, 50000), "outputs": rng.choice([0, 10, 1000]), "dtype": dtype,
            "vectors": rng.choice([dtype, "f32"]), "loss_scale": 1024 if dtype == "f16" else 1,
            "clips": rng.random() < 0.7}


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / (1e15 if case["kind"].startswith("dense") else 2e13)


def draw(rng):
    most = {}
    for c in listed():
        kind = c["kind"].split("_")[0]
        most[kind] = max(most.get(kind, 0), _cost(c))
    while True:
        case = _drawn(rng)
        if _cost(case) <= most[case["kind"].split("_")[0]]:
            return case


# ---------------------------------------------------------------- inputs
def _gradient_shapes(case):
    """(shape, is a matrix) of every gradient: an input layer, `blocks`
    transformer blocks, an output layer."""
    h = case["hidden"]
    shapes = [((case["inputs"], h), True)]
    if case["blocks"] == 0:
        shapes.append(((h,), False))
    for _ in range(case["blocks"]):
        shapes += [((h,), False)] * 4 + [((h, h), True), ((h,), False)] * 4
        shapes += [((h, 4 * h), True), ((4 * h,), False), ((4 * h, h), True), ((h,), False)]
    if case["outputs"]:
        shapes += [((h, case["outputs"]), True), ((case["outputs"],), False)]
    return shapes


GRADIENT = 0.01  # of the scaled-down loss


def _slices(case):
    """For every gradient: the buffer its clipped values lie in ("matrices"
    or "vectors", each one run of memory as an optimizer keeps it), its first
    element there and its shape."""
    at = {"matrices": 0, "vectors": 0}
    for shape, matrix in _gradient_shapes(case):
        buffer = "matrices" if matrix else "vectors"
        yield buffer, at[buffer], shape
        at[buffer] += math.prod(shape)


def _totals(case):
    total = {"matrices": 0, "vectors": 0}
    for buffer, _, shape in _slices(case):
        total[buffer] += math.prod(shape)
    return {k: v for k, v in total.items() if v}


def _max_norm(case):
    count = sum(math.prod(s) for s, _ in _gradient_shapes(case))
    return GRADIENT * math.sqrt(count) * (0.25 if case["clips"] else 4.0)


def _tensors(case, seed):
    """The case's inputs on the GPU, by name, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 71)
    kind, dt = case["kind"], TORCH[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, dtype=dt):
        draws = torch.float64 if dtype == torch.float64 else torch.float32
        return (torch.randn(*shape, generator=g, device="cuda", dtype=draws) * scale + mean).to(dtype)

    if kind == "clip":
        return {f"g{i}": normal(*shape, scale=GRADIENT * case["loss_scale"],
                                dtype=TORCH[case["dtype" if matrix else "vectors"]])
                for i, (shape, matrix) in enumerate(_gradient_shapes(case))}
    if kind in ("dense", "dense_adjoint"):
        rows, k, n = case["rows"], case["k"], case["n"]
        t = {"x": normal(rows, k), "w": normal(*((k, n) if case["weights"] == "kn" else (n, k)), scale=k ** -0.5)}
        if kind == "dense":
            if case["bias"]:
                t["bias"] = normal(n, scale=0.1)
            if case["residual"]:
                t["residual"] = normal(rows, n, scale=1.5)
            return t
        t["g"] = normal(rows, n, scale=0.01)
        if case["act"] != "none":
            t["z"] = normal(rows, n, scale=1.0)
        return t
    shape, n, wt = (case["groups"], case["rows"], case["n"]), case["n"], TORCH[case["weights"]]
    t = {"b": normal(*shape, scale=0.8, mean=0.1)}
    for place in ("post", "pre"):
        if case[place] != "none":
            t[place + "_gamma"] = normal(n, scale=0.1, mean=1.0, dtype=wt)
        if case[place] == "layer":
            t[place + "_beta"] = normal(n, scale=0.1, dtype=wt)
    if case["gate"]:
        t["gate"] = normal(*((case["groups"], n) if case["groups"] > 1 else (n,)), scale=0.3, mean=0.5, dtype=wt)
    if kind == "residual":
        t["x"] = normal(*shape, scale=1.5, mean=0.25)
        return t
    t["u"] = normal(*shape, scale=1.7, mean=0.3)
    t["du"] = normal(*shape, scale=0.01)
    if case["pre"] != "none":
        t["dh"] = normal(*shape, scale=0.01)
    acc = torch.float64 if dt == torch.float64 else torch.float32
    for place, rows in (("post", t["b"]), ("pre", t["u"])):
        if case[place] == "none":
            continue
        rows = rows.double()
        if case[place] == "layer":
            mean = rows.mean(-1, keepdim=True)
            t[place + "_mean"] = mean.squeeze(-1).to(acc)
            rows = rows - mean
        t[place + "_rstd"] = (rows.square().mean(-1) + EPS).rsqrt_().to(acc)
    return t


SCALE = 0.7  # of a block's result where it joins the stream


# ---------------------------------------------------------------- the plain form
def _act(z, name):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * torch.erfc(z * -0.5 ** 0.5)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * torch.erfc(z * -0.5 ** 0.5) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _matrix(case, t, acc):
    w = t["w"].to(acc)
    return w if case["weights"] == "kn" else w.t()


def _plain_dense(case, t):
    dt = TORCH[case["dtype"]]
    z = t["x"].float() @ _matrix(case, t, torch.float32)
    if case["bias"]:
        z = z + t["bias"].float()
    y = _act(z, case["act"])
    if case["residual"]:
        y = y + t["residual"].float()
    return {"y": y.to(dt), "z": z.to(dt)} if case["z"] else {"y": y.to(dt)}


def _plain_dense_adjoint(case, t):
    dz = t["g"].float()
    if case["act"] != "none":
        dz = dz * _act_slope(t["z"].float(), case["act"])
    w = _matrix(case, t, torch.float32)
    x, dt = t["x"].float(), TORCH[case["dtype"]]
    dw = x.t() @ dz if case["weights"] == "kn" else dz.t() @ x
    return {"dx": (dz @ w.t()).to(dt), "dw": dw.to(dt), "dbias": dz.sum(0).to(dt)}


def _unit(x, kind):
    """The rows of x at zero mean ("layer") and unit size, with the statistics."""
    mean = x.mean(-1, keepdim=True) if kind == "layer" else None
    c = x - mean if kind == "layer" else x
    rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)
    return c * rstd, mean, rstd


def _weighted(hat, t, place):
    y = hat * t[place + "_gamma"].to(hat.dtype)
    return y + t[place + "_beta"].to(hat.dtype) if place + "_beta" in t else y


def _gate(case, t, acc):
    if not case["gate"]:
        return SCALE
    gate = t["gate"].to(acc)
    return SCALE * (gate[:, None] if case["groups"] > 1 else gate)


def _plain_residual(case, t):
    dt = TORCH[case["dtype"]]
    acc = torch.float64 if dt == torch.float64 else torch.float32
    out, v = {}, t["b"].to(acc)
    if case["post"] != "none":
        hat, mean, rstd = _unit(v, case["post"])
        v, out["post_rstd"] = _weighted(hat, t, "post"), rstd.squeeze(-1)
        if mean is not None:
            out["post_mean"] = mean.squeeze(-1)
    u = t["x"].to(acc) + _gate(case, t, acc) * v
    out["u"] = u.to(dt)
    if case["pre"] != "none":
        hat, mean, rstd = _unit(u, case["pre"])
        out["h"], out["pre_rstd"] = _weighted(hat, t, "pre").to(dt), rstd.squeeze(-1)
        if mean is not None:
            out["pre_mean"] = mean.squeeze(-1)
    return out


def _stored_unit(x, t, place):
    x = x - t[place + "_mean"][..., None] if place + "_mean" in t else x
    return x * t[place + "_rstd"][..., None]


def _norm_back(g, hat, t, place):
    """The cotangent of a norm's rows for the cotangent g of their unit rows."""
    c = hat * (g * hat).mean(-1, keepdim=True)
    if place + "_mean" in t:
        c = c + g.mean(-1, keepdim=True)
    return t[place + "_rstd"][..., None] * (g - c)


def _plain_residual_adjoint(case, t):
    dt, wt = TORCH[case["dtype"]], TORCH[case["weights"]]
    acc = torch.float64 if dt == torch.float64 else torch.float32
    out, total = {}, t["du"].to(acc)
    if case["pre"] != "none":
        dh, hat = t["dh"].to(acc), _stored_unit(t["u"].to(acc), t, "pre")
        out["pre_dgamma"] = (dh * hat).sum((0, 1)).to(wt)
        if case["pre"] == "layer":
            out["pre_dbeta"] = dh.sum((0, 1)).to(wt)
        total = total + _norm_back(dh * t["pre_gamma"].to(acc), hat, t, "pre")
    out["dx"] = total.to(dt)
    gated, b = total * _gate(case, t, acc), t["b"].to(acc)
    hat = _stored_unit(b, t, "post") if case["post"] != "none" else b
    if case["gate"]:
        v = _weighted(hat, t, "post") if case["post"] != "none" else b
        dgate = SCALE * (total * v).sum(1)
        out["dgate"] = (dgate if case["groups"] > 1 else dgate[0]).to(wt)
    if case["post"] == "none":
        out["db"] = gated.to(dt)
        return out
    out["post_dgamma"] = (gated * hat).sum((0, 1)).to(wt)
    if case["post"] == "layer":
        out["post_dbeta"] = gated.sum((0, 1)).to(wt)
    out["db"] = _norm_back(gated * t["post_gamma"].to(acc), hat, t, "post").to(dt)
    return out


def _plain_clip(case, t):
    scale = 1.0 / case["loss_scale"]
    total = sum(g.float().square().sum(dtype=torch.float64) for g in t.values())
    norm = scale * torch.sqrt(total)
    factor = scale * torch.where(norm > _max_norm(case), _max_norm(case) / norm, torch.ones_like(norm))
    out = {k: torch.empty(count, device="cuda", dtype=TORCH[case["dtype" if k == "matrices" else "vectors"]])
           for k, count in _totals(case).items()}
    for g, (buffer, first, _) in zip(t.values(), _slices(case)):
        out[buffer][first:first + g.numel()] = (g.float() * factor.float()).flatten()
    out["norm"] = norm.float()
    return out


PLAIN = {"dense": _plain_dense, "dense_adjoint": _plain_dense_adjoint, "residual": _plain_residual,
         "residual_adjoint": _plain_residual_adjoint, "clip": _plain_clip}


# ---------------------------------------------------------------- the package's calls
def _results(case, t):
    """name -> (shape, torch dtype) of the case's results."""
    kind, dt = case["kind"], TORCH[case["dtype"]]
    if kind == "clip":
        out = {k: ((count,), TORCH[case["dtype" if k == "matrices" else "vectors"]])
               for k, count in _totals(case).items()}
        out["norm"] = ((), torch.float32)
        return out
    if kind == "dense":
        shape = (case["rows"], case["n"])
        return {"y": (shape, dt), "z": (shape, dt)} if case["z"] else {"y": (shape, dt)}
    if kind == "dense_adjoint":
        return {"dx": (tuple(t["x"].shape), dt), "dw": (tuple(t["w"].shape), dt), "dbias": ((case["n"],), dt)}
    rows, n, wt = (case["groups"], case["rows"]), case["n"], TORCH[case["weights"]]
    acc = torch.float64 if dt == torch.float64 else torch.float32
    out = {"u": (rows + (n,), dt)} if kind == "residual" else {"dx": (rows + (n,), dt), "db": (rows + (n,), dt)}
    if kind == "residual" and case["pre"] != "none":
        out["h"] = (rows + (n,), dt)
    for place in ("post", "pre"):
        if case[place] == "none":
            continue
        if kind == "residual":
            out[place + "_rstd"] = (rows, acc)
            if case[place] == "layer":
                out[place + "_mean"] = (rows, acc)
        else:
            out[place + "_dgamma"] = ((n,), wt)
            if case[place] == "layer":
                out[place + "_dbeta"] = ((n,), wt)
    if kind == "residual_adjoint" and case["gate"]:
        out["dgate"] = (tuple(t["gate"].shape), wt)
    return out


def _wrap(C, t):
    """A torch tensor's storage as a borrowed device tensor of the library."""
    import numpy as np
    names = {torch.float32: np.float32, torch.float64: np.float64, torch.bfloat16: np.uint16,
             torch.float16: np.float16}
    return C.borrow(tuple(t.shape), names[t.dtype], t.data_ptr(), t.numel() * t.element_size())


def _transposed(x):
    """The [k, n] view of a wrapped [n, k] tensor."""
    n, k = x.shape
    return x.view((k, n), (1, k))


def prepare(case, seed):
    t = _tensors(case, seed)
    state = {"case": case, "in": t}
    if own:
        import chelis_amd as C
        out = {k: torch.zeros(shape, dtype=dt, device="cuda") for k, (shape, dt) in _results(case, t).items()}
        i, o = {k: _wrap(C, v) for k, v in t.items()}, {k: _wrap(C, v) for k, v in out.items()}
        kind = case["kind"]
        if kind == "clip":
            state["grads"] = C.tensor_list([i[k] for k in t])
            strides = lambda shape: tuple(math.prod(shape[a + 1:]) for a in range(len(shape)))
            state["clipped"] = C.tensor_list([o[buffer].view(shape, strides(shape), first)
                                              for buffer, first, shape in _slices(case)])
        elif kind.startswith("dense"):
            if case["weights"] == "nk":  # weights stored along k are a stride swap
                i["w"] = _transposed(i["w"])
                if kind == "dense_adjoint":
                    o["dw"] = _transposed(o["dw"])
        else:
            stats = o if kind == "residual" else i
            for place in ("post", "pre"):
                state[place] = None if case[place] == "none" else C.Norm(
                    case[place], i[place + "_gamma"], i.get(place + "_beta"), stats.get(place + "_mean"),
                    stats[place + "_rstd"])
        state.update(C=C, wrapped=i, to=o, out=out)
        # the library works on its own stream: what torch has in flight is finished first
        torch.cuda.synchronize()
    return state


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return PLAIN[kind](case, state["in"])
    C, i, o = state["C"], state["wrapped"], state["to"]
    if kind == "dense":
        C.dense(i["x"], i["w"], i.get("bias"), case["act"], i.get("residual"), o["y"], o.get("z"))
    elif kind == "dense_adjoint":
        C.dense_adjoint(i["x"], i["w"], i["g"], i.get("z"), case["act"], o["dx"], o["dw"], o["dbias"])
    elif kind == "residual":
        C.residual_norm(i["x"], i["b"], state["post"], i.get("gate"), SCALE, state["pre"], EPS, o["u"], o.get("h"))
    elif kind == "residual_adjoint":
        C.residual_norm_adjoint(i["u"], i["b"], state["post"], i.get("gate"), SCALE, state["pre"], i["du"], i.get("dh"),
                                dx=o["dx"], db=o["db"], dgate=o.get("dgate"),
                                dpost=(o.get("post_dgamma"), o.get("post_dbeta")),
                                dpre=(o.get("pre_dgamma"), o.get("pre_dbeta")))
    else:
        scale = 1.0 / case["loss_scale"]
        C.gradient_norm(state["grads"], scale, o["norm"])
        C.clip_gradients(state["grads"], o["norm"], _max_norm(case), scale, state["clipped"])
    return state["out"]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, w = case["kind"], WIDTH[case["dtype"]]
    if kind == "clip":
        elements = [(math.prod(s), WIDTH[case["dtype" if matrix else "vectors"]])
                    for s, matrix in _gradient_shapes(case)]
        return {"bytes": 2 * sum(c * b for c, b in elements) + 4, "flops": 3 * sum(c for c, _ in elements)}
    if kind == "dense":
        rows, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": w * (rows * k + k * n + case["bias"] * n + rows * n * (1 + case["residual"] + case["z"])),
                "flops": 2 * rows * k * n}
    if kind == "dense_adjoint":
        rows, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": w * (2 * rows * k + 2 * k * n + n + rows * n * (1 + (case["act"] != "none"))),
                "flops": 4 * rows * k * n}
    rows, n, ww, acc = case["groups"] * case["rows"], case["n"], WIDTH[case["weights"]], 8 if w == 8 else 4
    vectors = {"none": 0, "rms": 1, "layer": 2}[case["post"]] + {"none": 0, "rms": 1, "layer": 2}[case["pre"]]
    weights = ww * n * (vectors + case["groups"] * case["gate"])
    if kind == "residual":
        return {"bytes": w * rows * n * (3 + (case["pre"] != "none")) + weights + acc * rows * vectors,
                "flops": 14 * rows * n}
    return {"bytes": w * rows * n * (4 + 2 * (case["pre"] != "none")) + 2 * weights + acc * rows * vectors,
            "flops": 30 * rows * n}


# ---------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    kind, raw = case["kind"], {k: v.double() for k, v in _tensors(case, seed).items()}
    if kind == "clip":
        scale = 1.0 / case["loss_scale"]
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g) for g in raw.values()])) * scale
        most = _max_norm(case)
        factor = scale * (most / norm.item() if norm.item() > most else 1.0)
        out = {"norm": norm}
        for buffer in _totals(case):
            out[buffer] = torch.cat([g.flatten() * factor for g, (b, _, _) in zip(raw.values(), _slices(case))
                                     if b == buffer])
        return out
    if kind in ("dense", "dense_adjoint"):
        w = raw["w"] if case["weights"] == "kn" else raw["w"].T
        normal_cdf = lambda v: torch.special.ndtr(v)
        if kind == "dense":
            z = raw["x"] @ w + raw.get("bias", 0.0)
            y = {"none": lambda: z, "relu": lambda: z.clamp_min(0), "gelu": lambda: z * normal_cdf(z),
                 "silu": lambda: z * torch.sigmoid(z)}[case["act"]]() + raw.get("residual", 0.0)
            return {"y": y, "z": z} if case["z"] else {"y": y}
        slope = 1.0
        if case["act"] != "none":
            z = raw["z"]
            slope = {"relu": lambda: torch.heaviside(z, torch.zeros_like(z)),
                     "gelu": lambda: normal_cdf(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
                     "silu": lambda: torch.sigmoid(z) * (1 + z * torch.sigmoid(-z))}[case["act"]]()
        dz = raw["g"] * slope
        dw = raw["x"].T @ dz
        return {"dx": dz @ w.T, "dw": dw if case["weights"] == "kn" else dw.T, "dbias": dz.sum(0)}
    n, out = case["n"], {}
    rows = {k: v.reshape(-1, n) if k in ("x", "b", "u", "du", "dh") else v for k, v in raw.items()}
    gate = raw["gate"].reshape(-1, n).repeat_interleave(case["rows"], 0) if case["gate"] and case["groups"] > 1 else \
        raw.get("gate", torch.ones(n, device="cuda", dtype=torch.float64))
    shape = (case["groups"], case["rows"])
    if kind == "residual":
        def norm(x, place):
            if case[place] == "layer":
                var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
                out[place + "_mean"] = mean.reshape(shape)
                x = x - mean
            else:
                var = torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / n
            rstd = (var + EPS) ** -0.5
            out[place + "_rstd"] = rstd.reshape(shape)
            return x * rstd * raw[place + "_gamma"] + raw.get(place + "_beta", 0.0)
        v = rows["b"] if case["post"] == "none" else norm(rows["b"], "post")
        u = torch.addcmul(rows["x"], gate, v, value=SCALE)
        out["u"] = u.reshape(shape + (n,))
        if case["pre"] != "none":
            out["h"] = norm(u, "pre").reshape(shape + (n,))
        return out

    def hat_of(x, place):
        centre = raw[place + "_mean"].reshape(-1, 1) if case[place] == "layer" else 0.0
        return (x - centre) * raw[place + "_rstd"].reshape(-1, 1)

    def through(cot, hat, place):
        """A norm's rows' cotangent: cot with its parts along the unit row and, for "layer", along ones taken out."""
        left = cot - hat * ((cot * hat).sum(1, keepdim=True) / n)
        if case[place] == "layer":
            left = left - cot.sum(1, keepdim=True) / n
        return left * raw[place + "_rstd"].reshape(-1, 1)

    total = rows["du"]
    if case["pre"] != "none":
        hat = hat_of(rows["u"], "pre")
        out["pre_dgamma"] = (rows["dh"] * hat).sum(0)
        if case["pre"] == "layer":
            out["pre_dbeta"] = rows["dh"].sum(0)
        total = total + through(rows["dh"] * raw["pre_gamma"], hat, "pre")
    out["dx"] = total.reshape(shape + (n,))
    hat = rows["b"] if case["post"] == "none" else hat_of(rows["b"], "post")
    v = hat if case["post"] == "none" else torch.addcmul(raw.get("post_beta", torch.zeros_like(gate[..., :n])), hat,
                                                         raw["post_gamma"])
    if case["gate"]:
        dgate = (SCALE * total * v).reshape(shape + (n,)).sum(1)
        out["dgate"] = dgate if case["groups"] > 1 else dgate[0]
    dv = SCALE * gate * total
    if case["post"] == "none":
        out["db"] = dv.reshape(shape + (n,))
    else:
        out["post_dgamma"] = (dv * hat).sum(0)
        if case["post"] == "layer":
            out["post_dbeta"] = dv.sum(0)
        out["db"] = through(dv * raw["post_gamma"], hat, "post").reshape(shape + (n,))
    return out
