"""Cases of the dense-network operators: linear layers (bias, activation and residual in the product's epilogue) and their
backward pass, layer norm and its backward pass, and the clipping of gradients by their global norm.

With ``own`` false ``run`` computes the plain form with elementary torch operations in 32 bits (64 where a long sum asks for
it); with ``own`` true it calls neus2_b200.ops."""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"f16": 2, "bf16": 2, "f32": 4}
ACTIVATIONS = ("none", "relu", "gelu", "silu")
EPS = 1e-5
MAX_FLOPS, MAX_BYTES = 2.7e11, 2.6e8  # of the largest listed cases; drawn ones stay below


def listed():
    return [
        # one sample through a wide layer, as when a trained network answers a single query: the weights' way from memory
        dict(name="linear_one_row", op="linear", n=1, in_width=4096, out_width=4096, type="bf16", activation="silu", bias=True, residual=False,
             preact=False, pad=0),
        # the batch and the widths of the framework's own networks (encoding and spherical harmonics into 64 neurons)
        dict(name="linear_network_width", op="linear", n=262144, in_width=48, out_width=64, type="f16", activation="relu", bias=False,
             residual=False, preact=False, pad=0),
        # widths that fit no tile and no 16-byte row, rows cut out of a wider matrix
        dict(name="linear_odd", op="linear", n=2000, in_width=1001, out_width=777, type="f16", activation="gelu", bias=True, residual=True,
             preact=True, pad=3),
        # the second half of a residual block, training batch: the largest product
        dict(name="linear_wide", op="linear", n=8192, in_width=4096, out_width=4096, type="bf16", activation="gelu", bias=True, residual=True,
             preact=False, pad=0),
        # backward pass of a hidden layer of a residual block, with the layer below's activation and its skip connection
        dict(name="linear_backward_wide", op="linear_backward", n=8192, in_width=4096, out_width=1024, type="bf16", activation="gelu", skip=False,
             bias=True, pad=0),
        # backward pass at the framework's own width and batch
        dict(name="linear_backward_network_width", op="linear_backward", n=262144, in_width=64, out_width=64, type="f16", activation="relu",
             skip=True, bias=True, pad=0),
        # rows of a wide network, 16 bits with 32-bit weights
        dict(name="layer_norm_wide", op="layer_norm", n=16384, width=4096, type="bf16", weights="f32", beta=True, pad=0),
        # 64 neurons, the framework's batch
        dict(name="layer_norm_network_width", op="layer_norm", n=262144, width=64, type="f16", weights="f16", beta=True, pad=0),
        # backward pass in a residual block: the gradient of the skip connection joins
        dict(name="layer_norm_backward_block", op="layer_norm_backward", n=8192, width=1024, type="bf16", weights="bf16", skip=True, pad=0),
        # odd width, few rows: the shortest call
        dict(name="layer_norm_backward_odd", op="layer_norm_backward", n=33, width=1111, type="f32", weights="f32", skip=False, pad=0),
        # the gradients of the framework's own model: MLPs in 32 bits, hash grid in 16, variance
        dict(name="clip_model", op="clip", tensors=3, total=12612212, type="mixed", ratio=3.0, align=16),
        # the gradients of a deep stack of layers, many of them small, all of them within the bound
        dict(name="clip_many_tensors", op="clip", tensors=400, total=40000000, type="bf16", ratio=0.5, align=16),
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """Half of the widths are multiples of 16, as networks have them; the others are any number."""
    w = _between(rng, lo, hi)
    return max(16, w // 16 * 16) if rng.random() < 0.5 else w


def draw(rng):
    op = rng.choice(("linear", "linear", "linear_backward", "linear_backward", "layer_norm", "layer_norm_backward", "clip"))
    kind = rng.choice(("f16", "bf16"))
    while True:
        if op in ("linear", "linear_backward"):
            c = dict(op=op, n=_between(rng, 1, 262144), in_width=_width(rng, 16, 8192), out_width=_width(rng, 16, 8192), type=kind,
                     activation=rng.choice(ACTIVATIONS), bias=rng.random() < 0.7, pad=rng.choice((0, 0, 0, 8, 5)))
            if op == "linear":
                c.update(residual=rng.random() < 0.5, preact=rng.random() < 0.3)
            else:
                c.update(skip=rng.random() < 0.5)
        elif op in ("layer_norm", "layer_norm_backward"):
            kind = rng.choice(("f16", "bf16", "f32"))
            c = dict(op=op, n=_between(rng, 1, 262144), width=_width(rng, 16, 16384), type=kind, weights=rng.choice((kind, "f32")),
                     pad=rng.choice((0, 0, 0, 8, 5)))
            c.update(beta=rng.random() < 0.7) if op == "layer_norm" else c.update(skip=rng.random() < 0.5)
        else:
            c = dict(op=op, tensors=_between(rng, 1, 1500), total=_between(rng, 3000, 60000000), type=rng.choice(("mixed", "f16", "bf16", "f32")),
                     ratio=rng.choice((0.3, 3.0, 30.0)), align=rng.choice((16, 16, 1)))
        w = work(c)
        if w["bytes"] <= MAX_BYTES and w["flops"] <= MAX_FLOPS:
            return c


def _clip_tensors(case):
    """(type, size) of every tensor: the framework's own three buffers, or sizes that fall off like those of layers."""
    total, count = case["total"], case["tensors"]
    if count == 3 and case["type"] == "mixed":
        return [("f32", 12288), ("f16", total - 12288 - 4), ("f32", 4)]
    shares = [1.0 / (1 + (7 * i) % 61) ** 2 for i in range(count)]
    sizes = [max(1, int(total * s / sum(shares))) for s in shares]
    kinds = ("f32", "f16", "bf16") if case["type"] == "mixed" else (case["type"],)
    return [(kinds[i % len(kinds)], s) for i, s in enumerate(sizes)]


def work(case):
    op = case["op"]
    if op == "clip":
        return {"bytes": 2 * sum(SIZES[t] * s for t, s in _clip_tensors(case)) + 8, "flops": 3 * sum(s for _, s in _clip_tensors(case))}
    b = SIZES[case["type"]]
    n = case["n"]
    if op == "linear":
        i, o = case["in_width"], case["out_width"]
        return {"bytes": b * (n * i + o * i + o * case["bias"] + n * o * (1 + case["residual"] + case["preact"])), "flops": 2 * n * i * o}
    if op == "linear_backward":
        i, o = case["in_width"], case["out_width"]
        return {"bytes": b * (n * o + o * i + n * i * (2 + (case["activation"] != "none") + case["skip"])) + 4 * (o * i + o * case["bias"]),
                "flops": 4 * n * i * o}
    w = case["width"]
    if op == "layer_norm":
        return {"bytes": 2 * b * n * w + SIZES[case["weights"]] * w * (1 + case["beta"]) + 8 * n, "flops": 8 * n * w}
    return {"bytes": b * n * w * (3 + case["skip"]) + SIZES[case["weights"]] * w + 8 * n + 8 * w, "flops": 14 * n * w}


def _rows(gen, n, width, dtype, scale, pad, shift=0.0):
    """[n][width] values in rows of width + pad entries."""
    full = torch.empty((n, width + pad), dtype=torch.float32, device="cuda").normal_(shift, scale, generator=gen).to(dtype)
    return full[:, :width]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op = case["op"]
    s = {"case": dict(case)}
    if op == "clip":
        # gradients of very different sizes from layer to layer, as training has them, in one buffer for each type (`align`: every
        # tensor starts on a multiple of so many entries); the bound is the expected norm over `ratio` (below 1: nothing is clipped)
        sizes = _clip_tensors(case)
        scale = [10.0 ** (-1 - (5 * i) % 3) for i in range(len(sizes))]
        s["max_norm"] = math.sqrt(sum(size * a * a for (_, size), a in zip(sizes, scale))) / case["ratio"]
        s["flat"], s["out"], views = {}, {}, {}
        for kind in sorted({t for t, _ in sizes}):
            at, places = 0, []
            for i, (t, size) in enumerate(sizes):
                if t == kind:
                    places.append((i, at, size))
                    at += -(-size // case["align"]) * case["align"]
            s["flat"][kind], s["out"][kind] = (torch.zeros(at, dtype=TYPES[kind], device="cuda") for _ in range(2))
            for i, start, size in places:
                views[i] = (s["flat"][kind][start:start + size], s["out"][kind][start:start + size])
                views[i][0].copy_(torch.empty(size, dtype=torch.float32, device="cuda").normal_(0.0, scale[i], generator=gen))
        if own:
            from neus2_b200 import ops
            s["set"] = ops.GradientSet([views[i][0] for i in range(len(sizes))], out=[views[i][1] for i in range(len(sizes))])
        return s
    t, n, pad = TYPES[case["type"]], case["n"], case["pad"]
    if op in ("linear", "linear_backward"):
        i, o = case["in_width"], case["out_width"]
        bound = math.sqrt(6.0 / (i + o))
        s["x"] = _rows(gen, n, i, t, 1.0, pad)
        s["w"] = torch.empty((o, i), dtype=torch.float32, device="cuda").uniform_(-bound, bound, generator=gen).to(t)
        if op == "linear":
            s["bias"] = _rows(gen, 1, o, t, 0.1, 0)[0] if case["bias"] else None
            s["residual"] = _rows(gen, n, o, t, 1.0, pad) if case["residual"] else None
        else:
            s["dy"] = _rows(gen, n, o, t, 0.05, pad)
            s["z_below"] = _rows(gen, n, i, t, 1.0, pad) if case["activation"] != "none" else None
            s["skip"] = _rows(gen, n, i, t, 0.05, pad) if case["skip"] else None
        return s
    w, wt = case["width"], TYPES[case["weights"]]
    s["x"] = _rows(gen, n, w, t, 1.5, pad, shift=0.5)
    s["gamma"] = torch.empty(w, dtype=torch.float32, device="cuda").normal_(1.0, 0.2, generator=gen).to(wt)
    if op == "layer_norm":
        s["beta"] = torch.empty(w, dtype=torch.float32, device="cuda").normal_(0.0, 0.2, generator=gen).to(wt) if case["beta"] else None
    else:
        x = s["x"].float()
        mean = x.mean(1)
        s["mean"], s["rstd"] = mean, ((x - mean[:, None]).square().mean(1) + EPS).rsqrt()
        s["dy"] = _rows(gen, n, w, t, 0.05, pad)
        s["skip"] = _rows(gen, n, w, t, 0.05, pad) if case["skip"] else None
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
GELU_C, GELU_A = math.sqrt(2.0 / math.pi), 0.044715


def _act(kind, z):
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "gelu":
        return z / (1 + torch.exp(-2 * GELU_C * (z + GELU_A * z * z * z)))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(kind, z):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu":
        p = 1 / (1 + torch.exp(-2 * GELU_C * (z + GELU_A * z * z * z)))
        return p + z * p * (1 - p) * 2 * GELU_C * (1 + 3 * GELU_A * z * z)
    p = 1 / (1 + torch.exp(-z))
    return p + z * p * (1 - p)


def _plain_linear(s, case):
    t = TYPES[case["type"]]
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(case["activation"], z)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return (y.to(t), z.to(t)) if case["preact"] else y.to(t)


def _plain_linear_backward(s, case):
    dy, x = s["dy"].float(), s["x"].float()
    dx = dy @ s["w"].float()
    if s["z_below"] is not None:
        dx = dx * _act_slope(case["activation"], s["z_below"].float())
    if s["skip"] is not None:
        dx = dx + s["skip"].float()
    out = [dx.to(TYPES[case["type"]]), dy.t() @ x]
    return out + [dy.sum(0)] if case["bias"] else out


def _plain_layer_norm(s, case):
    x = s["x"].float()
    mean = x.mean(1)
    centred = x - mean[:, None]
    rstd = (centred.square().mean(1) + EPS).rsqrt()
    y = centred * rstd[:, None] * s["gamma"].float()
    if s["beta"] is not None:
        y = y + s["beta"].float()
    return y.to(TYPES[case["type"]]), mean, rstd


def _plain_layer_norm_backward(s, case):
    dy = s["dy"].float()
    xhat = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    a = dy * s["gamma"].float()
    dx = s["rstd"][:, None] * (a - a.mean(1, keepdim=True) - xhat * (a * xhat).mean(1, keepdim=True))
    if s["skip"] is not None:
        dx = dx + s["skip"].float()
    return dx.to(TYPES[case["type"]]), (dy * xhat).sum(0), dy.sum(0)


def _plain_clip(s, case):
    kinds = sorted(s["flat"])
    norm = torch.stack([s["flat"][k].double().square().sum() for k in kinds]).sum().sqrt()
    c = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm))
    return [torch.stack([norm, c]).float()] + [(s["flat"][k].float() * c.float()).to(TYPES[k]) for k in kinds]


# ---------------------------------------------------------------------------------------------------- the framework's
def _own(s, case):
    from neus2_b200 import _lib as L
    from neus2_b200 import ops
    op = case["op"]
    if op == "linear":
        return ops.linear_forward(s["x"], s["w"], bias=s["bias"], residual=s["residual"], activation=L.ACTIVATIONS[case["activation"]],
                                  want_preact=case["preact"])
    if op == "linear_backward":
        dx, dw, db = ops.linear_backward(s["x"], s["w"], s["dy"], below_activation=L.ACTIVATIONS[case["activation"]], below_preact=s["z_below"],
                                         skip=s["skip"], want_bias=case["bias"])
        return [dx, dw, db] if case["bias"] else [dx, dw]
    if op == "layer_norm":
        return ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], eps=EPS, want_stats=True)
    if op == "layer_norm_backward":
        return ops.layer_norm_backward(s["x"], s["gamma"], s["mean"], s["rstd"], s["dy"], skip=s["skip"])
    return [s["set"].clip(s["max_norm"])] + [s["out"][k] for k in sorted(s["out"])]


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    return {"linear": _plain_linear, "linear_backward": _plain_linear_backward, "layer_norm": _plain_layer_norm,
            "layer_norm_backward": _plain_layer_norm_backward, "clip": _plain_clip}[case["op"]](state, case)


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _logistic(v):
    return torch.sigmoid(v)


def _exact_act(kind, z):
    if kind == "relu":
        return z.clamp(min=0)
    if kind == "gelu":
        return 0.5 * z * (1 + torch.tanh(GELU_C * (z + GELU_A * z.pow(3))))
    if kind == "silu":
        return z * _logistic(z)
    return z


def _exact_slope(kind, z):
    """The derivative by the product rule of the tanh and logistic forms."""
    if kind == "relu":
        return torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
    if kind == "gelu":
        t = torch.tanh(GELU_C * (z + GELU_A * z.pow(3)))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * GELU_C * (1 + 3 * GELU_A * z * z)
    return _logistic(z) * (1 + z * (1 - _logistic(z)))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    up = lambda name: None if s.get(name) is None else s[name].double()  # noqa: E731
    if op == "clip":
        flat = {k: v.double() for k, v in s["flat"].items()}
        norm = math.sqrt(sum(float((v * v).sum()) for v in flat.values()))
        c = min(1.0, s["max_norm"] / norm)
        return [torch.tensor([norm, c], dtype=torch.float64, device="cuda")] + [flat[k] * c for k in sorted(flat)]
    x = up("x")
    if op == "linear":
        z = torch.matmul(x, up("w").T) + (0 if s["bias"] is None else up("bias"))
        y = _exact_act(case["activation"], z) + (0 if s["residual"] is None else up("residual"))
        return (y, z) if case["preact"] else y
    if op == "linear_backward":
        dy = up("dy")
        dx = torch.matmul(dy, up("w"))
        dx = dx if s["z_below"] is None else dx * _exact_slope(case["activation"], up("z_below"))
        dx = dx if s["skip"] is None else dx + up("skip")
        return [dx, torch.matmul(dy.T, x)] + ([torch.matmul(dy.T, torch.ones(len(dy), dtype=torch.float64, device="cuda"))] if case["bias"] else [])
    gamma, width = up("gamma"), case["width"]
    if op == "layer_norm":
        mean = x.sum(1) / width
        var = ((x - mean[:, None]) ** 2).sum(1) / width
        y = (x - mean[:, None]) / torch.sqrt(var + EPS)[:, None] * gamma + (0 if s["beta"] is None else up("beta"))
        return y, mean, 1 / torch.sqrt(var + EPS)
    # the backward pass is a function of the statistics that it is handed
    mean, rstd, dy = up("mean")[:, None], up("rstd")[:, None], up("dy")
    xhat, a = (x - mean) * rstd, dy * gamma
    dx = rstd * (a - a.sum(1, keepdim=True) / width - xhat * ((a * xhat).sum(1, keepdim=True) / width))
    return dx + (0 if s["skip"] is None else up("skip")), (dy * xhat).sum(0), dy.sum(0)
