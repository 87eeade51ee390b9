"""The block operators under measurement: the matrix product with bias, activation and residual in its epilogue
(``yolo_amd.layers.linear``) and the norms after and before a block with gate and residual scale
(``yolo_amd.layers.block_norm``), forward and with their gradients.

``run`` computes them in plain torch operations in 32 bits (``own`` false) or calls the framework's kernels (``own``
true); ``exact`` gives the same outputs from the definitions in 64 bits."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # one token through a small square layer of the network's own widest channel count: launch latency
        dict(name="linear_token", op="linear", m=1, k=1024, n=1024, type="bf16", act="none", residual=False, out="bf16"),
        # sixteen sequences, one token each, into a wide output layer whose scores are wanted in 32 bits: reads the weights
        dict(name="linear_scores", op="linear", m=16, k=4096, n=16384, type="bf16", act="none", residual=False, out="fp32"),
        # a few hundred tokens, every size odd and no row aligned: the general path
        dict(name="linear_ragged", op="linear", m=333, k=1021, n=755, type="fp16", act="leaky", residual=True, out="fp16"),
        # a 1x1 layer of the detection network at batch 32 on its 52 x 52 map, with a shortcut: thin, bound by memory
        dict(name="linear_pixels", op="linear", m=32 * 52 * 52, k=256, n=128, type="bf16", act="leaky", residual=True, out="bf16"),
        # a long prompt through the widening layer of a feed-forward block: bound by the matrix units
        dict(name="linear_prompt", op="linear", m=8192, k=4096, n=16384, type="bf16", act="gelu_tanh", residual=False, out="bf16"),
        # a training step's widening layer: output and every gradient
        dict(name="linear_train", op="linear_train", m=4096, k=1024, n=4096, type="bf16", act="gelu", residual=False, out="bf16"),
        # a training step on an uneven batch, with the residual's gradient
        dict(name="linear_train_ragged", op="linear_train", m=1531, k=520, n=1030, type="fp16", act="silu", residual=True, out="fp16"),
        # one token between two blocks: launch latency
        dict(name="norm_token", op="norm", batch=1, tokens=1, d=4096, type="bf16", stream="bf16", norm="rms", after=True, gate="none"),
        # a long prompt between two blocks, stream kept in 32 bits, one gate for each sequence: bound by memory
        dict(name="norm_prompt", op="norm", batch=8, tokens=2048, d=4096, type="bf16", stream="fp32", norm="rms", after=True, gate="sequence"),
        # rows of odd length: no row after the first is aligned
        dict(name="norm_ragged", op="norm", batch=3, tokens=413, d=1021, type="fp16", stream="fp16", norm="layer", after=False, gate="channel"),
        # a training step between two blocks: outputs and every gradient
        dict(name="norm_train", op="norm_train", batch=8, tokens=1024, d=2048, type="bf16", stream="bf16", norm="rms", after=True, gate="channel"),
        # a training step in 32 bits on an uneven batch, gates from the condition of each sequence
        dict(name="norm_train_ragged", op="norm_train", batch=7, tokens=601, d=769, type="fp32", stream="fp32", norm="layer", after=True, gate="sequence"),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A width: mostly whole multiples of 8 or 64, one in four any number."""
    v = _spread(rng, low, high)
    step = rng.choice((1, 8, 64, 64))
    return max(low, v // step * step)


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear_train", "norm", "norm", "norm_train"))
    if kind.startswith("linear"):
        train = kind == "linear_train"
        while True:
            m, k, n = _spread(rng, 1, 16384), _width(rng, 64, 8192), _width(rng, 64, 16384)
            if m * k * n <= (2 ** 36 if train else 2 ** 39):
                break
        kind_of = rng.choice(("bf16", "fp16"))
        # the slope of leaky jumps at zero, where two roundings of one sum may differ: its gradients are not drawn
        acts = ("none", "gelu", "gelu_tanh", "silu") + (() if train else ("leaky", "relu"))
        out = kind_of if train else rng.choice((kind_of, kind_of, "fp32"))
        return dict(op=kind, m=m, k=k, n=n, type=kind_of, act=rng.choice(acts), residual=rng.random() < 0.5, out=out)
    batch, d = rng.randint(1, 16), _width(rng, 64, 8192)
    tokens = _spread(rng, 1, max(1, (2 ** 24 if kind == "norm_train" else 2 ** 26) // (batch * d)))
    kind_of = rng.choice(("bf16", "fp16", "fp32"))
    return dict(op=kind, batch=batch, tokens=tokens, d=d, type=kind_of, stream=rng.choice((kind_of, "fp32")),
                norm=rng.choice(("rms", "layer")), after=rng.random() < 0.7,
                gate=rng.choice(("none", "channel", "sequence", "token")))


def _is_train(case):
    return case["op"].endswith("train")


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    e = size[case["type"]]
    if case["op"].startswith("linear"):
        m, k, n = case["m"], case["k"], case["n"]
        o, res = size[case["out"]], case["residual"]
        moved = e * (m * k + n * k + n) + o * m * n * (2 if res else 1)
        if not _is_train(case):
            return {"bytes": moved, "flops": 2 * m * n * k}
        moved += o * m * n * (2 if res else 1) + e * (m * k + n * k + n)
        return {"bytes": moved, "flops": 6 * m * n * k}
    rows, d = case["batch"] * case["tokens"], case["d"]
    s = size[case["stream"]]
    gate = {"none": 0, "channel": d, "sequence": case["batch"] * d, "token": rows * d}[case["gate"]] * e
    weights = 4 * d * (1 + case["after"]) * (2 if case["norm"] == "layer" else 1)
    moved = rows * d * 2 * (e + s) + gate + weights
    if not _is_train(case):
        return {"bytes": moved, "flops": 12 * rows * d}
    return {"bytes": moved + rows * d * 2 * (e + s) + gate + weights, "flops": 40 * rows * d}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale

    t, train = TYPES[case["type"]], _is_train(case)
    s = {"case": case}
    if case["op"].startswith("linear"):
        m, k, n = case["m"], case["k"], case["n"]
        # activations whose channels differ in size, weights that keep the variance
        s["x"] = (normal(m, k) * torch.exp(normal(k, scale=0.5))).to(t)
        s["weight"] = normal(n, k, scale=k ** -0.5).to(t)
        s["bias"] = normal(n, scale=0.3).to(t)
        s["residual"] = normal(m, n).to(TYPES[case["out"]]) if case["residual"] else None
        leaves = ("x", "weight", "bias", "residual")
        if train:
            s["dy"] = normal(m, n).to(TYPES[case["out"]])
    else:
        b, n, d = case["batch"], case["tokens"], case["d"]
        r = TYPES[case["stream"]]
        layer = case["norm"] == "layer"
        scale = torch.exp(normal(d, scale=0.5))
        s["x"] = (normal(b, n, d) * scale + 0.2).to(t)
        s["residual"] = (normal(b, n, d) * 3 * scale).to(r)
        shape = {"none": None, "channel": (d,), "sequence": (b, 1, d), "token": (b, n, d)}[case["gate"]]
        s["gate"] = None if shape is None else normal(*shape, scale=0.5).to(t)
        s["after_weight"] = 1 + normal(d, scale=0.2) if case["after"] else None
        s["after_bias"] = normal(d, scale=0.2) if case["after"] and layer else None
        s["before_weight"] = 1 + normal(d, scale=0.2)
        s["before_bias"] = normal(d, scale=0.2) if layer else None
        leaves = ("x", "residual", "gate", "after_weight", "after_bias", "before_weight", "before_bias")
        if train:
            s["dstream"] = normal(b, n, d).to(r)
            s["dnormed"] = normal(b, n, d).to(t)
    if train:
        s["leaves"] = [s[name].requires_grad_() for name in leaves if s[name] is not None]
    return s


# ------------------------------------------------------------------ the plain forms, in 32 bits
def _act(p, kind):
    if kind == "leaky":
        return torch.where(p > 0, p, 0.1 * p)
    if kind == "relu":
        return torch.where(p > 0, p, torch.zeros_like(p))
    if kind == "gelu":
        return 0.5 * p * (1 + torch.erf(p * 0.5 ** 0.5))
    if kind == "gelu_tanh":
        return 0.5 * p * (1 + torch.tanh((2 / math.pi) ** 0.5 * (p + 0.044715 * p * p * p)))
    if kind == "silu":
        return p / (1 + torch.exp(-p))
    return p


def _slope(p, kind):
    if kind == "leaky":
        return torch.where(p > 0, 1.0, 0.1)
    if kind == "relu":
        return torch.where(p > 0, 1.0, 0.0)
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(p * 0.5 ** 0.5)) + p * torch.exp(-0.5 * p * p) * (2 * math.pi) ** -0.5
    if kind == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        h = torch.tanh(c * (p + 0.044715 * p * p * p))
        return 0.5 * (1 + h) + 0.5 * p * (1 - h * h) * c * (1 + 3 * 0.044715 * p * p)
    if kind == "silu":
        z = 1 / (1 + torch.exp(-p))
        return z * (1 + p * (1 - z))
    return torch.ones_like(p)


def _linear_plain(s):
    case = s["case"]
    p = s["x"].float() @ s["weight"].float().t() + s["bias"].float()
    y = _act(p, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    y = y.to(TYPES[case["out"]])
    if not _is_train(case):
        return y
    dp = s["dy"].float() * _slope(p, case["act"])
    outs = [y, (dp @ s["weight"].float()).to(s["x"].dtype), (dp.t() @ s["x"].float()).to(s["weight"].dtype),
            dp.sum(0).to(s["bias"].dtype)]
    return outs + ([s["dy"]] if s["residual"] is not None else [])


def _unit(v, norm):
    """(v normalised without its weights, the factor)."""
    if norm == "layer":
        v = v - v.mean(-1, keepdim=True)
    f = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return v * f, f


def _unit_back(d, unit, f, norm):
    d = d - unit * (d * unit).mean(-1, keepdim=True) - (d.mean(-1, keepdim=True) if norm == "layer" else 0)
    return d * f


def _norm_plain(s):
    case, scale = s["case"], 0.5
    norm = case["norm"]
    u, r = s["x"].float(), s["residual"].float()
    p = u
    if case["after"]:
        u_unit, u_f = _unit(u, norm)
        p = u_unit * s["after_weight"]
        if s["after_bias"] is not None:
            p = p + s["after_bias"]
    gate = s["gate"].float() if s["gate"] is not None else None
    h = r + scale * (p * gate if gate is not None else p)
    h_unit, h_f = _unit(h, norm)
    y = h_unit * s["before_weight"]
    if s["before_bias"] is not None:
        y = y + s["before_bias"]
    outs = [h.to(s["residual"].dtype), y.to(s["x"].dtype)]
    if not _is_train(case):
        return outs
    dy = s["dnormed"].float()
    dh = s["dstream"].float() + _unit_back(dy * s["before_weight"], h_unit, h_f, norm)
    dp = scale * (dh * gate if gate is not None else dh)
    du = _unit_back(dp * s["after_weight"], u_unit, u_f, norm) if case["after"] else dp
    outs += [du.to(s["x"].dtype), dh.to(s["residual"].dtype)]
    if gate is not None:
        dg = scale * dh * p
        dg = dg.sum((0, 1)) if case["gate"] == "channel" else dg.sum(1, keepdim=True) if case["gate"] == "sequence" else dg
        outs.append(dg.to(s["gate"].dtype))
    if case["after"]:
        outs.append((dp * u_unit).sum((0, 1)))
    if s["after_bias"] is not None:
        outs.append(dp.sum((0, 1)))
    outs.append((dy * h_unit).sum((0, 1)))
    if s["before_bias"] is not None:
        outs.append(dy.sum((0, 1)))
    return outs


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return _linear_plain(state) if case["op"].startswith("linear") else _norm_plain(state)
    from yolo_amd import layers
    if case["op"].startswith("linear"):
        y = layers.linear(state["x"], state["weight"], state["bias"], activation=None if case["act"] == "none" else case["act"],
                          residual=state["residual"], out_dtype=TYPES[case["out"]])
        if not _is_train(case):
            return y
        return [y.detach(), *torch.autograd.grad(y, state["leaves"], state["dy"])]
    h, y = layers.block_norm(state["x"], state["residual"], norm=case["norm"], after=case["after"],
                             after_weight=state["after_weight"], after_bias=state["after_bias"], gate=state["gate"],
                             residual_scale=0.5, before_weight=state["before_weight"],
                             before_bias=state["before_bias"], eps=EPS)
    if not _is_train(case):
        return [h, y]
    return [h.detach(), y.detach(),
            *torch.autograd.grad((h, y), state["leaves"], (state["dstream"], state["dnormed"]))]


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    v = {k: t.detach().double().requires_grad_(_is_train(case)) if torch.is_tensor(t) else t for k, t in s.items()}
    if case["op"].startswith("linear"):
        acts = {"none": lambda z: z, "leaky": lambda z: torch.nn.functional.leaky_relu(z, 0.1), "relu": torch.relu,
                "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu,
                "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}
        y = acts[case["act"]](torch.matmul(v["x"], v["weight"].transpose(0, 1)) + v["bias"])
        if v["residual"] is not None:
            y = y + v["residual"]
        if not _is_train(case):
            return y
        names = ("x", "weight", "bias", "residual")
        return [y.detach(), *torch.autograd.grad(y, [v[n] for n in names if v[n] is not None], v["dy"].detach())]

    def normed(t, w, b):
        if case["norm"] == "layer":
            return torch.nn.functional.layer_norm(t, t.shape[-1:], w, b, EPS)
        return t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + EPS) * w

    branch = normed(v["x"], v["after_weight"], v["after_bias"]) if case["after"] else v["x"]
    if v["gate"] is not None:
        branch = branch * v["gate"]
    h = v["residual"] + 0.5 * branch
    y = normed(h, v["before_weight"], v["before_bias"])
    if not _is_train(case):
        return [h, y]
    names = ("x", "residual", "gate", "after_weight", "after_bias", "before_weight", "before_bias")
    grads = torch.autograd.grad((h, y), [v[n] for n in names if v[n] is not None],
                                (v["dstream"].detach(), v["dnormed"].detach()))
    return [h.detach(), y.detach(), *grads]
