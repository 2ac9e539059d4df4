"""The 8-bit linear layer (serving and training) and the orthogonalised weight update, as measured cases.

Every case names one of four passes:

``serve``  y = (q(x) s_x) (q_w s_w)^T + b for tokens x and a weight matrix held in 8 bits: one scale a token, one a channel.
``train``  the same product with the weight in floating point, quantised on the way, and its straight-through gradients.
``orth``   the quintic Newton-Schulz iteration that takes a matrix's singular values towards one.
``muon``   one optimiser step: momentum, the iteration above, and the update of the weights.

`run` computes them with elementary torch operations where ``own`` is false and through ``dpd_amd`` where it is true.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
FLOOR = 2.0 ** -100          # rows below this magnitude share its scale: a row of zeros has a finite one
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01


def listed():
    return [
        # one token of a decoding loop, square projection: latency and the read of the weights
        {"name": "serve 1 token", "op": "serve", "tokens": 1, "ins": 4096, "outs": 4096, "type": "bf16", "bias": False},
        # a few streams decoded together, sizes that divide nothing
        {"name": "serve 17 tokens, odd", "op": "serve", "tokens": 17, "ins": 1030, "outs": 515, "type": "fp32", "bias": True},
        # a decoding batch against a wide layer
        {"name": "serve 128 tokens", "op": "serve", "tokens": 128, "ins": 4096, "outs": 16384, "type": "fp16", "bias": False},
        # a long prompt: bound by the matrix cores
        {"name": "serve 8192 tokens", "op": "serve", "tokens": 8192, "ins": 8192, "outs": 8192, "type": "bf16", "bias": True},
        # a training step of one layer
        {"name": "train 4096 tokens", "op": "train", "tokens": 4096, "ins": 4096, "outs": 4096, "type": "bf16", "bias": True},
        # the same in single precision with ragged sizes
        {"name": "train 1000 tokens, odd", "op": "train", "tokens": 1000, "ins": 515, "outs": 333, "type": "fp32", "bias": True},
        # the generator's first layer: one matrix that fits into a compute unit
        {"name": "orth 32x30", "op": "orth", "batch": 1, "rows": 32, "cols": 30, "type": "fp32"},
        # three single-precision matrices of one shape, odd sizes, more rows than columns
        {"name": "orth 3 of 1000x777", "op": "orth", "batch": 3, "rows": 1000, "cols": 777, "type": "fp32"},
        # a wide layer's update in the type that it is trained in
        {"name": "orth 1024x4096", "op": "orth", "batch": 1, "rows": 1024, "cols": 4096, "type": "bf16"},
        # the largest square layer
        {"name": "orth 4096x4096", "op": "orth", "batch": 1, "rows": 4096, "cols": 4096, "type": "bf16"},
        # every weight matrix of the 30-32-16-2 generator and of the 4-64-32-16-1 critic
        {"name": "muon generator, critic", "op": "muon", "shapes": "32x30,16x32,2x16,64x4,32x64,16x32,1x16", "type": "fp32"},
        # the matrices of one wide block
        {"name": "muon block", "op": "muon", "shapes": "2048x2048,2048x2048,4096x2048,2048x4096", "type": "bf16"},
    ]


def _log_size(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    op = rng.choice(("serve", "serve", "train", "orth", "muon"))
    kind = rng.choice(("bf16", "fp16", "fp32"))
    if op == "serve":
        while True:
            t, i, o = _log_size(rng, 1, 8192), _log_size(rng, 16, 8192), _log_size(rng, 16, 16384)
            if t * i * o <= 8192 ** 3:
                return {"op": op, "tokens": t, "ins": i, "outs": o, "type": kind, "bias": rng.random() < 0.5}
    if op == "train":
        return {"op": op, "tokens": _log_size(rng, 1, 8192), "ins": _log_size(rng, 16, 4096), "outs": _log_size(rng, 16, 4096), "type": kind,
                "bias": rng.random() < 0.5}
    if op == "orth":
        while True:
            b, r, c = _log_size(rng, 1, 8), _log_size(rng, 8, 4096), _log_size(rng, 8, 4096)
            if b * r * c * min(r, c) <= (2048 ** 3 if kind == "fp32" else 4096 ** 3):
                return {"op": op, "batch": b, "rows": r, "cols": c, "type": kind}
    shapes = ["%dx%d" % (_log_size(rng, 8, 2048), _log_size(rng, 8, 2048)) for _ in range(rng.randint(1, 4))]
    return {"op": op, "shapes": ",".join(shapes), "type": rng.choice(("bf16", "fp32"))}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


# ---------------------------------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def _tokens(g, n, k):
    """Activations: channels of different spread, tokens of different size."""
    return _normal(g, n, k) * torch.exp(0.5 * _normal(g, 1, k)) * torch.exp(0.3 * _normal(g, n, 1))


def _weight(g, n, k):
    return _normal(g, n, k) * torch.exp(0.2 * _normal(g, n, 1)) / math.sqrt(k)


def _update(g, b, r, c):
    """A gradient as a batch leaves it: rows and columns of different size."""
    return 1e-3 * _normal(g, b, r, c) * torch.exp(0.5 * _normal(g, b, r, 1)) * torch.exp(0.5 * _normal(g, b, 1, c))


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]
    if case["op"] in ("serve", "train"):
        n, k, m = case["tokens"], case["ins"], case["outs"]
        d = {"x": _tokens(g, n, k).to(kind), "w": _weight(g, m, k).to(kind), "b": (0.1 * _normal(g, m)).to(kind) if case["bias"] else None}
        if case["op"] == "train":
            d["g"] = (1e-3 * _normal(g, n, m) * torch.exp(0.5 * _normal(g, n, 1))).to(kind)
        return d
    if case["op"] == "orth":
        return {"x": _update(g, case["batch"], case["rows"], case["cols"]).to(kind)}
    d = {"p": [], "g": [], "m": []}
    for r, c in _shapes(case):
        d["p"].append(_weight(g, r, c).to(kind))
        d["g"].append(_update(g, 1, r, c)[0].to(kind))
        d["m"].append(5 * _update(g, 1, r, c)[0])
    return d


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if case["op"] == "serve":       # the weights are quantised once, ahead of the tokens
        s["wq"], s["ws"] = _quantise(s.pop("w"))
        s["wq"] = s["wq"].to(torch.int8)
        if own:
            from dpd_amd.utils import Int8Inference
            s["engine"] = Int8Inference({"weight": s["wq"], "scale": s["ws"], "bias": s["b"]})
    elif case["op"] == "train" and own:
        for name in ("x", "w", "b"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    elif case["op"] == "muon" and own:
        from dpd_amd.training import Muon
        s["p"] = [torch.nn.Parameter(p) for p in s["p"]]
        for p, grad in zip(s["p"], s["g"]):
            p.grad = grad
        s["opt"] = Muon(s["p"], lr=LR, momentum=MOMENTUM, nesterov=True, weight_decay=DECAY, steps=STEPS, coefficients=COEFFICIENTS)
        for p, m in zip(s["p"], s["m"]):
            s["opt"].state[p]["momentum_buffer"] = m
    return s


# ---------------------------------------------------------------------------------------- one pass
def _quantise(x):
    """Integers of at most 127, rounded half to even from the exact quotient, and the scale of each row in 32 bits."""
    scale = torch.clamp_min(x.float().abs().amax(-1, keepdim=True), FLOOR) / 127
    return torch.round(x.double() / scale.double()).float(), scale[..., 0]


def _linear(xq, xs, wq, ws, b):
    y = (xq @ wq.t()) * xs[:, None] * ws
    return y if b is None else y + b.float()


def _orthogonal(x):
    wide = x.shape[-2] <= x.shape[-1]
    x = x if wide else x.transpose(-2, -1)
    size = torch.clamp_min(x.double().square().sum((-2, -1), keepdim=True).sqrt(), 1e-7)
    x = (x.double() / size).float().contiguous()
    c1, c3, c5 = COEFFICIENTS
    for _ in range(STEPS):
        a = x @ x.transpose(-2, -1).contiguous()
        x = c1 * x + (c3 * a + c5 * (a @ a)) @ x
    return x if wide else x.transpose(-2, -1)


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "serve":
            return s["engine"](s["x"])
        if op == "train":
            from dpd_amd.utils import int8_linear
            y = int8_linear(s["x"], s["w"], s["b"])
            leaves = [t for t in (s["x"], s["w"], s["b"]) if t is not None]
            return [y, *torch.autograd.grad(y, leaves, s["g"])]
        if op == "orth":
            from dpd_amd.utils import orthogonalize
            return orthogonalize(s["x"], steps=STEPS, coefficients=COEFFICIENTS)
        s["opt"].step()
        return [*s["p"], *s["m"]]
    kind = TYPES[s["case"]["type"]]
    if op == "serve":
        xq, xs = _quantise(s["x"])
        return _linear(xq, xs, s["wq"].float(), s["ws"], s["b"]).to(kind)
    if op == "train":
        xq, xs = _quantise(s["x"])
        wq, ws = _quantise(s["w"])
        g = s["g"].float()
        out = [_linear(xq, xs, wq, ws, s["b"]), (g * ws) @ wq, (g * xs[:, None]).t() @ xq]
        if s["b"] is not None:
            out.append(g.sum(0))
        return [t.to(kind) for t in out]
    if op == "orth":
        return _orthogonal(s["x"]).to(kind)
    for p, g, m in zip(s["p"], s["g"], s["m"]):
        m.mul_(MOMENTUM).add_(g.float())
        o = _orthogonal(g.float() + MOMENTUM * m)
        factor = LR * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        p.copy_((p.float() * (1 - LR * DECAY) - factor * o).to(kind))
    return [*s["p"], *s["m"]]


# ---------------------------------------------------------------------------------------- what a pass needs, and its value
def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] in ("serve", "train"):
        n, k, m = case["tokens"], case["ins"], case["outs"]
        bias = m * size if case["bias"] else 0
        if case["op"] == "serve":
            return {"bytes": n * k * size + m * k + 4 * m + bias + n * m * size, "flops": 2 * n * k * m}
        return {"bytes": 2 * size * (n * k + m * k + n * m) + 2 * bias, "flops": 6 * n * k * m}

    def iteration(r, c):            # two symmetric products and one full one
        r, c = min(r, c), max(r, c)
        return STEPS * (3 * r * r * c + r ** 3)
    if case["op"] == "orth":
        r, c = case["rows"], case["cols"]
        return {"bytes": 2 * size * case["batch"] * r * c, "flops": case["batch"] * iteration(r, c)}
    return {"bytes": sum(r * c * (3 * size + 8) for r, c in _shapes(case)), "flops": sum(iteration(r, c) for r, c in _shapes(case))}


def _grid64(x):
    """The values that 8 bits and a 32-bit scale leave of x, in 64 bits."""
    x = x.double()
    top = x.abs().max(dim=-1, keepdim=True).values
    step = (torch.maximum(top, torch.full_like(top, FLOOR)).float() / 127.0).double()
    return torch.round(x / step) * step


def _iterate64(x):
    x = x.double()
    flip = x.shape[0] > x.shape[1]
    if flip:
        x = x.t().contiguous()
    x = x / max(float(torch.linalg.vector_norm(x)), 1e-7)
    eye = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        k = torch.mm(x, x.t().contiguous())
        x = torch.mm(a * eye + torch.mm(k, b * eye + c * k), x)
    return x.t() if flip else x


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] in ("serve", "train"):
        x, w = _grid64(d["x"]), _grid64(d["w"])
        y = torch.mm(x, w.t().contiguous())
        if d["b"] is not None:
            y = y + d["b"].double()
        if case["op"] == "serve":
            return y
        g = d["g"].double()
        return [y, torch.mm(g, w), torch.mm(g.t().contiguous(), x)] + ([torch.mv(g.t().contiguous(), torch.ones_like(g[:, 0]))] if d["b"] is not None else [])
    if case["op"] == "orth":
        return torch.stack([_iterate64(x) for x in d["x"]])
    params, buffers = [], []
    for p, g, m in zip(d["p"], d["g"], d["m"]):
        m = MOMENTUM * m.double() + g.double()
        o = _iterate64(MOMENTUM * m + g.double())
        params.append((1.0 - LR * DECAY) * p.double() - LR * math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * o)
        buffers.append(m)
    return params + buffers
