"""Plain 64-bit statements of the 8-bit linear layer and of the Newton-Schulz iteration, on the CPU."""
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # half a step, relative
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
COEF = (3.4445, -4.7750, 2.0315)


def quantize_rows(x):
    """(q int8, scale fp32) of the rows of x: a quotient of two fp32 numbers that is not half-way between two integers is
    further than 2^-33 from it, so its rounding to fp64 cannot cross; a half-way one is exact in fp64."""
    x = x.float().cpu()
    top = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    s = torch.where(bad, torch.full_like(top, float("nan")), torch.clamp_min(top, 2.0 ** -100) * torch.tensor(1 / 127, dtype=torch.float32))
    q = torch.where(bad, torch.zeros((), dtype=torch.float64), torch.round(x.double() / s.double()))
    return q.to(torch.int8), s[..., 0]


def matmul(qa, sa, qb, sb, bias=None):
    """(value, sum of the magnitudes that are added) in 64 bits."""
    y = (qa.double() @ qb.double().t()) * sa.double()[:, None] * sb.double()
    size = y.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def gradients(g, qx, sx, qw, sw):
    """(gx, its term sum), (gw, its term sum), (gb, its term sum) of the straight-through backward in 64 bits."""
    g, x, w = g.double(), qx.double() * sx.double()[:, None], qw.double() * sw.double()[:, None]
    return (g @ w, g.abs() @ w.abs()), (g.t() @ x, g.abs().t() @ x.abs()), (g.sum(0), g.abs().sum(0))


def _fp16(v, scale):
    return (v * scale).half().double() / scale


def _fp16_two(v, scale):
    v = v * scale
    h = v.half().double()
    return (h + (v - h).half().double()) / scale


def _bits22(v, scale):
    """Two values of 11 bits, without a smallest exponent."""
    def eleven(u):
        m, e = torch.frexp(u)
        return torch.ldexp(torch.round(m * 2048) / 2048, e)
    h = eleven(v)
    return h + eleven(v - h)


def iterate(x, steps=5, coef=COEF, eps=1e-7, form="exact", device="cpu"):
    """The iterate of one matrix in 64 bits.  form "fp16" / "two": X, A and B rounded as the kernels' factors are (to one
    fp16 value or to two, scaled by S and by 4096), "22 bits": to two values of 11 bits each, "fp32": to fp32; everything else exact.  The distance of such a result
    from the exact one is what those roundings do to this matrix."""
    x = x.double().to(device)
    flip = x.shape[0] > x.shape[1]
    if flip:
        x = x.t()
    r, c = x.shape
    log_s = 0
    while log_s < 14 and 1 << (2 * log_s + 2) <= r * c:
        log_s += 1
    S = float(1 << log_s)
    rnd = {"exact": lambda v, s: v, "fp16": _fp16, "two": _fp16_two, "22 bits": _bits22, "fp32": lambda v, s: v.float().double()}[form]
    triples = coef if isinstance(coef[0], (tuple, list)) else [coef] * steps
    x = rnd(x / max(float(x.norm()), eps), S)
    for k, (a, b, c5) in enumerate(triples):
        A = rnd(x @ x.t(), 4096.0)
        B = rnd(b * A + c5 * (A @ A), 4096.0)
        x = a * x + B @ x
        if k + 1 < len(triples):
            x = rnd(x, S)
    return x.t() if flip else x
