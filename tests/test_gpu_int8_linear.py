"""The 8-bit linear layer against its 64-bit statement (operator_oracle.py).

Tolerances, before any run: the quantiser is exact (integers and scales equal).  A product's sum is exact; its conversion to
fp32, the two scales and the bias are one rounding of 2^-24 each of numbers no larger than |sum| sa sb + |bias|, the result is
rounded once to its type (U = half a step).  A gradient adds n fp32 products: every one of the n additions and the roundings
of the terms (V: bf16 gradients 2^-8, fp16 2^-16, fp32 2^-24, plus 2^-24 for g times a scale) act on at most the sum of
the magnitudes, so |error| <= (V + (n + 1) 2^-23) sum|terms| + U |value|."""
import pytest
import torch

import dpd_amd  # noqa: F401
from dpd_amd.training import Muon
from dpd_amd.utils import Int8Inference, Int8Linear, int8_linear, int8_matmul, quantize_rows_int8
from gpu_util import DEV
import operator_oracle as oo
from operator_oracle import TINY, U

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
V = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8 + 2.0 ** -24, torch.float16: 2.0 ** -16 + 2.0 ** -24}


def tokens(m, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=g) * torch.exp(0.5 * torch.randn(1, k, generator=g)) * torch.exp(torch.randn(m, 1, generator=g))).to(dtype)


def close(got, want, size, dtype, n=3, v=0.0):
    got, want = got.double().cpu(), want.cpu()
    tol = (v + (n + 1) * 2.0 ** -23) * size.cpu() + U[dtype] * want.abs() * (1 + 2.0 ** -7) + TINY[dtype]
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), (got - want).abs().max(), ((got - want).abs() / tol).max())


# ------------------------------------------------------------------------------- quantiser
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, k", [(1, 1), (1, 7), (3, 30), (5, 1024), (4, 1025), (2, 4099), (301, 64), (3, 40000)])
def test_quantiser_is_exact(m, k, dtype):
    x = tokens(m, k, dtype, m + k)
    q, s = quantize_rows_int8(x.to(DEV))
    qo, so = oo.quantize_rows(x)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and q.shape == x.shape and s.shape == (m,)
    assert torch.equal(s.cpu(), so) and torch.equal(q.cpu(), qo)


def test_quantiser_half_way_values_and_special_rows():
    half = torch.arange(-127, 127).float() + 0.5
    rows = []
    for scale in (1.0, 2.0 ** -20, 3.0 * 2.0 ** 5, 2.0 ** 100):           # s = scale exactly: every entry but the last lies half-way
        rows.append(torch.cat([half * scale, torch.tensor([127.0 * scale, 0.0])]))
    inf = float("inf")
    extra = torch.zeros(10, 256)
    extra[1, 3], extra[2, 5], extra[3, 7], extra[4, 0] = float("nan"), inf, -inf, 3.4e38
    extra[5, 0], extra[5, 1] = 1e-45, -1e-45                              # below the floor of the scale
    extra[6] = torch.linspace(-1, 1, 256) * 2.0 ** -101
    extra[7] = torch.linspace(-1, 1, 256) * 1e-38
    extra[8] = -2.5
    extra[9, 255] = 2.0 ** -100
    x = torch.cat([torch.stack(rows), extra])
    q, s = quantize_rows_int8(x.to(DEV))
    qo, so = oo.quantize_rows(x)
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(so)) and torch.equal(s.cpu().nan_to_num(7.0), so.nan_to_num(7.0))
    assert torch.equal(q.cpu(), qo)
    assert torch.isnan(s[5:8]).all() and not q[5:8].any() and s[4] > 0


def test_quantiser_layouts():
    x = tokens(12, 96, torch.float32).to(DEV)
    qo, so = oo.quantize_rows(x)
    q, s = quantize_rows_int8(x.view(3, 4, 96))
    assert torch.equal(q.cpu().view(12, 96), qo) and torch.equal(s.cpu().view(12), so) and s.shape == (3, 4)
    wide = torch.full((12, 131), float("nan"), device=DEV)                # what lies between the rows is not looked at
    wide[:, 1:97] = x
    q, s = quantize_rows_int8(wide[:, 1:97])
    assert torch.equal(q.cpu(), qo) and torch.equal(s.cpu(), so)
    q, s = quantize_rows_int8(x.t().contiguous().t())                     # columns one behind the other: copied
    assert torch.equal(q.cpu(), qo)
    q, s = quantize_rows_int8(x[:1].expand(5, 96))
    assert torch.equal(q.cpu(), qo[:1].expand(5, 96))
    q, s = quantize_rows_int8(x[:0])
    assert q.shape == (0, 96) and s.shape == (0,)
    with pytest.raises(ValueError):
        quantize_rows_int8(x[:, :0])
    with pytest.raises(RuntimeError):
        quantize_rows_int8(x.double())


# ------------------------------------------------------------------------------- product
def ints(m, k, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, (m, k), generator=g).to(torch.int8), torch.rand(m, generator=g) + 0.01


@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (1, 5, 16), (2, 3, 129), (17, 515, 1030), (63, 65, 128), (64, 64, 144), (130, 257, 4112), (300, 1, 64),
                                     (1, 300, 2048), (129, 1030, 100), (16, 16, 20000), (513, 770, 384), (5, 4096, 512), (33, 70, 96)])
def test_matmul(m, n, k):
    (a, sa), (b, sb) = ints(m, k, 1), ints(n, k, 2)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(3))
    want, size = oo.matmul(a, sa, b, sb)
    for dtype in TYPES:
        got = int8_matmul(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), out_dtype=dtype)
        assert got.dtype == dtype and got.shape == (m, n)
        finite = want.abs() < 6e4 if dtype == torch.float16 else torch.ones_like(want, dtype=torch.bool)
        close(got[finite.to(DEV)], want[finite], size[finite], dtype)
    for bt in TYPES:
        want, size = oo.matmul(a, sa, b, sb, bias.to(bt))
        close(int8_matmul(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), bias.to(bt).to(DEV)), want, size, torch.float32)


def test_matmul_sum_is_exact_at_the_longest_row():
    k = 131071
    a = torch.full((2, k), -128, dtype=torch.int8)
    a[1] = 127
    a[1, ::2] = -127
    b = torch.full((3, k), -128, dtype=torch.int8)
    b[2] = 1
    one = lambda r: torch.ones(r, device=DEV)
    got = int8_matmul(a.to(DEV), one(2), b.to(DEV), one(3))
    want = (a.long() @ b.long().t()).float()                              # 2147467264 and its neighbours, rounded once to fp32
    assert torch.equal(got.cpu(), want)
    with pytest.raises(ValueError, match="32-bit"):
        int8_matmul(torch.zeros(1, k + 1, dtype=torch.int8, device=DEV), one(1), torch.zeros(1, k + 1, dtype=torch.int8, device=DEV), one(1))


@pytest.mark.parametrize("k", [128, 80, 77])
def test_matmul_strides_and_what_lies_outside(k):
    (a, sa), (b, sb) = ints(40, k, 4), ints(70, k, 5)
    want, size = oo.matmul(a, sa, b, sb)
    for pad, off in ((0, 0), (16, 0), (3, 0), (16, 16), (16, 5)):
        wa = torch.full((40, k + pad + off), 99, dtype=torch.int8, device=DEV)
        wb = torch.full((70, k + pad + off), -77, dtype=torch.int8, device=DEV)
        wa[:, off:off + k], wb[:, off:off + k] = a.to(DEV), b.to(DEV)
        close(int8_matmul(wa[:, off:off + k], sa.to(DEV), wb[:, off:off + k], sb.to(DEV)), want, size, torch.float32)
    close(int8_matmul(a.to(DEV).view(5, 8, k), sa.to(DEV), b.to(DEV), sb.to(DEV)).view(40, 70), want, size, torch.float32)
    got = int8_matmul(a.to(DEV).t().contiguous().t(), sa.to(DEV), b.to(DEV), sb.to(DEV))
    close(got, want, size, torch.float32)


def test_matmul_refusals():
    a, s = torch.zeros(4, 32, dtype=torch.int8, device=DEV), torch.ones(4, device=DEV)
    with pytest.raises(ValueError):
        int8_matmul(a, s, a[:, :16], s)
    with pytest.raises(ValueError, match="a_scale"):
        int8_matmul(a, s[:3], a, s)
    with pytest.raises(ValueError, match="b_scale"):
        int8_matmul(a, s, a, s.double())
    with pytest.raises(ValueError, match="bias"):
        int8_matmul(a, s, a, s, bias=s[:2])
    with pytest.raises(RuntimeError):
        int8_matmul(a.float(), s, a, s)
    with pytest.raises(RuntimeError):
        int8_matmul(a, s, a, s, out_dtype=torch.float64)
    assert int8_matmul(a[:0], s[:0], a, s).shape == (0, 4) and int8_matmul(a, s, a[:0], s[:0]).shape == (4, 0)


# ------------------------------------------------------------------------------- layer and gradients
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (1, 64, 64), (3, 5, 7), (64, 128, 192), (65, 33, 130), (300, 515, 333), (700, 96, 257)])
def test_layer_and_gradients(m, n, k, dtype):
    x, w, b = tokens(m, k, dtype, 6), (tokens(n, k, dtype, 7).float() / k ** 0.5).to(dtype), tokens(1, n, dtype, 8)[0]
    g = tokens(m, n, dtype, 9) * 0.1
    xd, wd, bd = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    y = int8_linear(xd, wd, bd)
    y.backward(g.to(DEV))
    (qx, sx), (qw, sw) = oo.quantize_rows(x), oo.quantize_rows(w)
    close(y.detach(), *oo.matmul(qx, sx, qw, sw, b), dtype)
    (gx, gxs), (gw, gws), (gb, gbs) = oo.gradients(g, qx, sx, qw, sw)
    for t, src in ((xd, x), (wd, w), (bd, b)):
        assert t.grad.dtype == dtype and t.grad.shape == src.shape
    close(xd.grad, gx, gxs, dtype, n, V[dtype])
    close(wd.grad, gw, gws, dtype, m, V[dtype])
    close(bd.grad, gb, gbs, dtype, m)


def test_gradients_against_differences():
    """On inputs that are multiples of their row's scale the layer is linear in steps of that scale, so a difference of two
    outputs, one step apart, is the derivative itself."""
    g = torch.Generator().manual_seed(10)
    qx, qw = torch.randint(-100, 101, (6, 24), generator=g), torch.randint(-100, 101, (9, 24), generator=g)
    qx[:, 0], qw[:, 0] = 127, -127
    x, w = (qx * 2.0 ** -6).to(DEV).requires_grad_(True), (qw * 2.0 ** -8).to(DEV).requires_grad_(True)
    b = torch.randn(9, generator=g).to(DEV).requires_grad_(True)
    c = torch.randint(-8, 9, (6, 9), generator=g).float().to(DEV) / 8
    f = lambda x, w, b: (int8_linear(x, w, b).detach().double() * c.double()).sum().item()
    int8_linear(x, w, b).backward(c)
    for t, step in ((x, 2.0 ** -6), (w, 2.0 ** -8), (b, 2.0 ** -4)):
        flat = t.detach().reshape(-1)
        for i in (1, 5, flat.numel() - 1) if t is not b else (0, 4, 8):
            v = []
            for sign in (1, -1):
                moved = flat.clone()
                moved[i] += sign * step
                v.append(f(*(moved.view(t.shape) if u is t else u.detach() for u in (x, w, b))))
            # values of |y| <= 24 * 127 * 127 * 2^-14 + 4 < 32 with 2^-24 of rounding each, 54 of them, over 2 * 2^-8
            assert abs((v[0] - v[1]) / (2 * step) - t.grad.reshape(-1)[i].item()) <= 54 * 4 * 32 * 2.0 ** -24 / (2 * step) * 2


def test_gradient_subsets_types_and_shapes():
    x, w = tokens(24, 40, torch.bfloat16, 11).view(2, 3, 4, 40).to(DEV), tokens(8, 40, torch.float32, 12).to(DEV)
    b = torch.zeros(8, dtype=torch.float16, device=DEV)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = int8_linear(*full)
    assert y.shape == (2, 3, 4, 8) and y.dtype == torch.bfloat16
    y.sum().backward()                                                    # the gradient of a sum has no strides
    assert [t.grad.dtype for t in full] == [torch.bfloat16, torch.float32, torch.float16]
    assert torch.equal(full[2].grad, torch.full_like(b, 24))
    for i in range(3):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        int8_linear(*some).sum().backward()
        assert all((t.grad is None) == (j != i) for j, t in enumerate(some)) and torch.equal(some[i].grad, full[i].grad)
    xt = x.clone().requires_grad_(True)
    gy = torch.randn(8, 2, 3, 4, device=DEV, dtype=torch.bfloat16).permute(1, 2, 3, 0)
    int8_linear(xt, w).backward(gy)
    xc = x.clone().requires_grad_(True)
    int8_linear(xc, w).backward(gy.contiguous())
    assert torch.equal(xt.grad, xc.grad)
    empty = torch.zeros(0, 40, device=DEV, requires_grad=True)
    wr = w.clone().requires_grad_(True)
    int8_linear(empty, wr).sum().backward()
    assert empty.grad.shape == (0, 40) and not wr.grad.any()
    with pytest.raises(RuntimeError, match="once_differentiable|twice|does not require grad"):
        gx, = torch.autograd.grad(int8_linear(xt.float(), w).sum(), xt, create_graph=True)
        gx.sum().backward()
    with pytest.raises(ValueError):
        int8_linear(x, w[:, :8])
    with pytest.raises(ValueError):
        int8_linear(x, w, b[:3])
    with pytest.raises(RuntimeError):
        int8_linear(x.double(), w)


def test_values_that_are_not_finite():
    x, w = tokens(5, 33, torch.float32, 13), tokens(6, 33, torch.float32, 14)
    x[1, 2], x[3, 0] = float("nan"), float("-inf")
    w[4, 32] = float("inf")
    y = int8_linear(x.to(DEV), w.to(DEV)).cpu()
    nan = torch.zeros(5, 6, dtype=torch.bool)
    nan[[1, 3]] = True
    nan[:, 4] = True
    assert torch.equal(torch.isnan(y), nan) and torch.isfinite(y[~nan]).all()
    xg = tokens(5, 33, torch.float32, 13).to(DEV).requires_grad_(True)
    g = torch.ones(5, 6, device=DEV)
    g[2, 3] = float("inf")
    int8_linear(xg, tokens(6, 33, torch.float32, 14).to(DEV)).backward(g)
    assert torch.isfinite(xg.grad[[0, 1, 3, 4]]).all() and not torch.isfinite(xg.grad[2]).any()


def test_offsets_beyond_32_bits():
    """The last rows of 70000 x 32768 (2.3e9 elements) come out as they do alone.  The product is exact; a gradient's sum may
    be grouped otherwise, so that two results differ by twice what one may be off (head of this file; V is the same for both)."""
    m, k, n, last = 70000, 32768, 24, 40
    gen = torch.Generator(device=DEV).manual_seed(40)
    x = torch.randn(m, k, generator=gen, device=DEV, dtype=torch.bfloat16).requires_grad_(True)
    w = tokens(n, k, torch.float32, 41).to(DEV).requires_grad_(True)
    tail = x.detach()[-last:].clone().requires_grad_(True)
    g = torch.zeros(m, n, device=DEV, dtype=torch.bfloat16)
    g[-last:] = tokens(last, n, torch.bfloat16, 42).to(DEV)
    y = int8_linear(x, w)
    want = int8_linear(tail, w)
    assert torch.equal(y[-last:], want)
    gx, gw = torch.autograd.grad(y, (x, w), g)
    wx, ww = torch.autograd.grad(want, (tail, w), g[-last:])
    assert not gx[:-last].any()
    near = g[-last:].abs().float()
    for a, b, size, terms, u in ((gx[-last:], wx, near @ w.detach().abs(), n, U[torch.bfloat16]), (gw, ww, near.t() @ tail.detach().abs().float(), last, U[torch.float32])):
        assert ((a.double() - b.double()).abs() <= 2 * (u * b.double().abs() * 1.01 + (terms + 1) * 2.0 ** -23 * 1.02 * size.double())).all()
    q, s = quantize_rows_int8(x)
    qt, st = quantize_rows_int8(tail)
    assert torch.equal(q[-last:], qt) and torch.equal(s[-last:], st)
    eng = Int8Inference(dict(zip(("weight", "scale"), quantize_rows_int8(w))))
    assert torch.equal(eng(x.detach())[-last:], want)


# ------------------------------------------------------------------------------- serving
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (1, 515, 1030), (1, 4096, 4096), (2, 64, 30), (3, 100, 12000), (7, 1000, 700), (16, 130, 4096),
                                     (17, 515, 1030), (2, 40, 2047), (3, 4096, 2048), (31, 4097, 60), (32, 33, 1000), (32, 20, 1030), (40, 2048, 1024), (128, 640, 130), (300, 333, 600)])
def test_serving_is_the_quantiser_and_the_product(m, n, k, dtype):
    x, w, b = tokens(m, k, dtype, 15).to(DEV), tokens(n, k, dtype, 16).to(DEV), tokens(1, n, dtype, 17)[0].to(DEV)
    qw, sw = quantize_rows_int8(w)
    for bias in (None, b):
        eng = Int8Inference({"weight": qw, "scale": sw, "bias": bias})
        qx, sx = quantize_rows_int8(x)
        want = int8_matmul(qx, sx, qw, sw, bias, out_dtype=dtype)
        got = eng(x)
        assert torch.equal(got, want)
        out = torch.full((m, n), 7.0, dtype=dtype, device=DEV)
        assert eng(x, out=out) is out and torch.equal(out, want)
    rows = torch.full((m, k + 3), float("nan"), dtype=dtype, device=DEV)
    rows[:, 1:k + 1] = x
    assert torch.equal(eng(rows[:, 1:k + 1]), want)
    close(want, *oo.matmul(*oo.quantize_rows(x.cpu()), qw.cpu(), sw.cpu(), b.cpu()), dtype)


def test_serving_rows_with_special_values_and_one_by_one():
    w = tokens(200, 520, torch.float32, 18).to(DEV)
    eng = Int8Inference(dict(zip(("weight", "scale"), quantize_rows_int8(w))))
    x = tokens(9, 520, torch.float32, 19).to(DEV)
    x[2] = 0
    x[4, 100], x[5, 519] = float("nan"), float("inf")
    y = eng(x)
    assert torch.isnan(y[4:6]).all() and torch.isfinite(y[[0, 1, 2, 3, 6, 7, 8]]).all() and not y[2].any()
    for i in range(9):                                                    # a token's result does not depend on its batch
        assert torch.equal(eng(x[i:i + 1]).nan_to_num(5.0), y[i:i + 1].nan_to_num(5.0))
    assert eng(x[:0]).shape == (0, 200) and eng(x[0]).shape == (200,) and eng(x.view(3, 3, 520)).shape == (3, 3, 200)


def test_serving_refusals():
    w = tokens(8, 32, torch.float32, 20).to(DEV)
    q, s = quantize_rows_int8(w)
    eng = Int8Inference({"weight": q, "scale": s})
    x = tokens(4, 32, torch.float32, 21).to(DEV)
    for bad in (torch.empty(4, 7, device=DEV), torch.empty(4, 8, device=DEV, dtype=torch.bfloat16), torch.empty(8, 4, device=DEV).t()):
        with pytest.raises(RuntimeError, match="out"):
            eng(x, out=bad)
    square = Int8Inference(dict(zip(("weight", "scale"), quantize_rows_int8(tokens(32, 32, torch.float32, 22).to(DEV)))))
    with pytest.raises(RuntimeError, match="share"):
        square(x, out=x)
    with pytest.raises(ValueError):
        eng(x[:, :31])
    with pytest.raises(ValueError):
        Int8Inference({"weight": w, "scale": s})
    with pytest.raises(ValueError):
        Int8Inference({"weight": q, "scale": s[:4]})
    with pytest.raises(RuntimeError):
        eng(x.cpu())
    assert eng(torch.empty(0, x.shape[1], device=DEV), out=torch.empty(0, eng.out_features, device=DEV)).shape == (0, eng.out_features)
    with pytest.raises(RuntimeError, match="gradient"):
        eng(x.clone().requires_grad_(True))
    q.zero_()                                                             # the engine keeps a copy
    assert eng(x).abs().max() > 0


def test_streams_and_graphs():
    """Two engines on two streams at once, and two captured graphs replayed in turn with the program's own work in between."""
    engines = [Int8Inference(dict(zip(("weight", "scale"), quantize_rows_int8(tokens(n, 640, torch.bfloat16, n).to(DEV))))) for n in (300, 1100)]
    xs = [[tokens(m, 640, torch.bfloat16, 23 + m + i).to(DEV) for i in range(4)] for m in (1, 90)]
    want = [[e(x) for x in row] for e, row in zip(engines, xs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(4):
        for j in range(2):
            with torch.cuda.stream(streams[j]):
                got[j].append(engines[j](xs[j][i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for u, v in zip(got, want) for a, b in zip(u, v))
    static = [x[0].clone() for x in xs]
    graphs, outs = [], []
    for j in range(2):
        with torch.cuda.stream(streams[j]):
            engines[j](static[j])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(engines[j](static[j]))
        graphs.append(g)
    for i in (1, 2, 3, 0):
        for j in range(2):
            static[j].copy_(xs[j][i])
        for g in graphs:
            g.replay()
        engines[0](xs[0][0])
        torch.cuda.synchronize()
        for j in range(2):
            assert torch.equal(outs[j], want[j][i])


def test_training_pass_in_a_graph():
    x, w, b = (t.to(DEV) for t in (tokens(70, 90, torch.float32, 24), tokens(50, 90, torch.float32, 25), tokens(1, 50, torch.float32, 26)[0]))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    gy = tokens(70, 50, torch.float32, 27).to(DEV)
    run = lambda: [(y := int8_linear(*leaves)).detach(), *torch.autograd.grad(y, leaves, gy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = run()
    for i in range(4):
        with torch.no_grad():
            leaves[0].copy_(tokens(70, 90, torch.float32, 30 + i))
        g.replay()
        torch.cuda.synchronize()
        for u, v in zip(captured, run()):
            assert torch.equal(u, v)


def test_a_layer_is_trained_and_then_served():
    """Quantiser, product, gradients and optimiser together: two layers with an activation, Muon steps, then 8-bit serving of
    single tokens equals the trained module's own forward bit for bit."""
    torch.manual_seed(28)
    net = torch.nn.Sequential(Int8Linear(48, 160), torch.nn.LeakyReLU(0.2), Int8Linear(160, 10)).to(DEV)
    opt = Muon(net.parameters(), lr=0.02, adam=dict(lr=1e-3))
    x, t = torch.randn(64, 48, device=DEV), torch.randn(64, 10, device=DEV)
    before = [p.detach().clone() for p in net.parameters()]
    for _ in range(3):
        opt.zero_grad()
        torch.nn.functional.mse_loss(net(x), t).backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in net.parameters())
        opt.step()
    assert all(not torch.equal(p.detach(), q) and torch.isfinite(p).all() for p, q in zip(net.parameters(), before))
    first, second = Int8Inference(net[0].get_quantized_weights()), Int8Inference(net[2].get_quantized_weights())
    with torch.no_grad():
        want = net(x)
        got = torch.cat([second(torch.nn.functional.leaky_relu(first(x[i:i + 1]), 0.2)) for i in range(64)])
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m, n, k", [(1, 8, 16), (64, 64, 64), (96, 40, 72), (130, 65, 33), (520, 256, 128)])
def test_gradients_are_rounded_to_their_type_once(m, n, k, dtype):
    """A term g s q enters as two bf16 terms, off by 2^-16 (and g s by 2^-24): the type's own rounding of the result is
    the only one of its size."""
    x, w, g = tokens(m, k, dtype, 50), (tokens(n, k, dtype, 51).float() / k ** 0.5).to(dtype), tokens(m, n, dtype, 52) * 0.1
    xd, wd = (t.to(DEV).requires_grad_(True) for t in (x, w))
    int8_linear(xd, wd).backward(g.to(DEV))
    (gx, gxs), (gw, gws), _ = oo.gradients(g, *oo.quantize_rows(x), *oo.quantize_rows(w))
    close(xd.grad, gx, gxs, dtype, n, 2.0 ** -16 + 2.0 ** -24)
    close(wd.grad, gw, gws, dtype, m, 2.0 ** -16 + 2.0 ** -24)


def test_the_weights_of_an_engine_are_not_rebound():
    """The calls use the addresses of what the engine holds, so nothing else can take its place (and free it)."""
    eng = Int8Inference({**dict(zip(("weight", "scale"), quantize_rows_int8(tokens(8, 32, torch.float32, 20).to(DEV)))), "bias": torch.ones(8, device=DEV)})
    x = tokens(4, 32, torch.float32, 21).to(DEV)
    want = eng(x)
    for name in ("scale", "image", "bias"):
        with pytest.raises(AttributeError):
            setattr(eng, name, torch.zeros_like(getattr(eng, name)))
    assert torch.equal(eng(x), want) and eng.scale.shape == (8,) and eng.image.shape == (8, 128) and torch.equal(eng.bias, torch.ones(8, device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [(1 << 20) + 777, 2_200_001])
def test_more_tokens_than_one_backward_call_takes(m, dtype):
    """Rows of whole numbers with a largest of 127 have the scale 1, and every partial sum below is a whole number of fewer than
    24 bits: the gradients are exact whatever the order.  (|gw| <= |sum of m terms of at most 127|: a walk of m steps of
    127 would reach 2^24 only at 114 times its deviation.)"""
    n, k = 20, 16
    gen = torch.Generator().manual_seed(60)
    x, w = torch.randint(-3, 4, (m, k), generator=gen), torch.randint(-3, 4, (n, k), generator=gen)
    x[:, 0], w[:, 0] = 127, 127
    g = torch.randint(-1, 2, (m, n), generator=gen)
    xd, wd, bd = (t.to(dtype).to(DEV).requires_grad_(True) for t in (x, w, torch.zeros(n)))
    y = int8_linear(xd, wd, bd)
    for leaves in ((xd, wd, bd), (xd,), (wd,), (bd,)):
        for t, got in zip(leaves, torch.autograd.grad(y, leaves, g.to(dtype).to(DEV), retain_graph=True)):
            want = (g.double() @ w.double() if t is xd else g.double().t() @ x.double() if t is wd else g.double().sum(0)).to(dtype)
            assert got.dtype == dtype and torch.equal(got.cpu(), want)


def test_output_features_that_have_no_gradient_of_x_are_refused_before_the_forward():
    w = torch.ones(1398081, 1, device=DEV, requires_grad=True)
    x = torch.ones(2, 1, device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="output features"):
        int8_linear(x, w)
    with torch.no_grad():
        assert int8_linear(x, w).shape == (2, 1398081)
    gw, = torch.autograd.grad(int8_linear(x.detach(), w).sum(), w)
    assert torch.equal(gw, torch.full_like(w, 2.0))


def test_gradients_are_not_dropped_in_silence():
    import torch.autograd.forward_ad as fwd
    from dpd_amd.utils import orthogonalize
    x = tokens(4, 32, torch.float32, 21).to(DEV)
    q, s = quantize_rows_int8(x)
    eng, leaf = Int8Inference({"weight": q, "scale": s}), lambda t: t.clone().requires_grad_(True)
    for call in (lambda: int8_matmul(q, leaf(s), q, s), lambda: int8_matmul(q, s, q, leaf(s)), lambda: int8_matmul(q, s, q, s, bias=leaf(s)),
                 lambda: eng(leaf(x)), lambda: orthogonalize(leaf(x))):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        for call in (lambda: int8_matmul(q, dual(s), q, s), lambda: int8_matmul(q, s, q, s, bias=dual(s)), lambda: eng(dual(x)), lambda: orthogonalize(dual(x)),
                     lambda: quantize_rows_int8(dual(x))):
            with pytest.raises(RuntimeError, match="gradient"):
                call()
        with pytest.raises((RuntimeError, NotImplementedError)):
            int8_linear(dual(x), x)
        assert torch.equal(eng(x), int8_matmul(q, s, q, s))               # tensors without a tangent pass


def test_serving_into_a_part_of_one_buffer():
    """x and out may be parts of one allocation, and may not overlap in whatever way they came to."""
    w = tokens(8, 32, torch.float32, 20).to(DEV)
    eng = Int8Inference(dict(zip(("weight", "scale"), quantize_rows_int8(w))))
    x = tokens(4, 32, torch.float32, 21).to(DEV)
    want = eng(x)
    buf = torch.empty(32 + 128 + 32, device=DEV)
    for lo in (0, 160):
        part, out = buf[32:160].view(4, 32), buf[lo:lo + 32].view(4, 8)
        part.copy_(x)
        assert eng(part, out=out) is out and torch.equal(out, want) and torch.equal(part, x)
    for lo in (1, 32, 100, 159):
        with pytest.raises(RuntimeError, match="share"):
            eng(part, out=buf[lo:lo + 32].view(4, 8))
    rows = buf[:160].view(4, 40)[:, :32]                                  # rows with gaps, the last one without
    rows.copy_(x)
    assert torch.equal(eng(rows, out=buf[152:184].view(4, 8)), want)
    with pytest.raises(RuntimeError, match="share"):
        eng(rows, out=buf[151:183].view(4, 8))
    turned = buf[:128].view(32, 4)
    turned.copy_(x.t())
    assert torch.equal(eng(turned.t(), out=buf[:32].view(4, 8)), want)    # copied before anything is written


def test_matmul_rows_far_apart():
    (a, sa), (b, sb) = ints(3, 64, 70), ints(5, 64, 71)
    want, size = oo.matmul(a, sa, b, sb)
    far = torch.zeros(5, 9_000_000, dtype=torch.int8, device=DEV)
    far[:3, 16:80], far[:, 100:164] = a.to(DEV), b.to(DEV)
    x, y = far[:3, 16:80], far[:, 100:164]
    close(int8_matmul(x, sa.to(DEV), y, sb.to(DEV)), want, size, torch.float32)
    close(int8_matmul(x[1:2], sa[1:2].to(DEV), y, sb.to(DEV)), want[1:2], size[1:2], torch.float32)
