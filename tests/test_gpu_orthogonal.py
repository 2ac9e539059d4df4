"""The Newton-Schulz iteration and the Muon step against their 64-bit statement (operator_oracle.py).

Tolerances, before any run: operator_oracle.iterate repeats the iteration in 64 bits with the documented roundings of the
factors and nothing else ("fp16" one half, "two" halves, "fp32"); its distance D from the exact iterate is what those
roundings do to this matrix.  The kernel's own roundings are others of the same size, and its fp32 sums (over up to c terms,
2^-24 each) come on top: allowed are 3 D in the Frobenius norm (a sum of independent roundings of one size varies far less),
for the accurate forms 3 D(fp32) + 3 D(two) + sqrt(c) 2^-22 |X| to count the sums, and half a step of the output type."""
import copy

import pytest
import torch

import dpd_amd  # noqa: F401
from dpd_amd.training import Muon
from dpd_amd.utils import orthogonalize
from gpu_util import DEV
import operator_oracle as oo
from operator_oracle import COEF, U

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def update(r, c, seed=0):
    g = torch.Generator().manual_seed(seed)
    return 1e-2 * torch.randn(r, c, generator=g) * torch.exp(0.5 * torch.randn(r, 1, generator=g)) * torch.exp(0.5 * torch.randn(1, c, generator=g))


def small(r, c):
    return min(r, c) <= 64 and max(r, c) <= 128


def allowed(x, want, accurate, **kw):
    """How far an iterate of x may be from `want`, in the Frobenius norm, before it is rounded to its type."""
    dist = lambda form: float((oo.iterate(x, form=form, **kw) - want).norm())
    sums = max(x.shape) ** 0.5 * 2.0 ** -22 * float(want.norm())
    if small(*x.shape):
        return 3 * dist("fp32") + sums
    return 3 * dist("fp32") + 3 * dist("two") + sums if accurate else 3 * dist("fp16") + 3 * dist("fp32") + sums


def check(got, x, dtype, accurate, **kw):
    want = oo.iterate(x, **kw)
    tol = allowed(x, want, accurate, **kw) + U[dtype] * float(want.norm()) * 1.01
    err = float((got.double().cpu() - want).norm())
    assert err <= tol, (err, tol, float(want.norm()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r, c", [(1, 1), (1, 9), (9, 1), (2, 16), (32, 30), (16, 32), (64, 4), (64, 64), (64, 128), (128, 63), (1, 129), (65, 65), (64, 129),
                                  (129, 64), (200, 70), (127, 300), (256, 256), (130, 515)])
def test_iterate(r, c, dtype):
    x = update(r, c, r + c).to(dtype)
    got = orthogonalize(x.to(DEV))
    assert got.shape == x.shape and got.dtype == dtype
    check(got, x, dtype, dtype != torch.bfloat16)


@pytest.mark.parametrize("accurate", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_both_forms_of_the_factors(dtype, accurate):
    for r, c in ((150, 220), (70, 100), (40, 400), (300, 33)):
        x = update(r, c, 3).to(dtype)
        check(orthogonalize(x.to(DEV), accurate=accurate), x, dtype, accurate)


def test_batches_and_layouts():
    x = torch.stack([update(70, 90, s) * 10.0 ** (s - 3) for s in range(6)]).view(2, 3, 70, 90).to(DEV)
    got = orthogonalize(x)
    assert got.shape == x.shape
    for i in range(6):
        one = orthogonalize(x.view(6, 70, 90)[i])
        assert torch.equal(got.view(6, 70, 90)[i], one)
        check(one, x.view(6, 70, 90)[i].cpu(), torch.float32, True)
    for r, c in ((40, 30), (70, 90)):
        y = update(r, c, 9).to(DEV)
        assert torch.equal(orthogonalize(y.t().contiguous().t()), orthogonalize(y))
        assert torch.equal(orthogonalize(y.t()), orthogonalize(y.t().contiguous()))
        pad = torch.full((r, c + 5), float("nan"), device=DEV)
        pad[:, 2:c + 2] = y
        assert torch.equal(orthogonalize(pad[:, 2:c + 2]), orthogonalize(y))
    assert orthogonalize(torch.zeros(0, 70, 90, device=DEV)).shape == (0, 70, 90)
    assert orthogonalize(torch.zeros(3, 0, 90, device=DEV)).shape == (3, 0, 90)


@pytest.mark.parametrize("r, c", [(20, 30), (100, 140)])
def test_special_values(r, c):
    zero = torch.zeros(r, c, device=DEV)
    assert not orthogonalize(zero).any()
    for bad in (float("nan"), float("inf"), float("-inf")):
        x = update(r, c, 1).to(DEV)
        x[r // 2, 3] = bad
        assert torch.isnan(orthogonalize(x)).all()
        both = torch.stack([x, update(r, c, 2).to(DEV)])
        out = orthogonalize(both)
        assert torch.isnan(out[0]).all() and torch.equal(out[1], orthogonalize(both[1]))
    for scale in (1e30, 1e-30, 3e37):                                     # squares far outside fp32
        x = update(r, c, 4) * scale
        check(orthogonalize(x.to(DEV), eps=1e-45), x, torch.float32, True, eps=1e-45)
    one = torch.zeros(r, c)
    one[1, 2] = -5.0                                                      # a single entry: the others stay zero
    got = orthogonalize(one.to(DEV)).cpu()
    check(got, one, torch.float32, True)
    assert int((got != 0).sum()) == 1
    tiny = update(r, c, 5) * 1e-9                                         # below eps: divided by eps
    check(orthogonalize(tiny.to(DEV), eps=1e-2), tiny, torch.float32, True, eps=1e-2)


@pytest.mark.parametrize("r, c", [(30, 44), (90, 130)])
def test_steps_and_coefficients(r, c):
    x = update(r, c, 6)
    for kw in (dict(steps=1), dict(steps=12, coef=(1.875, -1.25, 0.375)), dict(coef=[(3.9, -8.0, 4.5), (3.0, -4.0, 2.0), COEF], steps=3)):
        given = dict(steps=kw["steps"], coefficients=kw.get("coef", COEF))
        check(orthogonalize(x.to(DEV), **given), x, torch.float32, True, **kw)
    polar = orthogonalize(x.to(DEV), steps=20, coefficients=(1.875, -1.25, 0.375)).double().cpu()
    # 20 steps of the convergent triple from singular values of at least 1e-3 of the norm: the polar factor, to fp32
    assert float((polar @ polar.t() - torch.eye(r, dtype=torch.float64)).norm()) <= 1e-4
    for bad in ((30.0, 0.0, 0.0), (float("nan"), 0.0, 0.0)):
        with pytest.raises(ValueError, match="out of range"):
            orthogonalize(x.to(DEV), coefficients=bad)
    for bad in (dict(steps=0), dict(steps=40), dict(eps=0.0), dict(coefficients=(1.0,))):
        with pytest.raises(ValueError):
            orthogonalize(x.to(DEV), **bad)
    with pytest.raises(RuntimeError, match="gradient"):
        orthogonalize(x.to(DEV).requires_grad_(True))
    with pytest.raises(RuntimeError):
        orthogonalize(x.to(DEV).double())
    with pytest.raises(ValueError):
        orthogonalize(x.to(DEV)[0])


def test_streams_graphs_and_repeats():
    xs = [update(300, 420, s).to(DEV) for s in range(4)]
    want = [orthogonalize(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None] * 4
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = orthogonalize(xs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = xs[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = orthogonalize(static)
    for i in (1, 2, 3, 0):
        static.copy_(xs[i])
        g.replay()
        orthogonalize(xs[(i + 1) % 4])
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])


# ------------------------------------------------------------------------------- optimiser
def muon_oracle(p, g, m, lr, mu, nesterov, wd):
    m = mu * m.double() + g.double()
    u = g.double() + mu * m if nesterov else m
    o = oo.iterate(u)
    f = lr * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
    return p.double() * (1 - lr * wd) - f * o, m, u, f


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(dtype, nesterov):
    shapes = [(32, 30), (16, 32), (2, 16), (64, 4), (1, 16), (150, 70), (70, 200)]
    ps = [torch.nn.Parameter(update(r, c, r).to(dtype).to(DEV)) for r, c in shapes]
    opt = Muon(ps, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
    p0, m0 = [p.detach().cpu() for p in ps], [torch.zeros(s) for s in shapes]
    for step in range(2):
        for i, p in enumerate(ps):
            p.grad = update(*shapes[i], 100 * step + i).to(dtype).to(DEV)
        versions = [p._version for p in ps]
        opt.step()
        assert all(p._version > v for p, v in zip(ps, versions))
        for i, p in enumerate(ps):
            want, m, u, f = muon_oracle(p0[i], p.grad.cpu(), m0[i], 0.05, 0.9, nesterov, 0.1)
            got_m = opt.state[p]["momentum_buffer"]
            assert got_m.dtype == torch.float32
            # three roundings of 2^-24 (mu as an fp32 constant, the product, the sum), to first order, of at most mu |m| + |g|
            assert ((got_m.cpu().double() - m).abs() <= 3.01 * 2.0 ** -24 * (0.9 * m0[i].double().abs() + p.grad.cpu().double().abs())).all()
            # u carries roundings of 2^-23 of its parts; a relative change d of the input moves an iterate by at most
            # (max slope)^5 = 3.45^5 < 500 times as much
            tol = f * (allowed(u, oo.iterate(u), dtype != torch.bfloat16) + 500 * 2.0 ** -22) + (U[dtype] + 2.0 ** -22) * float(want.norm()) * 1.01
            assert float((p.detach().cpu().double() - want).norm()) <= tol, (shapes[i], step)
        p0, m0 = [p.detach().cpu() for p in ps], [opt.state[p]["momentum_buffer"].cpu() for p in ps]


def test_muon_groups_biases_and_state():
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.Linear(30, 5)).to(DEV)
    twin = torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.Linear(30, 5)).to(DEV)
    twin.load_state_dict(net.state_dict())
    opt, adam = Muon(net.parameters(), adam=dict(lr=1e-2)), torch.optim.Adam([twin[0].bias, twin[1].bias], lr=1e-2)
    x = torch.randn(8, 20, device=DEV)

    def one(o, n):
        o.zero_grad()
        n(x).square().mean().backward()
        o.step()
    one(opt, net)
    twin(x).square().mean().backward()
    adam.step()
    assert torch.equal(net[0].bias, twin[0].bias) and torch.equal(net[1].bias, twin[1].bias)
    # a second optimiser with the saved state goes on exactly as the first
    twin.load_state_dict(net.state_dict())
    other = Muon(twin.parameters(), adam=dict(lr=1e-2))
    other.load_state_dict(copy.deepcopy(opt.state_dict()))                # Adam's loaded state is not copied by the base class
    for _ in range(2):
        one(opt, net)
        one(other, twin)
    assert all(torch.equal(a, b) for a, b in zip(net.parameters(), twin.parameters()))


def test_muon_copies():
    """A deep copy of the optimiser goes on by itself, biases included."""
    torch.manual_seed(1)
    net = torch.nn.Linear(20, 30).to(DEV)
    opt = Muon(net.parameters(), adam=dict(lr=1e-2))
    net(torch.ones(4, 20, device=DEV)).square().mean().backward()
    opt.step()
    twin = copy.deepcopy(opt)
    mine, other = [p for g in opt.param_groups for p in g["params"]], [p for g in twin.param_groups for p in g["params"]]
    for p, q in zip(mine, other):
        q.grad = p.grad.clone()
    opt.step()
    twin.step()
    assert all(torch.equal(p, q) and p.data_ptr() != q.data_ptr() for p, q in zip(mine, other))


def test_muon_many_matrices_and_refusals():
    shapes = [(1 + i % 7, 3 + i % 11) for i in range(60)]                 # more than one launch's table
    ps = [torch.nn.Parameter(update(r, c, i).to(DEV)) for i, (r, c) in enumerate(shapes)]
    gs = [update(r, c, 200 + i).to(DEV) for i, (r, c) in enumerate(shapes)]
    alone = []
    for p, g in zip(ps, gs):
        q = torch.nn.Parameter(p.detach().clone())
        q.grad = g
        Muon([q]).step()
        alone.append(q)
        p.grad = g
    Muon(ps).step()
    assert all(torch.equal(p, q) for p, q in zip(ps, alone))
    p = torch.nn.Parameter(torch.randn(6, 4, device=DEV).t())
    p.grad = torch.randn(4, 6, device=DEV)
    with pytest.raises(RuntimeError, match="contiguous"):
        Muon([p]).step()
    q = torch.nn.Parameter(torch.randn(6, 4, device=DEV))
    q.grad = torch.randn(4, 6, device=DEV).t()                            # a gradient may have any layout
    r = torch.nn.Parameter(q.detach().clone())
    r.grad = q.grad.contiguous()
    Muon([q]).step()
    Muon([r]).step()
    assert torch.equal(q, r)


def test_offsets_beyond_32_bits():
    """The last of 5 matrices of 256 x 1700000 (2.2e9 elements) comes out as it does alone.  This looks for addresses, not for
    roundings: sums may be grouped otherwise, which the factors' and the result's roundings (2^-11, 2^-8) turn into less
    than 2^-6; a wrong address is off by the whole value."""
    gen = torch.Generator(device=DEV).manual_seed(50)
    x = torch.randn(5, 256, 1_700_000, generator=gen, device=DEV, dtype=torch.bfloat16)
    y, want = orthogonalize(x)[4], orthogonalize(x[4])
    assert torch.linalg.vector_norm(y.float() - want.float()) <= 2.0 ** -6 * torch.linalg.vector_norm(want.float())
    tall = orthogonalize(x[3:].transpose(1, 2).contiguous())[1]
    assert torch.linalg.vector_norm(tall.t().float() - want.float()) <= 2.0 ** -6 * torch.linalg.vector_norm(want.float())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_muon_matrices_of_one_size_go_together(dtype):
    """Wide and tall matrices of the same two sides share launches: each comes out as it does alone (the tile that is chosen
    may differ, and with it the order of a sum), within the tolerance of its step."""
    shapes = [(70, 200), (200, 70), (96, 96), (70, 200), (200, 70), (96, 96), (200, 70)] + [(130, 66)] * 9 + [(40, 40), (66, 130)]
    ps = [torch.nn.Parameter(update(r, c, i).to(dtype).to(DEV)) for i, (r, c) in enumerate(shapes)]
    p0 = [p.detach().cpu() for p in ps]
    for i, p in enumerate(ps):
        p.grad = update(*p.shape, 300 + i).to(dtype).to(DEV)
    opt = Muon(ps, lr=0.05, momentum=0.9)
    opt.step()
    for p, before in zip(ps, p0):
        want, m, u, f = muon_oracle(before, p.grad.cpu(), torch.zeros(p.shape), 0.05, 0.9, True, 0.0)
        tol = f * (allowed(u, oo.iterate(u), dtype != torch.bfloat16) + 500 * 2.0 ** -22) + (U[dtype] + 2.0 ** -22) * float(want.norm()) * 1.01
        assert float((p.detach().cpu().double() - want).norm()) <= tol, p.shape
        assert torch.equal(opt.state[p]["momentum_buffer"], p.grad.float())


def test_muon_in_a_graph():
    ps = [torch.nn.Parameter(update(r, c, r).to(DEV)) for r, c in ((30, 32), (140, 90))]
    for p in ps:
        p.grad = torch.zeros_like(p)
    with pytest.raises(RuntimeError, match="momentum"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            Muon(ps).step()
    opt, eager_ps = Muon(ps), [torch.nn.Parameter(p.detach().clone()) for p in ps]
    eager = Muon(eager_ps)
    for o, q in ((opt, ps), (eager, eager_ps)):
        for p in q:
            o.state[p]["momentum_buffer"] = torch.zeros_like(p)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step()
    for i in range(4):
        for p, q in zip(ps, eager_ps):
            p.grad.copy_(update(*p.shape, 50 + i))
            q.grad = p.grad.clone()
        g.replay()
        eager.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ps, eager_ps))


def test_training_command_with_muon(tmp_path):
    from dpd_amd.train import main
    args = ["--config", "", "--rows", "16", "--seq-len", "133", "--epochs", "2", "--stage1-epochs", "1", "--batch-size", "8", "--qat", "--optimizer", "muon",
            "--output-dir", str(tmp_path)]
    metrics = main(args)
    assert all(v == v for v in metrics.values()) and metrics["stage"] == 2
    main(args[:-2] + ["--epochs", "3", "--output-dir", str(tmp_path), "--resume", str(tmp_path / "latest.pth")])
    ck = torch.load(tmp_path / "latest.pth", weights_only=True)
    assert ck["epoch"] == 2 and ck["g_optimizer_state_dict"]["param_groups"][0]["kind"] == "matrix"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("r, c", [(65, 65), (70, 200), (300, 33), (130, 515), (600, 300)])
def test_the_default_is_off_by_its_types_rounding_alone(r, c, dtype):
    """An entry v that is computed with an error e comes out within e + U (|v| + e): what is left of an entry's distance behind
    U |v| is at most (1 + U) e, and e is that of the accurate form whatever the type is."""
    x = update(r, c, r + 2 * c).to(dtype)
    want = oo.iterate(x)
    left = ((orthogonalize(x.to(DEV)).double().cpu() - want).abs() - U[dtype] * want.abs()).clamp_min(0.0)
    assert float(left.norm()) <= (1 + U[dtype]) * allowed(x, want, True), (float(left.norm()), float(want.norm()))


@pytest.mark.parametrize("small_part", [1e-2, 1e-3, 1e-4, 1e-6])
@pytest.mark.parametrize("along", ["rows", "columns"])
@pytest.mark.parametrize("r, c", [(40, 60), (100, 120), (150, 300), (410, 260)])
def test_rows_and_columns_far_smaller_than_the_others(r, c, along, small_part):
    """Every second row or column scaled down: each of them comes out as accurate as the others, relative to itself.  Allowed,
    as for the whole matrix: three times what rounding X, A and B to fp32 and to 22 bits does to the worst of these rows, and the
    sums' roundings (max(r, c)^(1/2) 2^-22)."""
    x = update(r, c, 7)
    dim = 1 if along == "rows" else 0
    (x[::2] if dim else x[:, ::2]).mul_(small_part)
    want = oo.iterate(x)
    norm = want.norm(dim=dim)
    worst = lambda y: float(((y - want).norm(dim=dim) / norm).max())
    tol = 3 * worst(oo.iterate(x, form="fp32")) + 3 * worst(oo.iterate(x, form="22 bits")) + max(r, c) ** 0.5 * 2.0 ** -22 + U[torch.float32]
    err = worst(orthogonalize(x.to(DEV)).double().cpu())
    assert err <= tol, (err, tol)


def test_muon_refuses_before_the_first_weight_changes():
    def fresh():
        ps = [torch.nn.Parameter(update(r, c, r).to(DEV)) for r, c in ((30, 32), (20, 12))] + [torch.nn.Parameter(torch.ones(5, device=DEV))]
        for p in ps:
            p.grad = torch.ones_like(p)
        return ps, [p.detach().clone() for p in ps]

    wild = [(3.4, -4.7, 2.0), (30.0, 0.0, 0.0)]                           # in range only as two triples; refused by the library
    for groups, spoil in ((lambda ps: [{"params": ps[:1]}, {"params": ps[1:2], "steps": 2, "coefficients": wild}], lambda ps, o: None),
                          (lambda ps: [{"params": ps[:1]}, {"params": ps[1:2]}], lambda ps, o: o.param_groups[1].update(steps=50)),
                          (lambda ps: [{"params": ps[:1]}, {"params": ps[1:2]}], lambda ps, o: o.param_groups[1].update(eps=-1.0)),
                          (lambda ps: [{"params": ps[:1]}, {"params": ps[1:2]}], lambda ps, o: setattr(ps[1], "data", ps[1].data.double())),
                          (lambda ps: ps, lambda ps, o: setattr(ps[2], "grad", torch.ones(5, device=DEV).to_sparse()))):
        ps, before = fresh()
        opt = Muon(groups(ps))
        spoil(ps, opt)
        with pytest.raises((ValueError, RuntimeError)):
            opt.step()
        torch.cuda.synchronize()
        assert torch.equal(ps[0], before[0]) and not any(s["momentum_buffer"].any() for s in opt.state.values() if "momentum_buffer" in s)
    # the same memory under two names would be updated by two workgroups at once
    ps, before = fresh()
    other = torch.nn.Parameter(ps[0].data)
    other.grad = ps[0].grad
    with pytest.raises(ValueError, match="memory"):
        Muon([ps[0], other]).step()
    assert torch.equal(ps[0], before[0])
