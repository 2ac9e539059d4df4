"""Every tile of the products behind the 8-bit layer and the orthogonalised update (csrc/gemm_nt.h), forced in turn on small
ragged sizes, and large sizes at which the rule takes the large tiles by itself.

The tiles differ in their LDS layout, stages, groups along the sum, read-ahead and turned store, so each is run with one
step, with fewer steps than stages, with a short last step and with many; with rows and columns that end inside a tile; with odd row
strides of the result; symmetric products with more than one band of eight tile rows.  Tolerances are those of the tests of
the layer and of the iteration, which state them."""
import pytest
import torch

import dpd_amd  # noqa: F401
from dpd_amd import _lib as L
from dpd_amd.utils import int8_linear, int8_matmul, orthogonalize
from gpu_util import DEV
import operator_oracle as oo
from operator_oracle import U
from test_gpu_int8_linear import V, close, ints, tokens
from test_gpu_orthogonal import update

pytestmark = pytest.mark.gpu

TILES = range(11)


@pytest.fixture
def force():
    yield lambda tile: L.check(L.lib().dpd_set_option(b"product_tile", tile))
    L.check(L.lib().dpd_set_option(b"product_tile", -1))


@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (3, 70, 128), (257, 300, 1040), (515, 391, 400), (300, 517, 1030), (130, 260, 128 * 9)])
@pytest.mark.parametrize("tile", TILES)
def test_int8_product(tile, m, n, k, force):
    (a, sa), (b, sb) = ints(m, k, 1), ints(n, k, 2)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(3))
    want, size = oo.matmul(a, sa, b, sb, bias)
    args = [t.to(DEV) for t in (a, sa, b, sb, bias)]
    force(tile)
    got = int8_matmul(*args)
    close(got, want, size, torch.float32)
    half = int8_matmul(*args, out_dtype=torch.bfloat16)
    force(-1)
    assert torch.equal(got, int8_matmul(*args)) and torch.equal(half, int8_matmul(*args, out_dtype=torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m, n, k", [(2, 3, 5), (300, 515, 333), (580, 70, 264)])
@pytest.mark.parametrize("tile", TILES)
def test_gradients(tile, m, n, k, dtype, force):
    x, w, g = tokens(m, k, dtype, 6), (tokens(n, k, dtype, 7).float() / k ** 0.5).to(dtype), tokens(m, n, dtype, 9) * 0.1
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    force(tile)
    y = int8_linear(xd, wd)
    y.backward(g.to(DEV))
    (qx, sx), (qw, sw) = oo.quantize_rows(x), oo.quantize_rows(w)
    close(y.detach(), *oo.matmul(qx, sx, qw, sw), dtype)
    (gx, gxs), (gw, gws), _ = oo.gradients(g, qx, sx, qw, sw)
    close(xd.grad, gx, gxs, dtype, n, V[dtype])
    close(wd.grad, gw, gws, dtype, m, V[dtype])


def check(got, x, accurate):
    """The tolerance of an iterate of fp32 input (head of the iteration's tests), in 64 bits on the device."""
    x = x.to(DEV)
    want = oo.iterate(x, device=DEV)
    dist = lambda form: float((oo.iterate(x, form=form, device=DEV) - want).norm())
    tol = 3 * dist("fp32") + 3 * dist("two" if accurate else "fp16") + (max(x.shape) ** 0.5 * 2.0 ** -22 + U[torch.float32] * 1.01) * float(want.norm())
    err = float((got.double() - want).norm())
    assert err <= tol, (err, tol, float(want.norm()))
    # an entry that is left out or stored elsewhere is off by about its size, far more than any of these roundings
    assert float((got.double() - want).abs().max()) <= 0.05 * float(want.abs().max())


@pytest.mark.parametrize("accurate", [False, True])
@pytest.mark.parametrize("r, c", [(131, 140), (300, 517), (643, 290)])
@pytest.mark.parametrize("tile", TILES)
def test_iteration(tile, r, c, accurate, force):
    x = torch.stack([update(r, c, s) for s in (1, 2)])
    force(tile)
    got = orthogonalize(x.to(DEV), accurate=accurate)
    for i in range(2):
        check(got[i], x[i], accurate)


@pytest.mark.parametrize("accurate", [False, True])
@pytest.mark.parametrize("tile", [t for t in TILES if t not in (1, 5, 9)])
def test_symmetric_products_of_several_bands(tile, accurate, force):
    """8 tile rows a band: a matrix of 2100 rows has two bands of the largest tile."""
    x = update(2100, 2130, 5)
    force(tile)
    check(orthogonalize(x.to(DEV), accurate=accurate), x, accurate)


@pytest.mark.parametrize("batch, r, c", [(3, 777, 1000), (1, 1030, 1500), (1, 2050, 1990), (1, 900, 4100), (1, 4100, 4090)])
def test_iterations_by_the_rule(batch, r, c):
    x = torch.stack([update(r, c, s) for s in range(batch)])
    for accurate in (False, True):
        got = orthogonalize(x.to(DEV), accurate=accurate)
        for i in range(batch):
            check(got[i], x[i], accurate)


@pytest.mark.parametrize("m, n, k", [(4999, 4100, 2064), (2050, 3001, 1030), (128, 16390, 640), (1300, 700, 4112)])
def test_layers_by_the_rule(m, n, k):
    """Large layers against 64 bits on the device."""
    x, w, g = tokens(m, k, torch.bfloat16, 6).to(DEV), (tokens(n, k, torch.bfloat16, 7).float() / k ** 0.5).bfloat16().to(DEV), (tokens(m, n, torch.bfloat16, 9) * 0.1).to(DEV)
    xd, wd = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = int8_linear(xd, wd)
    y.backward(g)
    f = [t.to(DEV) for t in (*oo.quantize_rows(x), *oo.quantize_rows(w))]
    close(y.detach(), *oo.matmul(*f), torch.bfloat16)
    (gx, gxs), (gw, gws), _ = oo.gradients(g, *f)
    close(xd.grad, gx, gxs, torch.bfloat16, n, 2.0 ** -16 + 2.0 ** -24)
    close(wd.grad, gw, gws, torch.bfloat16, m, 2.0 ** -16 + 2.0 ** -24)
