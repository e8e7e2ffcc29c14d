"""Layer norm where float32 could lose what its definition keeps: rows of one value at widths whose reciprocal is rounded,
gradients of rows of a large mean.

A 16-bit value has at most 11 significant bits and a width is 8 * m with m <= 4096, so every sum of equal values of a row is
a float32 and their quotient is the value itself: mean, y and scale are compared bit for bit.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
BF, FP, F32, E4, I8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8
# one wave a row, four, eight and sixteen waves, rows that a lane cannot hold; each of widths that are no power of two
WIDTHS = [56, 520, 1000, 1032, 1992, 2056, 2880, 5000, 6152, 7168, 8200, 14336, 16392, 20000, 32760]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _constant(m, n, dtype):
    values = torch.tensor([3.0, 7.0, 1000.0, -0.3, 2.0**-14, -30000.0, 0.0], device=DEV).to(dtype)
    return values.repeat(-(-m // 7))[:m, None].expand(m, n).contiguous()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m", [7, 600])
@pytest.mark.parametrize("n", WIDTHS)
def test_a_row_of_one_value_is_its_bias(pkg, dtype, m, n):
    x = _constant(m, n, dtype)
    g = _gen(n)
    w, b = (1 + torch.randn(n, device=DEV, generator=g)).to(dtype), torch.randn(n, device=DEV, generator=g).to(dtype)
    o = pkg.layer_norm(x, w, b)
    assert torch.equal(o.mean, x[:, 0].float()) and bool((o.rstd == o.rstd[0]).all())
    assert torch.equal(o.y, b.expand(m, n))
    # of sums that are rounded to one value, too
    h = pkg.layer_norm(x, w, b, x)
    assert torch.equal(h.mean, h.h[:, 0].float()) and torch.equal(h.y, b.expand(m, n))
    # 8-bit outputs: nothing but zeros without a bias
    q = pkg.layer_norm(x, w, None, None, 1e-5, I8, "row")
    assert bool((q.y == 0).all()) and bool((q.scale == 1).all())
    e = pkg.layer_norm(x, w, None, None, 1e-5, E4)
    assert bool((e.y.float() == 0).all()) and float(e.scale) == 1.0


@pytest.mark.parametrize("m", [7, 600])
@pytest.mark.parametrize("n", WIDTHS)
def test_a_row_of_one_value_without_eps_is_nan(pkg, m, n):
    x = _constant(m, n, FP)
    w = torch.ones(n, device=DEV, dtype=FP)
    o = pkg.layer_norm(x, w, None, None, 0.0)
    assert torch.equal(o.mean, x[:, 0].float()) and bool(o.y.isnan().all())
    q = pkg.layer_norm(x, w, None, None, 0.0, I8, "row")
    assert bool(q.scale.isnan().all()) and bool((q.y == 0).all())


HALF = {BF: 2.0**-8, FP: 2.0**-11, F32: 2.0**-24}
TINY = {BF: 2.0**-134, FP: 2.0**-25, F32: 2.0**-150}  # half the least subnormal
F = 1e-5  # of the sum of magnitudes: a float32 chain of at most 64 terms a lane and a tree, below 100 * 2^-24


# few rows, many rows of each number of waves and pieces, and rows whose inputs are loaded again
@pytest.mark.parametrize("mean", [1000.0, -2000.0])
@pytest.mark.parametrize("m,n", [(8, 520), (1300, 1024), (8, 2880), (600, 2880), (8, 4096), (600, 4096), (4100, 6152), (600, 7168),
                                 (600, 12288), (8, 20000), (600, 20000)])
def test_gradient_of_rows_of_a_large_mean(pkg, mean, m, n):
    """A gradient along the normalised row, of which grad_x takes nearly all away again. h - mean is exact to its own last
    bit whatever the mean, so each of grad_x's terms is off by a few 2^-24 and the sums by F of their own magnitudes."""
    g = _gen(n)
    h = (mean + torch.randn(m, n, device=DEV, generator=g)).to(FP)
    w = torch.ones(n, device=DEV)
    o = pkg.layer_norm(h, w)
    d, r = h.double() - o.mean.double()[:, None], o.rstd.double()[:, None]
    gy = (d * r + 0.01 * torch.randn(m, n, device=DEV, generator=g)).to(FP)
    gx, gw, gb = pkg.layer_norm_backward(gy, h, w, o.mean, o.rstd)
    v = gy.double()
    want = r * (v - v.mean(1, keepdim=True)) - d * r**3 * (v * d).mean(1, keepdim=True)
    size = r * (v.abs() + v.abs().mean(1, keepdim=True)) + d.abs() * r**3 * (v * d).abs().mean(1, keepdim=True)
    assert bool(((gx.double() - want).abs() <= HALF[FP] * (want.abs() + F * size) + F * size + TINY[FP]).all())
    for got, t in ((gw, v * d * r), (gb, v)):
        off = F * t.abs().sum(0)
        assert bool(((got.double() - t.sum(0)).abs() <= HALF[F32] * (t.sum(0).abs() + off) + off).all())
