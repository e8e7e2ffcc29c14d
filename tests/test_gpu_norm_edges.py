"""RMS norm where it is easily off: the division by a scale, bit for bit; no rows; rows of very large and small values.

The kernels take y = (h * rstd) * weight in float32, divide it by the scale as float32 division rounds it, clamp and
round to the format. Given rstd and the scale that a call returned, the same steps on the CPU give the same codes:
each is one correctly rounded operation, so there is no tolerance.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
BF, FP, E4, E5 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float8_e5m2
TOP = {E4: 448.0, E5: 57344.0}


def _data(m, n, dtype, seed, wdtype=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(m, n, device=DEV, generator=g).to(dtype)
    x[:, 3] = -0.0
    w = (1 + 0.3 * torch.randn(n, device=DEV, generator=g)).to(wdtype or dtype)
    return x, w


def _codes(o, w, scale, out):
    y = (o.h.cpu().float() * o.rstd.cpu()[:, None]) * w.cpu().float()
    q = (y / scale.cpu().view(-1, 1)).clamp(-TOP[out], TOP[out])
    return q.to(out).view(torch.uint8), q.isnan()


def _same(o, w, scale, out):
    want, nan = _codes(o, w, scale, out)
    got = o.y.cpu()
    assert torch.equal(got.float().isnan(), nan)
    differ = (got.view(torch.uint8) != want) & ~nan
    assert not bool(differ.any()), int(differ.sum())


@pytest.mark.parametrize("out", [E4, E5])
@pytest.mark.parametrize("mode", ["tensor", "row"])
@pytest.mark.parametrize("dtype,m,n", [(BF, 700, 256), (FP, 900, 1032), (BF, 300, 5120), (FP, 65, 7168), (BF, 40, 32768)])
def test_codes_are_those_of_a_division(pkg, out, mode, dtype, m, n):
    x, w = _data(m, n, dtype, m + n)
    o = pkg.rms_norm(x, w, out_dtype=out, scale=mode)
    _same(o, w, o.scale, out)


# A third and its like make quotients that are ties; the ends of the range, where a reciprocal is infinite, zero or cut.
@pytest.mark.parametrize("out", [E4, E5])
@pytest.mark.parametrize("scale", [3.0, 0.3, 7.0 / 448, 2.0**-64, 2.0**-65, 2.0**64, 2.0**65, 1e-38, 1e-39, 1e-45, 3e38, 0.0,
                                   float("inf"), float("nan"), -0.75])
def test_given_scales(pkg, out, scale):
    x, w = _data(130, 1536, BF, 7, torch.float32)
    s = torch.tensor([scale], device=DEV)
    o = pkg.rms_norm(x, w, out_dtype=out, scale=s)
    _same(o, w, s, out)


@pytest.mark.parametrize("out", [E4, E5])
def test_no_rows_with_any_scale(pkg, out):
    x, w = torch.empty(0, 64, device=DEV, dtype=BF), torch.ones(64, device=DEV, dtype=BF)
    given = torch.full((1,), 0.5, device=DEV)
    for residual in (None, x):
        o = pkg.rms_norm(x, w, residual, out_dtype=out, scale="row")
        assert o.y.shape == (0, 64) and o.y.dtype == out and o.scale.shape == (0,) and o.rstd.shape == (0,)
        o = pkg.rms_norm(x, w, residual, out_dtype=out, scale=given)
        assert o.y.shape == (0, 64) and o.scale is given and float(given) == 0.5
        assert float(pkg.rms_norm(x, w, residual, out_dtype=out).scale) == 1.0


# rstd of 2^50 and 2^-50: its cube is past float32's range, the gradients are not.
@pytest.mark.parametrize("power", [-50, 50])
@pytest.mark.parametrize("m,n", [(5, 512), (5, 2880), (300, 1024), (300, 7168)])
def test_backward_of_large_and_small_rows(pkg, power, m, n):
    """Bounds as in the ordinary cases: float32 sums and products below 1e-5 of the terms' magnitudes, and half a unit
    of bf16 in the stored value (2^-8 of it, or half the least subnormal)."""
    g = torch.Generator(device=DEV).manual_seed(n)
    h = (torch.randn(m, n, device=DEV, generator=g) * 2.0**power).to(BF)
    w = (1 + 0.3 * torch.randn(n, device=DEV, generator=g)).to(BF)
    gy = torch.randn(m, n, device=DEV, generator=g).to(BF)
    o = pkg.rms_norm(h, w, None, 0.0)
    gx, gw = pkg.rms_norm_backward(gy, h, w, o.rstd)
    d, r, wg = h.double(), o.rstd.double()[:, None], gy.double() * w.double()
    dot = (wg * d).sum(1, keepdim=True) / n
    want = r * wg - d * r**3 * dot
    size = (r * wg).abs() + d.abs() * r**3 * (wg * d).abs().sum(1, keepdim=True) / n
    assert bool(((gx.double() - want).abs() <= 2.0**-8 * want.abs() + 1e-5 * size + 2.0**-134).all())
    terms = gy.double() * d * r
    assert bool(((gw.double() - terms.sum(0)).abs() <= 2.0**-8 * terms.sum(0).abs() + 1e-5 * terms.abs().sum(0) + 2.0**-134).all())
