"""RMS norm with the residual's addition and its gradients against 64-bit references.

Bounds (derived, not fitted): a float32 sum of the kernels is a chain of at most 64 terms per lane and a tree,
so its relative error (over the sum of magnitudes) is below 100 * 2^-24 < 1e-5 = F; a stored bf16 / fp16 value is
off by half a unit in the last place, up to 2^-8 / 2^-11 of it, an e4m3 / e5m2 value by 2^-4 / 2^-3 of it or half the
smallest subnormal.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
BF, FP, E4, E5 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float8_e5m2
HALF = {BF: 2.0**-8, FP: 2.0**-11, E4: 2.0**-4, E5: 2.0**-3, torch.float32: 2.0**-24}
TINY = {BF: 2.0**-134, FP: 2.0**-25, E4: 2.0**-10, E5: 2.0**-17, torch.float32: 2.0**-150}  # half the least subnormal
TOP = {E4: 448.0, E5: 57344.0}
F = 1e-5


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _data(m, n, dtype, seed, residual=True, wdtype=None):
    g = _gen(seed)
    x = torch.randn(m, n, device=DEV, generator=g).to(dtype)
    r = (3 * torch.randn(m, n, device=DEV, generator=g)).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(n, device=DEV, generator=g)).to(wdtype or dtype)
    return x, r, w


def _reference(x, r, w, eps):
    h = x if r is None else (x.double() + r.double()).to(x.dtype)
    d = h.double()
    rstd = (d.square().mean(1) + eps).rsqrt()
    return h, rstd, d * rstd[:, None] * w.double()


def _near(got, want, dtype, rel=F):
    err = (got.double() - want).abs()
    bound = want.abs() * (HALF[dtype] * (1 + rel) + rel) + TINY[dtype]
    assert bool((err <= bound).all()), float((err - bound).max())


SHAPES = [(1, 8), (3, 64), (5, 512), (7, 520), (4, 1024), (2, 1032), (9, 2048), (3, 2056), (6, 4096), (5, 7168), (2, 8200),
          (3, 14336), (2, 16384), (2, 16392), (1, 32768), (2100, 256), (1025, 1544)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("residual", [True, False])
def test_plain(pkg, dtype, m, n, residual):
    x, r, w = _data(m, n, dtype, m * n)
    o = pkg.rms_norm(x, w, r if residual else None, 1e-5)
    h, rstd, y = _reference(x, r if residual else None, w, 1e-5)
    assert torch.equal(o.h, h) and (residual or o.h is x) and o.scale is None
    assert o.y.dtype == dtype and bool(((o.rstd.double() - rstd).abs() <= F * rstd).all())
    _near(o.y, y, dtype)


@pytest.mark.parametrize("out", [E4, E5])
@pytest.mark.parametrize("mode", ["tensor", "row", "given"])
@pytest.mark.parametrize("dtype,m,n", [(BF, 1, 8), (BF, 5, 512), (FP, 3, 1040), (BF, 33, 7168), (FP, 2500, 264), (BF, 2049, 2880),
                                       (FP, 2, 16400)])
def test_fp8(pkg, out, mode, dtype, m, n):
    x, r, w = _data(m, n, dtype, m + n)
    h, rstd, y = _reference(x, r, w, 1e-6)
    given = torch.tensor([0.01], device=DEV) if mode == "given" else mode  # most values saturate at neither end
    o = pkg.rms_norm(x, w, r, out_dtype=out, scale=given)
    assert torch.equal(o.h, h) and o.y.dtype == out
    if mode == "given":
        s = given.double()
    else:
        s = (y.abs().amax(1) if mode == "row" else y.abs().amax().reshape(1)) / TOP[out]
        assert o.scale.shape == ((m,) if mode == "row" else (1,))
        assert bool(((o.scale.double() - s).abs() <= 2 * F * s).all())
    want = (y / (s[:, None] if mode == "row" else s)).clamp(-TOP[out], TOP[out])
    _near(o.y.float(), want, out, rel=4 * F)


@pytest.mark.parametrize("out", [E4, E5])
def test_fp8_rounding_is_to_nearest_even(pkg, out):
    """Halfway values: weight 1, rows whose rstd is exactly 1 and whose values are ties of the format."""
    n = 64
    ties = torch.arange(1, n + 1, device=DEV, dtype=torch.float32) / 8 + 1 / 32  # 3 bits and a half: e4m3 ties above 1
    x = torch.cat([ties, -ties]).to(BF).reshape(1, -1)
    w = torch.ones(2 * n, device=DEV, dtype=BF)
    o = pkg.rms_norm(x, w, None, 0.0, out_dtype=out, scale=torch.ones(1, device=DEV))
    want = (x.float() * o.rstd).clamp(-TOP[out], TOP[out]).to(out)
    assert torch.equal(o.y.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_float32_weight_and_strides(pkg, dtype):
    m, n = 37, 1536
    x, r, w = _data(m, n, dtype, 5, wdtype=torch.float32)
    wide_x, wide_r = torch.empty(m, n + 24, device=DEV, dtype=dtype), torch.empty(m, 2 * n, device=DEV, dtype=dtype)
    wide_x[:, 8:n + 8], wide_r[:, :n] = x, r
    h, rstd, y = _reference(x, r, w, 1e-6)
    o = pkg.rms_norm(wide_x[:, 8:n + 8], w, wide_r[:, :n])
    assert torch.equal(o.h, h)
    _near(o.y, y, dtype)
    # in place: h over the residual
    o2 = pkg.rms_norm(wide_x[:, 8:n + 8], w, wide_r[:, :n], out_h=wide_r[:, :n])
    assert o2.h.data_ptr() == wide_r.data_ptr() and torch.equal(wide_r[:, :n], h) and torch.equal(o2.y, o.y)
    # and over x, for a tensor scale, whose second pass reads h
    want = pkg.rms_norm(x, w, r, out_dtype=E4)
    xc = x.clone()
    o3 = pkg.rms_norm(xc, w, r, out_dtype=E4, out_h=xc)
    assert torch.equal(xc, h) and torch.equal(o3.y.view(torch.uint8), want.y.view(torch.uint8)) and torch.equal(o3.scale, want.scale)


def test_zeros_nan_and_infinity(pkg):
    m, n = 6, 1024
    x, _, w = _data(m, n, BF, 9)
    x[1] = 0
    x[3, 5] = float("nan")
    x[4, 7] = float("inf")
    o = pkg.rms_norm(x, w, out_dtype=E4, scale="row")
    q = o.y.float()
    assert bool((q[1] == 0).all()) and float(o.scale[1]) == 1.0
    assert bool(q[3].isnan().all()) and bool(q[4].isnan().any()) and bool(o.scale[3].isnan())
    clean = [0, 2, 5]
    ref = pkg.rms_norm(x[clean], w, out_dtype=E4, scale="row")
    assert torch.equal(q[clean], ref.y.float()) and torch.equal(o.scale[clean], ref.scale)
    t = pkg.rms_norm(x, w, out_dtype=E4)
    assert bool(t.scale.isnan()) and bool(t.y.float().isnan().all())
    z = pkg.rms_norm(torch.zeros_like(x), w, out_dtype=E5)
    assert float(z.scale) == 1.0 and bool((z.y.float() == 0).all())


def test_no_rows(pkg):
    x = torch.empty(0, 64, device=DEV, dtype=BF)
    w = torch.ones(64, device=DEV, dtype=BF)
    assert pkg.rms_norm(x, w).y.shape == (0, 64)
    assert float(pkg.rms_norm(x, w, x, out_dtype=E4).scale) == 1.0
    gx, gw = pkg.rms_norm_backward(x, x, w, torch.empty(0, device=DEV))
    assert gx.shape == (0, 64) and bool((gw == 0).all())


def _backward_reference(gy, h, w, rstd, gh):
    g, d, r, ww = gy.double(), h.double(), rstd.double()[:, None], w.double()
    n = h.shape[1]
    wg = g * ww
    dot = (wg * d).sum(1, keepdim=True) / n
    gx = r * wg - d * r**3 * dot
    size = (r * wg).abs() + d.abs() * r**3 * (wg * d).abs().sum(1, keepdim=True) / n  # of the float32 terms
    if gh is not None:
        gx, size = gx + gh.double(), size + gh.double().abs()
    return gx, size, (g * d * r).sum(0), (g * d * r).abs().sum(0)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("grad_h", [True, False])
def test_backward(pkg, dtype, m, n, grad_h):
    x, r, w = _data(m, n, dtype, m + 3 * n)
    g = _gen(n)
    gy = torch.randn(m, n, device=DEV, generator=g).to(dtype)
    gh = torch.randn(m, n, device=DEV, generator=g).to(dtype) if grad_h else None
    o = pkg.rms_norm(x, w, r)
    gx, gw = pkg.rms_norm_backward(gy, o.h, w, o.rstd, gh)
    want, size, want_w, size_w = _backward_reference(gy, o.h, w, o.rstd, gh)
    assert bool(((gx.double() - want).abs() <= HALF[dtype] * want.abs() + F * size + TINY[dtype]).all())
    assert gw.dtype == dtype
    assert bool(((gw.double() - want_w).abs() <= HALF[dtype] * want_w.abs() + F * size_w + TINY[dtype]).all())
    again = pkg.rms_norm_backward(gy, o.h, w, o.rstd, gh)
    assert torch.equal(gx, again[0]) and torch.equal(gw, again[1])


# Either side of the numbers of rows that choose how many waves take a row and how grad_weight is summed; every width of the
# instances for many rows.
@pytest.mark.parametrize("m,n", [(256, 1032), (257, 1032), (256, 2048), (256, 2056), (257, 2056), (257, 4104), (256, 5120), (512, 5128),
                                 (513, 7168), (512, 8192), (513, 8200), (513, 14336), (512, 16384), (513, 20000)])
def test_sizes_that_choose(pkg, m, n):
    x, r, w = _data(m, n, BF, m + n)
    o = pkg.rms_norm(x, w, r)
    h, rstd, y = _reference(x, r, w, 1e-6)
    assert torch.equal(o.h, h) and bool(((o.rstd.double() - rstd).abs() <= F * rstd).all())
    _near(o.y, y, BF)
    for scale in ("tensor", "row"):
        q = pkg.rms_norm(x, w, r, out_dtype=E4, scale=scale)
        top = y.abs().amax() if scale == "tensor" else y.abs().amax(1)
        assert torch.equal(q.h, h) and bool(((q.scale.double() - top / 448).abs() <= 2 * F * top / 448).all())
        back = q.y.double() * q.scale.double().view(-1, 1)
        # half a unit of e4m3's last place, 2^-4 of a value, and of its smallest one, 2^-10 of the scale
        assert bool(((back - y).abs() <= 2.0**-4 * (1 + 8 * F) * y.abs() + 2.0**-10 * (1 + F) * q.scale.double().view(-1, 1)).all())
    g = _gen(m)
    gy, gh = (torch.randn(m, n, device=DEV, generator=g).to(BF) for _ in range(2))
    gx, gw = pkg.rms_norm_backward(gy, o.h, w, o.rstd, gh)
    want, size, want_w, size_w = _backward_reference(gy, o.h, w, o.rstd, gh)
    assert bool(((gx.double() - want).abs() <= HALF[BF] * want.abs() + F * size + TINY[BF]).all())
    assert bool(((gw.double() - want_w).abs() <= HALF[BF] * want_w.abs() + F * size_w + TINY[BF]).all())
    # grad_x in the place of an input
    for i in range(3):
        a = [gy.clone(), o.h.clone(), gh.clone()]
        gx2, gw2 = pkg.rms_norm_backward(a[0], a[1], w, o.rstd, a[2], out=a[i])
        assert gx2 is a[i] and torch.equal(gx2, gx) and torch.equal(gw2, gw)


def test_backward_float32_weight_and_strides(pkg):
    m, n = 300, 2880
    x, r, w = _data(m, n, BF, 11, wdtype=torch.float32)
    wide = torch.randn(m, 2 * n + 16, device=DEV, generator=_gen(4)).to(BF)
    gy, gh = wide[:, :n], wide[:, n + 8:2 * n + 8]
    o = pkg.rms_norm(x, w, r)
    gx, gw = pkg.rms_norm_backward(gy, o.h, w, o.rstd, gh)
    want, size, want_w, size_w = _backward_reference(gy, o.h, w, o.rstd, gh)
    assert bool(((gx.double() - want).abs() <= HALF[BF] * want.abs() + F * size + TINY[BF]).all())
    assert gw.dtype == torch.float32 and bool(((gw.double() - want_w).abs() <= F * size_w).all())


def test_backward_against_differences(pkg):
    """<gradient, direction> against a central difference of the 64-bit loss sum(gy * y) along the direction."""
    m, n, eps = 5, 520, 1e-5
    x, r, w = _data(m, n, FP, 21)
    g = _gen(22)
    gy = torch.randn(m, n, device=DEV, generator=g).to(FP)
    o = pkg.rms_norm(x, w, r, eps)
    gx, gw = pkg.rms_norm_backward(gy, o.h, w, o.rstd)

    def loss(h, ww):
        return (gy.double() * h * (h.square().mean(1, keepdim=True) + eps).rsqrt() * ww).sum()

    h, ww, step = o.h.double(), w.double(), 1e-5
    for d, grad, move in ((torch.randn(m, n, device=DEV, generator=g).double(), gx, lambda d, t: loss(h + t * d, ww)),
                          (torch.randn(n, device=DEV, generator=g).double(), gw, lambda d, t: loss(h, ww + t * d))):
        numeric = float((move(d, step) - move(d, -step)) / (2 * step))
        exact = float((grad.double() * d).sum())
        # half a unit of each gradient value, float32 sums, and the difference's own error (step^2 and 1e-16 / step)
        bound = float((grad.double() * d).abs().sum()) * (HALF[FP] + F) + float(d.abs().sum()) * 1e-5
        assert abs(numeric - exact) <= bound, (numeric, exact, bound)


def test_other_stream_and_graph(pkg):
    x, r, w = _data(64, 2048, BF, 31)
    want = pkg.rms_norm(x, w, r, out_dtype=E4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = pkg.rms_norm(x, w, r, out_dtype=E4, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got.y.view(torch.uint8), want.y.view(torch.uint8)) and torch.equal(got.scale, want.scale)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = pkg.rms_norm(x, w, r, out_dtype=E4)
        gx, gw = pkg.rms_norm_backward(r, o.h, w, o.rstd, x)
    for k in range(3):
        x.copy_(torch.randn(64, 2048, device=DEV, generator=_gen(40 + k)).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        e = pkg.rms_norm(x, w, r, out_dtype=E4)
        ex, ew = pkg.rms_norm_backward(r, e.h, w, e.rstd, x)
        assert torch.equal(o.y.view(torch.uint8), e.y.view(torch.uint8)) and torch.equal(o.scale, e.scale)
        assert torch.equal(gx, ex) and torch.equal(gw, ew)


def test_torch_level_refusals(pkg):
    x, r, w = _data(4, 64, BF, 1)
    for bad, err in ((dict(residual=r.float()), ValueError), (dict(out_dtype=torch.float32), TypeError),
                     (dict(scale="row"), ValueError), (dict(out_dtype=E4, scale="column"), ValueError),
                     (dict(out_dtype=E4, scale=torch.ones(2, device=DEV)), ValueError),
                     (dict(out_h=torch.empty_like(x)), ValueError), (dict(out=torch.empty_like(x).t()), ValueError)):
        with pytest.raises(err):
            pkg.rms_norm(x, w, **bad)
    with pytest.raises(ValueError):
        pkg.rms_norm(x.t(), w[:4])
    with pytest.raises(pkg.GGError, match="multiple of 8"):
        pkg.rms_norm(x[:, :60], w[:60].clone())
    with pytest.raises(ValueError):
        pkg.rms_norm_backward(x[:2], x, w, torch.ones(4, device=DEV))
