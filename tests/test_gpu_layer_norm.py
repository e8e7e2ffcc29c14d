"""Layer norm with the residual's addition, its 8-bit outputs and its gradients against 64-bit references; RMS norm to int8.

Bounds (derived, not fitted): a float32 sum of the kernels is a chain of at most 64 terms per lane and a tree, so its
error is below 100 * 2^-24 < 1e-5 = F of the sum of magnitudes. So the mean is off by at most F mean|h|, which moves every
h - mean by as much; rstd by F of itself and the square of that shift; products and the bias's addition by a few 2^-24. A
stored bf16 / fp16 value is off by half a unit in the last place more, an int8 one by half a step of its row's scale.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
BF, FP, F32, E4, E5, I8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.float8_e5m2, torch.int8
HALF = {BF: 2.0**-8, FP: 2.0**-11, F32: 2.0**-24, E4: 2.0**-4, E5: 2.0**-3}
TINY = {BF: 2.0**-134, FP: 2.0**-25, F32: 2.0**-150, E4: 2.0**-10, E5: 2.0**-17}  # half the least subnormal
TOP = {E4: 448.0, E5: 57344.0, I8: 127.0}
F = 1e-5


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _data(m, n, dtype, seed, wdtype=None):
    g = _gen(seed)
    x = (torch.randn(m, n, device=DEV, generator=g) + 0.25).to(dtype)
    r = (3 * torch.randn(m, n, device=DEV, generator=g)).to(dtype)
    w = (1 + 0.3 * torch.randn(n, device=DEV, generator=g)).to(wdtype or dtype)
    b = (0.5 * torch.randn(n, device=DEV, generator=g)).to(wdtype or dtype)
    return x, r, w, b


def _reference(x, r, w, b, eps):
    """h, mean, rstd, y and how far float32 may be off in mean, rstd and y."""
    h = x if r is None else (x.double() + r.double()).to(x.dtype)
    d = h.double()
    mean = d.mean(1)
    shift = F * d.abs().mean(1)
    c = d - mean[:, None]
    rstd = (c.square().mean(1) + eps).rsqrt()
    scaled = c * rstd[:, None] * w.double()
    y = scaled if b is None else scaled + b.double()
    off_rstd = 2 * F * rstd + shift.square() * rstd**3
    off = scaled.abs() * (2 * F + (off_rstd / rstd)[:, None]) \
        + (shift * rstd)[:, None] * w.double().abs() + F * y.abs()
    return h, mean, rstd, y, shift, off_rstd, off


def _check(o, ref, dtype):
    h, mean, rstd, y, off_mean, off_rstd, off = ref
    assert torch.equal(o.h, h)
    assert bool(((o.mean.double() - mean).abs() <= off_mean).all())
    assert bool(((o.rstd.double() - rstd).abs() <= off_rstd).all())
    if dtype is not None:
        err = (o.y.double() - y).abs()
        assert bool((err <= HALF[dtype] * (y.abs() + off) + off + TINY[dtype]).all())


def _check_i8(q, scale, y, off):
    """Rows of int8 against float64 rows that float32 may have off by `off`."""
    assert q.dtype == I8 and scale.dtype == F32 and scale.shape == (y.shape[0],)
    s = y.abs().amax(1) / 127
    assert bool(((scale.double() - s).abs() <= off.amax(1) / 127 + 2.0**-23 * s).all())
    s = scale.double()[:, None]
    assert bool(((q.double() - y / s).abs() <= 0.5 + off / s + 2.0**-16).all())  # a quotient up to 127 is off by 2^-18
    assert int(q.min()) >= -127


SHAPES = [(1, 8), (3, 64), (5, 512), (7, 520), (4, 1024), (2, 1032), (9, 2048), (3, 2056), (6, 4096), (5, 7168), (2, 8200),
          (3, 14336), (2, 16384), (2, 16392), (1, 32768), (2100, 256), (1025, 1544), (520, 5128), (256, 4096), (257, 4096), (256, 6144),
          (300, 8192)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("residual,bias", [(True, True), (False, True), (True, False)])
def test_plain(pkg, dtype, m, n, residual, bias):
    x, r, w, b = _data(m, n, dtype, m * n)
    r, b = r if residual else None, b if bias else None
    o = pkg.layer_norm(x, w, b, r, 1e-5)
    assert o.scale is None and o.y.dtype == dtype and (residual or o.h is x)
    _check(o, _reference(x, r, w, b, 1e-5), dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,n", SHAPES)
def test_int8_rows(pkg, dtype, m, n):
    x, r, w, b = _data(m, n, dtype, m + n)
    o = pkg.layer_norm(x, w, b, r, 1e-5, I8, "row")
    ref = _reference(x, r, w, b, 1e-5)
    _check(o, ref, None)
    _check_i8(o.y, o.scale, ref[3], ref[6])
    # the RMS norm's, too
    o = pkg.rms_norm(x, w, r, 1e-6, I8, "row")
    d = o.h.double()
    rstd = (d.square().mean(1) + 1e-6).rsqrt()
    y = d * rstd[:, None] * w.double()
    assert bool(((o.rstd.double() - rstd).abs() <= F * rstd).all())
    _check_i8(o.y, o.scale, y, 2 * F * y.abs())


@pytest.mark.parametrize("out", [E4, E5])
@pytest.mark.parametrize("mode", ["tensor", "row", "given"])
@pytest.mark.parametrize("dtype,m,n", [(BF, 1, 8), (BF, 5, 512), (FP, 3, 1040), (BF, 33, 7168), (FP, 2500, 264), (BF, 2049, 2880),
                                       (FP, 2, 16400), (BF, 256, 2880), (FP, 40, 4096), (BF, 257, 4104), (FP, 30, 6144)])
def test_fp8(pkg, out, mode, dtype, m, n):
    x, r, w, b = _data(m, n, dtype, m + n)
    ref = _reference(x, r, w, b, 1e-5)
    y, off = ref[3], ref[6]
    given = torch.tensor([0.01], device=DEV) if mode == "given" else mode
    o = pkg.layer_norm(x, w, b, r, 1e-5, out, given)
    _check(o, ref, None)
    if mode != "given":
        s = (y.abs().amax(1) if mode == "row" else y.abs().amax().reshape(1)) / TOP[out]
        most = off.amax(1) if mode == "row" else off.amax().reshape(1)
        assert bool(((o.scale.double() - s).abs() <= most / TOP[out] + 2.0**-23 * s).all())
    s = (given if mode == "given" else o.scale).double().view(-1, 1)
    want = (y / s).clamp(-TOP[out], TOP[out])
    slack = off / s + 2.0**-23 * want.abs()
    assert o.y.dtype == out
    assert bool(((o.y.double() - want).abs() <= HALF[out] * (want.abs() + slack) + slack + TINY[out]).all())


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("dtype,m,n", [(BF, 700, 256), (FP, 900, 1032), (BF, 300, 5120), (FP, 65, 7168), (BF, 40, 32768)])
def test_int8_codes_are_those_of_a_division(pkg, norm, dtype, m, n):
    """Without a bias each step is one correctly rounded float32 operation: given mean, rstd and scale, the CPU gives the same."""
    x, _, w, _ = _data(m, n, dtype, m + n, F32)
    if norm == "layer":
        o = pkg.layer_norm(x, w, None, None, 1e-5, I8, "row")
        v = (x.cpu().float() - o.mean.cpu()[:, None]) * o.rstd.cpu()[:, None] * w.cpu()
    else:
        o = pkg.rms_norm(x, w, None, 1e-6, I8, "row")
        v = x.cpu().float() * o.rstd.cpu()[:, None] * w.cpu()
    assert torch.equal(o.scale.cpu(), v.abs().amax(1) / 127)
    assert torch.equal(o.y.cpu(), (v / o.scale.cpu()[:, None]).round().to(I8))


def test_rows_of_a_large_mean(pkg):
    """Squares about the mean: a mean 1000 times the spread costs the variance nothing but the mean's own error."""
    g = _gen(3)
    x = (1000 + torch.randn(40, 4096, device=DEV, generator=g)).to(FP)
    w, b = torch.ones(4096, device=DEV), torch.zeros(4096, device=DEV)
    o = pkg.layer_norm(x, w, b)
    _check(o, _reference(x, None, w, b, 1e-5), FP)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_float32_weight_and_strides(pkg, dtype):
    m, n = 37, 1536
    x, r, w, b = _data(m, n, dtype, 5, F32)
    wide_x, wide_r = torch.empty(m, n + 24, device=DEV, dtype=dtype), torch.empty(m, 2 * n, device=DEV, dtype=dtype)
    wide_x[:, 8:n + 8], wide_r[:, :n] = x, r
    ref = _reference(x, r, w, b, 1e-5)
    o = pkg.layer_norm(wide_x[:, 8:n + 8], w, b, wide_r[:, :n])
    _check(o, ref, dtype)
    # in place: h over the residual, which a tensor scale's second pass reads again
    t = pkg.layer_norm(x, w, b, r, out_dtype=E4)
    o2 = pkg.layer_norm(wide_x[:, 8:n + 8], w, b, wide_r[:, :n], out_dtype=E4, out_h=wide_r[:, :n])
    assert o2.h.data_ptr() == wide_r.data_ptr() and torch.equal(wide_r[:, :n], ref[0])
    assert torch.equal(o2.y.view(torch.uint8), t.y.view(torch.uint8)) and torch.equal(o2.scale, t.scale)
    # one row for all: a stride of zero
    same = x[:1].expand(m, n)
    o3 = pkg.layer_norm(same, w, b)
    assert bool((o3.y == o3.y[:1]).all()) and torch.equal(o3.y[0], pkg.layer_norm(x[:1], w, b).y[0])
    out = torch.empty(m, n, device=DEV, dtype=dtype)
    assert pkg.layer_norm(x, w, b, r, out=out).y is out


def test_constant_nan_and_infinite_rows(pkg):
    m, n = 7, 1024
    x, _, w, b = _data(m, n, BF, 9)
    x[1] = 0
    x[2] = 3.0
    x[4, 5] = float("nan")
    x[5, 7] = float("inf")
    o = pkg.layer_norm(x, w, b, None, 1e-5, I8, "row")
    # a constant row is its bias
    want = pkg.layer_norm(torch.zeros(1, n, device=DEV, dtype=BF), w, b, None, 1e-5, I8, "row")
    assert torch.equal(o.y[1], want.y[0]) and torch.equal(o.y[2], want.y[0]) and float(o.scale[2]) == float(want.scale)
    assert bool(o.scale[4].isnan()) and bool(o.scale[5].isnan()) and bool((o.y[4:6] == 0).all())
    clean = [0, 1, 2, 3, 6]
    ref = pkg.layer_norm(x[clean], w, b, None, 1e-5, I8, "row")
    assert torch.equal(o.y[clean], ref.y) and torch.equal(o.scale[clean], ref.scale)
    z = pkg.layer_norm(x[:2] * 0, w, None, None, 1e-5, I8, "row")
    assert bool((z.y == 0).all()) and bool((z.scale == 1).all())
    q = pkg.rms_norm(x, w, None, 1e-6, I8, "row")
    assert bool((q.y[1] == 0).all()) and float(q.scale[1]) == 1.0 and bool(q.scale[4].isnan()) and bool((q.y[4] == 0).all())
    assert bool(q.scale[5].isnan()) or bool(q.scale[5].isinf())


def test_no_rows(pkg):
    x = torch.empty(0, 64, device=DEV, dtype=BF)
    w = torch.ones(64, device=DEV, dtype=BF)
    for out, scale in ((None, None), (I8, "row"), (E4, "row")):
        o = pkg.layer_norm(x, w, w, x, out_dtype=out, scale=scale)
        assert o.y.shape == (0, 64) and o.mean.shape == (0,)
    assert float(pkg.layer_norm(x, w, w, out_dtype=E4).scale) == 1.0
    none = torch.empty(0, device=DEV)
    gx, gw, gb = pkg.layer_norm_backward(x, x, w, none, none)
    assert gx.shape == (0, 64) and bool((gw == 0).all()) and bool((gb == 0).all())


# ---- backward ----


def _back_reference(gy, h, w, mean, rstd, gh):
    g, r, ww = gy.double(), rstd.double()[:, None], w.double()
    d = h.double() - mean.double()[:, None]
    n = h.shape[1]
    wg = g * ww
    gx = r * (wg - wg.sum(1, keepdim=True) / n) - d * r**3 * (wg * d).sum(1, keepdim=True) / n
    # magnitudes of the float32 terms; h - mean is rounded once, relative to itself
    size = r * (wg.abs() + wg.abs().sum(1, keepdim=True) / n) + d.abs() * r**3 * (wg * d).abs().sum(1, keepdim=True) / n
    if gh is not None:
        gx, size = gx + gh.double(), size + gh.double().abs()
    t = g * d * r
    return gx, size, t.sum(0), t.abs().sum(0), g.sum(0), g.abs().sum(0)


def _check_back(got, ref, dtype, wdtype):
    gx, size, gw, size_w, gb, size_b = ref
    assert bool(((got[0].double() - gx).abs() <= HALF[dtype] * (gx.abs() + F * size) + F * size + TINY[dtype]).all())
    for a, want, s in ((got[1], gw, size_w), (got[2], gb, size_b)):
        assert a.dtype == wdtype
        assert bool(((a.double() - want).abs() <= HALF[wdtype] * (want.abs() + F * s) + F * s + TINY[wdtype]).all())


# either side of the numbers of rows that choose how many waves take a row and how the sums are added; every instance's width
BACK = SHAPES + [(256, 1544), (257, 1544), (512, 7168), (513, 7168), (300, 1024), (1300, 2048), (1100, 4096), (800, 6144),
                 (800, 8192), (600, 12288), (600, 16384), (520, 32768), (1281, 512)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,n", BACK)
@pytest.mark.parametrize("grad_h,w32", [(True, False), (False, True)])
def test_backward(pkg, dtype, m, n, grad_h, w32):
    wdtype = F32 if w32 else dtype
    x, r, w, b = _data(m, n, dtype, m + 3 * n, wdtype)
    g = _gen(n)
    gy = torch.randn(m, n, device=DEV, generator=g).to(dtype)
    gh = torch.randn(m, n, device=DEV, generator=g).to(dtype) if grad_h else None
    o = pkg.layer_norm(x, w, b, r)
    got = pkg.layer_norm_backward(gy, o.h, w, o.mean, o.rstd, gh)
    _check_back(got, _back_reference(gy, o.h, w, o.mean, o.rstd, gh), dtype, wdtype)
    again = pkg.layer_norm_backward(gy, o.h, w, o.mean, o.rstd, gh)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.parametrize("m,n", [(601, 1536), (602, 2880), (2047, 2056), (2050, 2880), (599, 6144), (1027, 8192), (4097, 7168), (4096, 6152),
                                 (4099, 1032), (3100, 4104)])
def test_backward_with_a_last_workgroup_that_is_not_full(pkg, m, n):
    """Workgroups have two or three rows at a time: those that are not there change nothing, in place as well."""
    x, r, w, b = _data(m, n, BF, m + n, F32)
    g = _gen(m)
    gy, gh = (torch.randn(m, n, device=DEV, generator=g).to(BF) for _ in range(2))
    o = pkg.layer_norm(x, w, b, r)
    whole = torch.full((m + 3, n), 7.0, device=DEV, dtype=BF)
    got = pkg.layer_norm_backward(gy, o.h, w, o.mean, o.rstd, gh, out=whole[:m])
    _check_back(got, _back_reference(gy, o.h, w, o.mean, o.rstd, gh), BF, F32)
    assert bool((whole[m:] == 7).all())
    own = o.h.clone()
    again = pkg.layer_norm_backward(gy, own, w, o.mean, o.rstd, gh, out=own)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.parametrize("m,n", [(5, 1544), (700, 1544), (600, 20000), (530, 12296)])
@pytest.mark.parametrize("place", ["grad_y", "h", "grad_h"])
def test_backward_strides_and_in_place(pkg, m, n, place):
    x, r, w, b = _data(m, n, BF, 11)
    g = _gen(12)
    t = {"grad_y": torch.randn(m, n, device=DEV, generator=g).to(BF), "grad_h": torch.randn(m, n, device=DEV, generator=g).to(BF)}
    o = pkg.layer_norm(x, w, b, r)
    t["h"] = o.h
    want = pkg.layer_norm_backward(t["grad_y"], t["h"], w, o.mean, o.rstd, t["grad_h"])
    wide = {}
    for k, v in t.items():
        wide[k] = torch.zeros(m, n + 40, device=DEV, dtype=BF)
        wide[k][:, 16:n + 16] = v
    got = pkg.layer_norm_backward(*(wide[k][:, 16:n + 16] for k in ("grad_y", "h")), w, o.mean, o.rstd, wide["grad_h"][:, 16:n + 16])
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    c = {k: v.clone() for k, v in t.items()}
    got = pkg.layer_norm_backward(c["grad_y"], c["h"], w, o.mean, o.rstd, c["grad_h"], out=c[place])
    assert got[0] is c[place] and all(torch.equal(a, b2) for a, b2 in zip(got, want))


@pytest.mark.parametrize("power", [-50, 50])
@pytest.mark.parametrize("m,n", [(5, 512), (5, 2880), (300, 1024), (300, 7168)])
def test_backward_of_large_and_small_rows(pkg, power, m, n):
    """rstd of 2^50 and 2^-50: its cube is past float32's range, the gradients are not."""
    g = _gen(n)
    h = (torch.randn(m, n, device=DEV, generator=g) * 2.0**power).to(BF)
    w = (1 + 0.3 * torch.randn(n, device=DEV, generator=g)).to(BF)
    gy = torch.randn(m, n, device=DEV, generator=g).to(BF)
    o = pkg.layer_norm(h, w, None, None, 0.0)
    got = pkg.layer_norm_backward(gy, h, w, o.mean, o.rstd)
    _check_back(got, _back_reference(gy, h, w, o.mean, o.rstd, None), BF, BF)


def test_gradients_against_differences(pkg):
    """The derivative of sum(y * grad_y) along random directions, by differences of the float64 definition (whose own error
    at this step is below 1e-7 of the terms), against the gradients' products; those are rounded to fp16 value by value."""
    m, n = 6, 520
    x, _, w, b = _data(m, n, FP, 21)
    g = _gen(22)
    gy = torch.randn(m, n, device=DEV, generator=g).to(FP)
    o = pkg.layer_norm(x, w, b)
    grads = pkg.layer_norm_backward(gy, x, w, o.mean, o.rstd)

    def f(x, w, b):
        c = x - x.mean(1, keepdim=True)
        return ((c * (c.square().mean(1, keepdim=True) + 1e-5).rsqrt() * w + b) * gy.double()).sum()

    at = [v.double() for v in (x, w, b)]
    for i, grad in enumerate(grads):
        v = torch.randn(at[i].shape, device=DEV, generator=g, dtype=torch.float64)
        step = 1e-5
        hi, lo = [list(at), list(at)]
        hi[i], lo[i] = at[i] + step * v, at[i] - step * v
        d = float((f(*hi) - f(*lo)) / (2 * step))
        bound = float((v.abs() * (HALF[FP] * grad.double().abs() + F * (gy.double().abs().sum() / gy.numel()) * 8)).sum())
        assert abs(float((grad.double() * v).sum()) - d) <= bound + 1e-6 * abs(d), i


# ---- capture ----


@pytest.mark.parametrize("m,n", [(9, 2048), (700, 1544)])
def test_captured_forward_and_backward(pkg, m, n):
    """Replays of a captured pass give the eager call's bits on what the inputs hold at the time."""
    x, r, w, b = _data(m, n, BF, 31)
    gy = torch.randn(m, n, device=DEV, generator=_gen(32)).to(BF)

    def step():
        o = pkg.layer_norm(x, w, b, r)
        q = pkg.layer_norm(x, w, b, r, 1e-5, I8, "row")
        return (*o[:4], q.y, q.scale, *pkg.layer_norm_backward(gy, o.h, w, o.mean, o.rstd, gy))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        x.copy_(torch.randn(m, n, device=DEV, generator=_gen(40 + i)).to(BF))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, want)), i


def test_more_rows_than_32_bits_of_bytes(pkg):
    """Offsets past 2^32: the last rows are those of a call of as many as take the same kernels."""
    m, n, k = 140000, 16384, 600
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB")
    g = torch.Generator(device=DEV).manual_seed(6)
    h, gy = torch.zeros(m, n, device=DEV, dtype=BF), torch.zeros(m, n, device=DEV, dtype=BF)
    for t in (h, gy):
        t[-k:] = torch.randn(k, n, device=DEV, generator=g).to(BF)
    w, b = torch.randn(2, n, device=DEV, generator=g).to(BF)
    o, last = pkg.layer_norm(h, w, b), pkg.layer_norm(h[-k:], w, b)
    assert all(torch.equal(o[i][-k:], last[i]) for i in (0, 2, 3))
    gx, gx_last = (pkg.layer_norm_backward(gy[i:], h[i:], w, o.mean[i:], o.rstd[i:])[0] for i in (0, m - k))
    assert torch.equal(gx[-k:], gx_last)
    del gx
    q, last = pkg.layer_norm(h, w, b, out_dtype=torch.int8, scale="row"), pkg.layer_norm(h[-k:], w, b, out_dtype=torch.int8, scale="row")
    assert torch.equal(q.y[-k:], last.y) and torch.equal(q.scale[-k:], last.scale)
