"""The gated activation and its gradient, and rows of int8, against 64-bit references.

Bounds (derived, not fitted), with e = 2^-23 and v a gate: exp(-v) in float32 comes from 2^(-v log2 e), whose argument's
rounding moves the result by |v| e and whose instruction by e; the sum, the quotient and the products add half an e each,
so silu(v) u is off by (8 + 2 |v|) e of itself. Where exp(-v) is past float32 (v < -88) the result is 0, less than
|v u| 2^-126 off. The gradient of the gate has a factor 1 + v (1 - p) whose terms are 1 and v (1 - p), off by a few e each
and by |v| e for 1 - p near p = 1. A stored value is off by half a unit in the last place more, an int8 one by half a step.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
BF, FP, I8 = torch.bfloat16, torch.float16, torch.int8
HALF = {BF: 2.0**-8, FP: 2.0**-11}
TINY = {BF: 2.0**-134, FP: 2.0**-25}
E = 2.0**-23

SHAPES = [(1, 8), (3, 64), (5, 512), (7, 520), (4, 1024), (2, 1032), (9, 2048), (3, 2056), (6, 2880), (5, 7168), (2, 8200),
          (3, 14336), (2, 16392), (1, 32768), (2100, 256), (1025, 1544), (257, 1032), (513, 5128),
          (1290, 1544), (1300, 2048), (1030, 12288), (1026, 16400), (1024, 9000)]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _data(m, n, dtype, seed):
    g = _gen(seed)
    gu = 2 * torch.randn(m, 2 * n, device=DEV, generator=g)
    gu[:, 3] *= 12  # gates far out on either side
    return gu.to(dtype), torch.randn(m, n, device=DEV, generator=g).to(dtype)


def _product(gu):
    """silu(gate) * up in 64 bits and how far float32 may have it off."""
    v, u = gu.double().chunk(2, dim=1)
    y = v * torch.sigmoid(v) * u
    return y, (8 + 2 * v.abs()) * E * y.abs() + (v * u).abs() * 2.0**-126


def _check_i8(q, scale, y, off):
    s = y.abs().amax(1) / 127
    assert q.dtype == I8 and scale.shape == s.shape
    assert bool(((scale.double() - s).abs() <= off.amax(1) / 127 + E * s).all())
    s = scale.double()[:, None]
    assert bool(((q.double() - y / s).abs() <= 0.5 + off / s + 2.0**-16).all()) and int(q.min()) >= -127


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,n", SHAPES)
def test_silu_product(pkg, dtype, m, n):
    gu, _ = _data(m, n, dtype, m + n)
    y, off = _product(gu)
    o = pkg.silu_product(gu)
    assert o.scale is None and o.y.dtype == dtype
    assert bool(((o.y.double() - y).abs() <= HALF[dtype] * (y.abs() + off) + off + TINY[dtype]).all())
    q = pkg.silu_product(gu, I8)
    _check_i8(q.y, q.scale, y, off)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,n", SHAPES)
def test_silu_product_backward(pkg, dtype, m, n):
    gu, gy = _data(m, n, dtype, m + 2 * n)
    got = pkg.silu_product_backward(gy, gu).double()
    v, u = gu.double().chunk(2, dim=1)
    p, g = torch.sigmoid(v), gy.double()
    gate, up = g * u * p * (1 + v * (1 - p)), g * v * p
    rel = (8 + 2 * v.abs()) * E
    size = (g * u * p).abs()
    off_gate = size * ((1 + v.abs() * (1 - p)) * (rel + 4 * E) + 2 * v.abs() * E) + (g * u).abs() * (1 + v.abs()) * 2.0**-126
    off_up = up.abs() * rel + (g * v).abs() * 2.0**-126
    want, off = torch.cat([gate, up], 1), torch.cat([off_gate, off_up], 1)
    assert bool(((got - want).abs() <= HALF[dtype] * (want.abs() + off) + off + TINY[dtype]).all())


def test_gradient_against_differences(pkg):
    """A central difference of the 64-bit loss sum(gy * y) along a direction; half a unit of each gradient's value."""
    gu, gy = _data(6, 520, FP, 3)
    grad = pkg.silu_product_backward(gy, gu).double()
    d = torch.randn(gu.shape, device=DEV, generator=_gen(4)).double()

    def loss(t):
        return float((_product(gu.double() + t * d)[0] * gy.double()).sum())

    numeric = (loss(1e-5) - loss(-1e-5)) / 2e-5
    bound = float((grad * d).abs().sum()) * (HALF[FP] + 1e-5) + float(d.abs().sum()) * 1e-5
    assert abs(numeric - float((grad * d).sum())) <= bound


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,n", SHAPES)
def test_quantize_rows(pkg, dtype, m, n):
    """Every step is one correctly rounded operation: the codes and scales are those of the CPU."""
    x = (3 * torch.randn(m, n, device=DEV, generator=_gen(m * n))).to(dtype)
    q = pkg.quantize_rows(x)
    v = x.cpu().float()
    s = v.abs().amax(1) / 127
    assert torch.equal(q.scale.cpu(), s) and torch.equal(q.y.cpu(), (v / s[:, None]).round().to(I8))


def test_quantize_rows_ties_zeros_and_what_is_not_finite(pkg):
    ties = torch.arange(-126.5, 127, 1.0)  # the scale is 1: halves go to even
    x = torch.zeros(8, 256)
    x[0, :254], x[0, 254] = ties, 127.0
    x[1] = 0.0
    x[2], x[2, 9] = 1.0, float("nan")
    x[3], x[3, 250], x[3, 3] = 2.0, float("inf"), -1.0
    x[4] = -5.0
    x[5] = 2.0**-24  # fp16's least value: 2^-24 / 127 is a normal float32
    x[6, 0] = -0.0
    x[7] = torch.linspace(-60000, 60000, 256)
    x = x.to(FP)
    q = pkg.quantize_rows(x.to(DEV))
    y, s = q.y.cpu(), q.scale.cpu()
    assert float(s[0]) == 1.0 and torch.equal(y[0, :254], ties.round().to(I8)) and int(y[0, 254]) == 127
    assert float(s[1]) == 1.0 and bool((y[1] == 0).all()) and float(s[6]) == 1.0 and bool((y[6] == 0).all())
    assert bool(s[2].isnan()) and bool((y[2] == 0).all())
    assert float(s[3]) == float("inf") and bool((y[3] == 0).all())
    assert bool((y[4] == -127).all()) and bool((y[5] == 127).all()) and int(y[7].min()) == -127 and int(y[7].max()) == 127
    tiny = torch.full((1, 8), 2.0**-133, device=DEV).to(BF)  # its 127th is subnormal: the scale is 1
    q = pkg.quantize_rows(tiny)
    assert float(q.scale) == 1.0 and bool((q.y == 0).all())


def test_gates_far_out_and_what_is_not_finite(pkg):
    n = 64
    v = torch.zeros(5, n)
    v[0] = torch.linspace(-100, 100, n)
    v[1, 0], v[1, 1], v[2, 0], v[3, 0] = float("inf"), 1.0, float("nan"), -300.0
    u = torch.ones(5, n)
    gu = torch.cat([v, u], 1).to(DEV).to(BF)
    y = pkg.silu_product(gu).y.double()
    want, off = _product(gu)
    assert bool(((y - want).abs() <= HALF[BF] * (want.abs() + off) + off + TINY[BF])[[0, 4]].all())
    assert float(y[1, 0]) == float("inf") and bool(y[2, 0].isnan()) and float(y[3, 0]) == 0.0 and bool(y[2, 1:].isfinite().all())
    q = pkg.silu_product(gu, I8)
    assert float(q.scale[1]) == float("inf") and bool((q.y[1] == 0).all()) and bool(q.scale[2].isnan()) and float(q.scale[4]) == 1.0
    g = pkg.silu_product_backward(torch.ones(5, n, device=DEV, dtype=BF), gu)
    assert bool(g[[0, 3, 4]].isfinite().all()) and float(g[4, 0]) == 0.5  # at a gate of zero


@pytest.mark.parametrize("dtype", [BF, FP])
def test_strides_in_place_and_given_outputs(pkg, dtype):
    m, n = 37, 1544
    gu, gy = _data(m, n, dtype, 5)
    wide, wide_g = torch.zeros(m, 2 * n + 24, device=DEV, dtype=dtype), torch.zeros(m, n + 8, device=DEV, dtype=dtype)
    wide[:, 8:2 * n + 8], wide_g[:, :n] = gu, gy
    y, q, g = pkg.silu_product(gu).y, pkg.silu_product(gu, I8), pkg.silu_product_backward(gy, gu)
    assert torch.equal(pkg.silu_product(wide[:, 8:2 * n + 8]).y, y)
    q2 = pkg.silu_product(wide[:, 8:2 * n + 8], I8)
    assert torch.equal(q2.y, q.y) and torch.equal(q2.scale, q.scale)
    assert torch.equal(pkg.silu_product_backward(wide_g[:, :n], wide[:, 8:2 * n + 8]), g)
    own = gu.clone()
    assert pkg.silu_product_backward(gy, own, out=own) is own and torch.equal(own, g)
    r, r2 = pkg.quantize_rows(gu), pkg.quantize_rows(wide[:, 8:2 * n + 8])
    assert torch.equal(r.y, r2.y) and torch.equal(r.scale, r2.scale)
    out = torch.empty(m, n, device=DEV, dtype=I8)
    assert pkg.silu_product(gu, I8, out).y is out and torch.equal(out, q.y)


def test_no_rows(pkg):
    gu = torch.empty(0, 128, device=DEV, dtype=BF)
    assert pkg.silu_product(gu).y.shape == (0, 64)
    q = pkg.silu_product(gu, I8)
    assert q.y.shape == (0, 64) and q.scale.shape == (0,)
    assert pkg.silu_product_backward(gu[:, :64], gu).shape == (0, 128) and pkg.quantize_rows(gu).y.shape == (0, 128)


def test_more_rows_than_32_bits_of_bytes(pkg):
    """Offsets past 2^32: the last rows of 9 GB of gates and ups are the ones that a small call gives."""
    m, n = 70000, 32768
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    gu = torch.zeros(m, 2 * n, device=DEV, dtype=BF)
    gu[-3:] = _data(3, n, BF, 8)[0]
    last = gu[-3:].contiguous()
    y = pkg.silu_product(gu).y
    assert torch.equal(y[-3:], pkg.silu_product(last).y)
    del y
    q, s = pkg.silu_product(gu, I8), pkg.silu_product(last, I8)
    assert torch.equal(q.y[-3:], s.y) and torch.equal(q.scale[-3:], s.scale)


def test_captured(pkg):
    gu, gy = _data(300, 1544, BF, 31)

    def step():
        q, r = pkg.silu_product(gu, I8), pkg.quantize_rows(gy)
        return [pkg.silu_product(gu).y, q.y, q.scale, r.y, r.scale, pkg.silu_product_backward(gy, gu)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        gu.copy_(_data(300, 1544, BF, 40 + i)[0])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_gradient_of_large_values(pkg):
    """grad_y * up or grad_y * gate past float32 where the gradient itself is not (the sigmoid is far below one)."""
    n = 64
    gy = torch.full((3, n), 2.0**100, device=DEV)
    v = torch.linspace(-60, -20, n, device=DEV).repeat(3, 1)
    u = torch.full((3, n), 2.0**100, device=DEV)
    u[0], gy[1], u[1] = 2.0**60, 2.0**126, 1.0
    v[2] = -200.0
    gu, gy = torch.cat([v, u], 1).to(BF), gy.to(BF)
    got = pkg.silu_product_backward(gy, gu).double()
    v, u = gu.double().chunk(2, dim=1)
    p, g = torch.sigmoid(v), gy.double()
    rel = (12 + 3 * v.abs()) * E * (1 + v.abs())  # as above, by the size of the terms of 1 + v (1 - p)
    for part, want in ((got[:, :n], g * u * p * (1 + v * (1 - p))), (got[:, n:], g * v * p)):
        here = want.abs() < 2.0**127
        off = rel * want.abs()
        assert int(here[:2].sum()) > n and not bool(part.isnan().any())
        assert bool(((part - want).abs() <= HALF[BF] * (want.abs() + off) + off + TINY[BF])[:2][here[:2]].all())
    assert bool((got[2] == 0).all())  # exp(200) is past float32: the sigmoid is 0
