"""dispatch, combine and their gradients against 64-bit references.

Copies have to be equal. A sum of at most 32 products in float32 is off by 33 * 2^-24 < 2.1e-6 = F of the sum of
its magnitudes, a stored value by half a unit more; the dot product of combine's gradient is a chain of at most
H / 64 terms and a tree: D = 1e-5 up to H = 8192.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
F, D = 2.1e-6, 1e-5


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _routing(pkg, t, e, k, seed, masked=False, closed=False):
    g = _gen(seed)
    logits = torch.randn(t, e, device=DEV, generator=g)
    if closed:
        logits[:, ::2] = float("-inf")  # slots past the open experts stay empty
    mask = torch.rand(t, device=DEV, generator=g) < 0.6 if masked else None
    return pkg.route(logits, k, mask)


CASES = [(1, 2, 1, 8, False, False), (1, 8, 8, 64, False, False), (5, 8, 2, 4096, True, False), (300, 16, 4, 520, True, True),
         (33, 60, 6, 7168, False, False), (1000, 32, 8, 128, True, False), (64, 64, 32, 264, False, True), (7, 8, 1, 16384, True, False),
         (2, 4, 4, 8, True, True)]


def _bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float32])
@pytest.mark.parametrize("t,e,k,h,masked,closed", CASES)
def test_dispatch(pkg, dtype, t, e, k, h, masked, closed):
    h = max(h, 16 // torch.empty(0, dtype=dtype).element_size())
    h -= h % 16 if dtype == torch.float8_e4m3fn else 0
    r = _routing(pkg, t, e, k, t + h, masked, closed)
    x = torch.randn(t, h, device=DEV, generator=_gen(h)).to(dtype)
    out = torch.full((t * k * h * x.element_size() + 64,), 0x5a, dtype=torch.uint8, device=DEV)
    xs = pkg.dispatch(x, r, out=out[:-64].view(dtype).view(t * k, h))
    want = torch.zeros(t * k, h * x.element_size(), dtype=torch.uint8, device=DEV)
    ok = r.rows >= 0
    tok = torch.arange(t, device=DEV)[:, None].expand(t, k)
    want[r.rows[ok].long()] = _bits(x).view(t, -1)[tok[ok]]
    assert torch.equal(_bits(xs).view(t * k, -1), want)
    assert bool((out[-64:] == 0x5a).all())
    # rows of another stride
    wide = torch.zeros(t, h * x.element_size() + 32, dtype=torch.uint8, device=DEV)
    wide[:, 16:-16] = _bits(x).view(t, -1)
    assert torch.equal(_bits(pkg.dispatch(wide.view(dtype)[:, 16 // x.element_size():][:, :h], r)).view(t * k, -1), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k,h,masked,closed", CASES)
def test_combine_and_gradients(pkg, dtype, t, e, k, h, masked, closed):
    r = _routing(pkg, t, e, k, t + h + 1, masked, closed)
    g = _gen(k)
    y = torch.randn(t * k, h, device=DEV, generator=g).to(dtype)
    used = int(r.offs[-1])
    y[used:] = float("nan")  # rows that belong to no slot are not read
    ok = r.rows >= 0
    at = r.rows.clamp(min=0).long()
    rows = torch.where(ok[:, :, None], y[at].double(), 0.0)
    w = r.weights.double()

    out = pkg.combine(y, r)
    want, size = (rows * w[:, :, None]).sum(1), (rows.abs() * w[:, :, None]).sum(1)
    assert bool(((out.double() - want).abs() <= HALF[dtype] * want.abs() + F * size + 2.0**-25).all())

    back = pkg.dispatch_backward(y, r)
    assert bool(((back.double() - rows.sum(1)).abs() <= HALF[dtype] * rows.sum(1).abs() + F * rows.abs().sum(1) + 2.0**-25).all())

    wide = torch.randn(t, h + 8, device=DEV, generator=g).to(dtype)
    go = wide[:, 8:]
    gy, gw = pkg.combine_backward(go, y, r)
    want_y = torch.zeros(t * k, h, dtype=torch.float64, device=DEV)
    tok = torch.arange(t, device=DEV)[:, None].expand(t, k)
    want_y[r.rows[ok].long()] = go.double()[tok[ok]] * w[ok][:, None]
    assert bool(((gy.double() - want_y).abs() <= HALF[dtype] * want_y.abs() * 1.001 + 2.0**-25).all())
    dots = (rows * go.double()[:, None, :])
    assert bool(((gw.double() - dots.sum(2)).abs() <= D * dots.abs().sum(2)).all())
    assert bool((gw[~ok] == 0).all()) and bool((gy[used:] == 0).all())
    again = pkg.combine_backward(go, y, r)
    assert torch.equal(gy, again[0]) and torch.equal(gw, again[1])


@pytest.mark.parametrize("t,e,k,h,masked", [(26000, 16, 2, 2056, False), (13000, 32, 4, 2048, True)])
def test_outputs_past_the_caches(pkg, t, e, k, h, masked):
    """More than 192 MB of rows: stores that bypass the caches, same results."""
    r = _routing(pkg, t, e, k, 5, masked)
    ok, at = r.rows >= 0, r.rows.clamp(min=0).long()
    x = torch.randn(t, h, device=DEV, generator=_gen(1)).to(torch.bfloat16)
    xs = pkg.dispatch(x, r)
    assert xs.numel() * 2 > 192 << 20
    assert bool((xs[int(r.offs[-1]):] == 0).all())
    for s in range(k):
        assert torch.equal(xs[at[ok[:, s], s]], x[ok[:, s]])
    gy, gw = pkg.combine_backward(x, xs, r)
    assert bool((gy[int(r.offs[-1]):] == 0).all())
    norm = x.double().square().sum(1)
    for s in range(k):
        o = ok[:, s]
        want = x[o].double() * r.weights[o, s, None].double()
        assert bool(((gy[at[o, s]].double() - want).abs() <= HALF[torch.bfloat16] * want.abs() * 1.001).all())
        assert bool(((gw[o, s].double() - norm[o]).abs() <= D * norm[o]).all())


def test_gradients_against_differences(pkg):
    """combine is linear in y and in the weights: the difference along a direction is exact."""
    t, e, k, h = 9, 8, 3, 64
    r = _routing(pkg, t, e, k, 4)
    g = _gen(5)
    y, go = torch.randn(t * k, h, device=DEV, generator=g).to(torch.float16), torch.randn(t, h, device=DEV, generator=g).to(torch.float16)
    gy, gw = pkg.combine_backward(go, y, r)

    def loss(yy, w):
        return (go.double() * (yy[r.rows.long()] * w[:, :, None]).sum(1)).sum()

    dy, dw = torch.randn(t * k, h, device=DEV, generator=g).double(), torch.randn(t, k, device=DEV, generator=g).double()
    ny = float(loss(y.double() + dy, r.weights.double()) - loss(y.double(), r.weights.double()))
    nw = float(loss(y.double(), r.weights.double() + dw) - loss(y.double(), r.weights.double()))
    assert abs(ny - float((gy.double() * dy).sum())) <= HALF[torch.float16] * float((gy.double() * dy).abs().sum()) * 1.01
    assert abs(nw - float((gw.double() * dw).sum())) <= D * float((gw.double() * dw).abs().sum()) + 1e-6 * float(dw.abs().sum())


def test_dispatch_combine_round_trip(pkg):
    """Renormalised weights sum to one: the weighted sum of copies is the token itself."""
    r = _routing(pkg, 500, 32, 4, 9)
    x = torch.randn(500, 256, device=DEV, generator=_gen(1)).to(torch.bfloat16)
    out = pkg.combine(pkg.dispatch(x, r), r)
    assert bool(((out.double() - x.double()).abs() <= 2.0**-8 * x.double().abs()).all())


def test_rows_out_of_range_are_ignored(pkg):
    t, k, h = 4, 2, 64
    r = _routing(pkg, t, 8, k, 2)
    rows = r.rows.clone()
    rows[1, 0], rows[2, 1] = 8, -5  # outside 0 .. t * k - 1
    bad = r._replace(rows=rows)
    x = torch.randn(t, h, device=DEV, generator=_gen(1)).to(torch.bfloat16)
    out = torch.full((t * k + 2, h), 7.0, dtype=torch.bfloat16, device=DEV)
    pkg.dispatch(x, bad, out=out[:t * k])
    assert bool((out[t * k:] == 7).all())
    y = torch.randn(t * k, h, device=DEV, generator=_gen(2)).to(torch.bfloat16)
    c = pkg.combine(y, bad)
    assert bool(c.isfinite().all())
    _, gw = pkg.combine_backward(x, y, bad)
    assert float(gw[1, 0]) == 0.0 and float(gw[2, 1]) == 0.0


def test_no_tokens(pkg):
    r = pkg.route(torch.empty(0, 8, device=DEV), 2)
    x = torch.empty(0, 64, device=DEV, dtype=torch.bfloat16)
    assert pkg.dispatch(x, r).shape == (0, 64) and pkg.combine(x, r).shape == (0, 64)
    gy, gw = pkg.combine_backward(x, x, r)
    assert gy.shape == (0, 64) and gw.shape == (0, 2)


def test_other_stream(pkg):
    r = _routing(pkg, 100, 16, 4, 3)
    x = torch.randn(100, 512, device=DEV, generator=_gen(3)).to(torch.bfloat16)
    want = pkg.combine(pkg.dispatch(x, r), r)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = pkg.combine(pkg.dispatch(x, r, stream=side.cuda_stream), r, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want)


def test_torch_level_refusals(pkg):
    r = _routing(pkg, 4, 8, 2, 1)
    x = torch.zeros(4, 64, device=DEV, dtype=torch.bfloat16)
    y = torch.zeros(8, 64, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        pkg.dispatch(x[:3], r)
    with pytest.raises(TypeError):
        pkg.dispatch(x.double(), r)
    with pytest.raises(ValueError):
        pkg.combine(y[:7], r)
    with pytest.raises(TypeError):
        pkg.combine(y.float(), r)
    with pytest.raises(ValueError):
        pkg.combine_backward(x.half(), y, r)
    with pytest.raises(pkg.GGError, match="16 bytes"):
        pkg.combine(torch.zeros(8, 60, device=DEV, dtype=torch.bfloat16), r)
