"""The router, its counting sort, balance loss and gradients against 64-bit references.

Whole numbers have to be equal. Probabilities: the exponent's argument is a float32 difference of logits of at
most 64, off by 2^-24 of it, exp and log by two units, sums of at most 1024 terms: below 1e-5 = F relative.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
F = 1e-5
INF = float("inf")
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0**-24}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _reference(logits, k, mask, renormalize):
    t, e = logits.shape
    l = logits.double()
    l = torch.where(mask[:, None], l, torch.zeros_like(l)) if mask is not None else l
    live = l.amax(1) > -INF
    live |= l.isnan().any(1)
    if mask is not None:
        live &= mask
    order = torch.sort(l, dim=1, descending=True, stable=True)
    experts, best = order.indices[:, :k], order.values[:, :k]
    ok = live[:, None] & ~(best == -INF)
    lse = torch.logsumexp(l, 1)
    w = torch.exp(best - lse[:, None])
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    flat = torch.where(ok, experts, e).reshape(-1)
    counts = torch.bincount(flat, minlength=e + 1)[:e]
    offs = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.empty_like(flat)
    place[torch.sort(flat, stable=True).indices] = torch.arange(t * k, device=DEV)
    p = torch.exp(l - lse[:, None])
    n = max(1, int(live.sum()))
    slope = counts.double() * e / max(1, int(counts.sum())) / n
    loss = (slope * torch.where(live[:, None], p, torch.zeros_like(p)).sum(0)).sum()
    return dict(experts=torch.where(ok, experts, -1).int(), weights=torch.where(ok, w, 0.0), counts=counts, offs=offs,
                rows=torch.where(ok, place.view(t, k), -1).int(), lse=torch.where(live, lse, -INF), slope=slope, loss=loss, p=p,
                live=live, ok=ok)


def _check(r, want, balance):
    for name in ("experts", "counts", "offs", "rows"):
        got = getattr(r, name)
        assert torch.equal(got, want[name].to(got.dtype)), name
    w = want["weights"]
    assert bool(((r.weights.double() - w).abs() <= F * w + 1e-37).all() if not w.isnan().any() else
                torch.equal(r.weights.isnan(), w.isnan()))
    live = want["live"] & want["lse"].isfinite()
    assert bool((r.lse[~want["live"]] == -INF).all())
    d = (r.lse.double() - want["lse"])[live]
    assert bool((d.abs() <= F * (1 + want["lse"][live].abs())).all())
    if balance:
        assert bool(((r.slope.double() - want["slope"]).abs() <= F * want["slope"]).all())
        assert abs(float(r.loss) - float(want["loss"])) <= F * float(want["loss"]) + 1e-37
    else:
        assert r.slope is None and r.loss is None


CASES = [(1, 1, 1), (1, 2, 2), (3, 5, 2), (2, 8, 8), (33, 16, 4), (40, 17, 3), (129, 32, 4), (128, 60, 6), (500, 64, 1), (130, 65, 8),
         (257, 100, 5), (64, 128, 32), (300, 129, 8), (1000, 256, 8), (129, 257, 7), (70, 512, 16), (100, 513, 9), (35, 1024, 32),
         (5000, 48, 2), (20000, 8, 2), (3, 1000, 1), (4097, 256, 8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k", CASES)
def test_route(pkg, dtype, t, e, k):
    g = _gen(t * e + k)
    logits = (2 * torch.randn(t, e, device=DEV, generator=g)).to(dtype)  # 16-bit ones tie often
    for renormalize, balance in ((True, False), (False, True)):
        r = pkg.route(logits, k, renormalize=renormalize, balance=balance)
        _check(r, _reference(logits, k, None, renormalize), balance)
        again = pkg.route(logits, k, renormalize=renormalize, balance=balance)
        assert all(torch.equal(a, b) for a, b in zip(r[:8], again[:8]) if a is not None)


# Either side of where 129 to 256 experts take other lanes; chunks beyond what the scan holds in registers at once.
@pytest.mark.parametrize("t,e,k", [(64, 200, 6), (65, 200, 6), (300, 256, 20), (64, 256, 12), (16384, 256, 8), (16385, 130, 9), (40000, 200, 3), (70001, 16, 1),
                                   (140000, 6, 2)])
def test_route_sizes_that_choose(pkg, t, e, k):
    g = _gen(t + e)
    logits = 2 * torch.randn(t, e, device=DEV, generator=g)
    mask = torch.rand(t, device=DEV, generator=g) < 0.9
    _check(pkg.route(logits, k, mask, True, True), _reference(logits, k, mask, True), True)


@pytest.mark.parametrize("t,e,k", [(1, 8, 2), (7, 33, 4), (200, 64, 8), (1500, 256, 8), (140, 1024, 12)])
def test_mask_hides_garbage(pkg, t, e, k):
    """Masked tokens hold NaN and infinities, masked experts -infinity; some tokens have no expert left, one
    call has no token left."""
    g = _gen(e)
    logits = torch.randn(t, e, device=DEV, generator=g)
    closed = torch.rand(t, e, device=DEV, generator=g) < 0.3
    logits[closed] = -INF
    logits[::5] = -INF
    if t > 1:
        logits[1, e // 2:] = -INF
        logits[1, 0] = 1.0
    mask = torch.rand(t, device=DEV, generator=g) < 0.7
    if t > 1:
        mask[1] = True
    want = _reference(torch.where(mask[:, None], logits, 0.0), k, mask, True)
    dirty = torch.where(mask[:, None], logits, float("nan"))
    dirty[~mask, 0] = INF
    r = pkg.route(dirty, k, mask, True, True)
    _check(r, want, True)
    none = pkg.route(dirty, k, torch.zeros_like(mask), True, True)
    assert bool((none.experts == -1).all()) and bool((none.rows == -1).all()) and int(none.counts.sum()) == 0
    assert float(none.loss) == 0.0 and bool((none.weights == 0).all()) and bool((none.slope == 0).all())
    grad = pkg.route_backward(dirty, r, torch.ones(t, k, device=DEV), torch.ones(1, device=DEV))
    assert bool((grad[~mask] == 0).all()) and bool(grad.isfinite().all())


@pytest.mark.parametrize("e", [40, 64, 100, 256, 300, 512, 1000])
@pytest.mark.parametrize("k", [1, 5, 8, 12])
@pytest.mark.parametrize("masked", [False, True])
def test_values_that_differ_in_the_last_bits(pkg, e, k, masked):
    """Float32 logits a unit or a few apart, in pairs, threes and more, among the chosen and at their end; equal ones too."""
    t, g = 700, _gen(e + k)
    logits = torch.randn(t, e, device=DEV, generator=g)
    order = logits.argsort(1, descending=True)
    bits = logits.view(torch.int32)
    every = torch.arange(t, device=DEV)
    for kind, tokens in enumerate(every.view(7, 100)):
        if kind == 6:  # all of a token's logits within 64 units
            bits[tokens] = 0x3f800000 + torch.randint(0, 64, (100, e), device=DEV, generator=g, dtype=torch.int32)
            continue
        for n in range(1, (2, 2, 3, 4, 2, 5)[kind]):  # the n values after the first of each run come near it
            for at in ((0, 3), (k - 1,), (max(k - 2, 0),), (1,), (k,), (k // 2,))[kind]:
                first, then = order[tokens, at], order[tokens, at + n]
                off = torch.randint(-3, 4, (100,), device=DEV, generator=g, dtype=torch.int32)
                bits[tokens, then] = bits[tokens, first] + off
    if masked:
        logits[torch.rand(t, e, device=DEV, generator=g) < 0.5] = -INF
    r = pkg.route(logits, k, balance=True)
    _check(r, _reference(logits, k, None, True), True)


def test_special_values(pkg):
    l = torch.zeros(6, 8, device=DEV)
    l[0] = torch.tensor([0.0, -0.0, 0.0, -0.0, 0.0, 0.0, 0.0, 0.0])           # all equal: by index
    l[1, 3], l[1, 6] = float("nan"), float("nan")                              # NaN first, by index
    l[2, 5] = INF
    l[3] = torch.finfo(torch.float32).min                                      # the type's lowest value is a value
    l[3, 7] = -INF
    l[4] = torch.tensor([-1e-45, 1e-45, 0.0, -3e38, 3e38, 1.0, -1.0, 2.0])     # subnormals keep their order
    r = pkg.route(l, 4)
    assert r.experts.tolist() == [[0, 1, 2, 3], [3, 6, 0, 1], [5, 0, 1, 2], [0, 1, 2, 3], [4, 7, 5, 1], [0, 1, 2, 3]]
    assert bool(r.weights[1].isnan().all()) and bool(r.weights[2].isnan().any())
    assert r.weights[0].tolist() == [0.25] * 4 and r.weights[3].tolist() == [0.25] * 4
    assert int(r.counts.sum()) == 24 and sorted(r.rows.flatten().tolist()) == list(range(24))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,shift", [(3, 0), (4, 0), (8, 1), (16, 8)])
def test_strides(pkg, dtype, pad, shift):
    t, e, k = 300, 64, 4
    wide = torch.randn(t, e + pad + shift, device=DEV, generator=_gen(pad)).to(dtype)
    view = wide[:, shift:shift + e]
    r, want = pkg.route(view, k, balance=True), pkg.route(view.contiguous(), k, balance=True)
    assert all(torch.equal(a, b) for a, b in zip(r[:8], want[:8]))
    gw = torch.randn(t, k, device=DEV, generator=_gen(1))
    assert torch.equal(pkg.route_backward(view, r, gw), pkg.route_backward(view.contiguous(), r, gw))


def test_no_tokens(pkg):
    r = pkg.route(torch.empty(0, 8, device=DEV), 2, balance=True)
    assert r.counts.tolist() == [0] * 8 and r.offs.tolist() == [0] * 9 and float(r.loss) == 0.0 and r.rows.shape == (0, 2)
    assert pkg.route_backward(torch.empty(0, 8, device=DEV), r, torch.empty(0, 2, device=DEV)).shape == (0, 8)


def _grad_reference(logits, r, want, gw, gl, renormalize):
    """(gradient, sum of the magnitudes of its terms), in 64 bits."""
    p = torch.where(want["live"][:, None], want["p"], 0.0)
    e = r.experts.clamp(min=0).long()
    sel = torch.where(want["ok"], torch.take_along_dim(p, e, 1), 0.0)
    gp = torch.zeros_like(p) if gl is None else (gl.double() * want["slope"]).expand_as(p).clone()
    size = gp.abs()
    if gw is not None:
        g = torch.where(want["ok"], gw.double(), 0.0)
        if renormalize:
            total = sel.sum(1, keepdim=True).clamp(min=1e-300)
            mean = (g * sel).sum(1, keepdim=True) / total
            size = size.clone().scatter_add_(1, e, (g.abs() + (g.abs() * sel).sum(1, keepdim=True) / total) / total * want["ok"])
            g = (g - mean) / total
        else:
            size = size.clone().scatter_add_(1, e, g.abs())
        gp = gp.scatter_add(1, e, g * want["ok"])
    out = p * (gp - (p * gp).sum(1, keepdim=True))
    return out, p * (size + (p * size).sum(1, keepdim=True))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k", [(1, 4, 1), (3, 5, 2), (50, 16, 4), (129, 33, 6), (500, 64, 8), (77, 100, 4), (300, 256, 8), (40, 500, 8),
                                   (20, 1024, 32)])
def test_backward(pkg, dtype, t, e, k):
    g = _gen(t + e)
    logits = torch.randn(t, e, device=DEV, generator=g).to(dtype)
    mask = torch.rand(t, device=DEV, generator=g) < 0.8
    gw, gl = torch.randn(t, k, device=DEV, generator=g), torch.tensor(0.7, device=DEV)
    for renormalize in (True, False):
        r = pkg.route(logits, k, mask, renormalize, True)
        want = _reference(logits, k, mask, renormalize)
        for a, b in ((gw, gl), (gw, None), (None, gl)):
            got = pkg.route_backward(logits, r, a, b)
            ref, size = _grad_reference(logits, r, want, a, b, renormalize)
            assert got.dtype == dtype
            err = (got.double() - ref).abs()
            assert bool((err <= HALF[dtype] * ref.abs() + 4 * F * size + TINY[dtype]).all())
    assert bool((pkg.route_backward(logits, r) == 0).all())


def test_backward_against_differences(pkg):
    """Weights' and loss's gradient along a direction against a central difference in 64 bits, with the chosen
    experts and the counts held (they are whole numbers)."""
    t, e, k = 11, 24, 3
    g = _gen(3)
    logits = torch.randn(t, e, device=DEV, generator=g)
    gw, gl = torch.randn(t, k, device=DEV, generator=g), torch.tensor([1.3], device=DEV)
    for renormalize in (True, False):
        r = pkg.route(logits, k, None, renormalize, True)
        got = pkg.route_backward(logits, r, gw, gl)

        def loss(l):
            p = torch.softmax(l, 1)
            w = torch.take_along_dim(p, r.experts.long(), 1)
            if renormalize:
                w = w / w.sum(1, keepdim=True)
            return (gw.double() * w).sum() + gl.double() * (r.slope.double() * p.sum(0)).sum()

        for s in range(3):
            d = torch.randn(t, e, device=DEV, generator=_gen(100 + s)).double()
            step, l = 1e-5, logits.double()
            numeric = float((loss(l + step * d) - loss(l - step * d)) / (2 * step))
            exact = float((got.double() * d).sum())
            assert abs(numeric - exact) <= 4 * F * float((got.double() * d).abs().sum()) + 1e-6, (numeric, exact)


def test_other_stream_and_graph(pkg):
    logits = torch.randn(3000, 64, device=DEV, generator=_gen(8))
    want = pkg.route(logits, 6, balance=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = pkg.route(logits, 6, balance=True, stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got[:8], want[:8]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = pkg.route(logits, 6, balance=True)
        grad = pkg.route_backward(logits, r, r.weights, r.loss)
    for i in range(3):
        logits.copy_(torch.randn(3000, 64, device=DEV, generator=_gen(50 + i)))
        graph.replay()
        torch.cuda.synchronize()
        e = pkg.route(logits, 6, balance=True)
        assert all(torch.equal(a, b) for a, b in zip(r[:8], e[:8]))
        assert torch.equal(grad, pkg.route_backward(logits, e, e.weights, e.loss))


def test_torch_level_refusals(pkg):
    l = torch.zeros(4, 8, device=DEV)
    r = pkg.route(l, 2)
    with pytest.raises(ValueError):
        pkg.route(l, 9)
    with pytest.raises(TypeError):
        pkg.route(l, 2, torch.ones(4, device=DEV))
    with pytest.raises(ValueError):
        pkg.route(l, 2, torch.ones(5, dtype=torch.bool, device=DEV))
    with pytest.raises(ValueError, match="balance"):
        pkg.route_backward(l, r, None, torch.ones(1, device=DEV))
    with pytest.raises(ValueError):
        pkg.route_backward(l, r, torch.ones(4, 3, device=DEV))
    with pytest.raises(pkg.GGError, match="at most 1024"):
        pkg.route(torch.zeros(2, 1025, device=DEV), 2)
