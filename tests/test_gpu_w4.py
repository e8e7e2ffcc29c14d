"""Grouped products with 4-bit weights against a 64-bit reference.

Bound: the kernel sums x (16 + q) and sum x in float32, each product exact; over K terms the error is below
(K / 32 + 16) * 2^-24 of the sum of |x| (16 + q + 16 + z) |s| (a matrix instruction adds 32 products at a time, the
rest is a chain), and a stored value is off by half a unit in the last place.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _weights(b, n, k, group, dtype, zeros, seed):
    g = _gen(seed)
    q = torch.randint(0, 16, (b, n, k), device=DEV, generator=g, dtype=torch.uint8)
    s = (0.01 + 0.1 * torch.rand(b, n, k // group, device=DEV, generator=g)).to(dtype)
    s = torch.where(torch.rand(s.shape, device=DEV, generator=g) < 0.5, s, -s)
    z = torch.randint(0, 16, (b, n, k // group), device=DEV, generator=g, dtype=torch.uint8) if zeros else None
    return q, s, z


def _dense(q, s, z, group):
    b, n, k = q.shape
    zero = 8.0 if z is None else z.double()[..., None]
    v = q.double().view(b, n, k // group, group)
    return ((v - zero) * s.double()[..., None]).view(b, n, k), ((v + 32 + zero) * s.double().abs()[..., None]).view(b, n, k)


def _check(out, x, w, size, offs, lens, dtype, k):
    written = torch.zeros(x.shape[0], dtype=torch.bool, device=DEV)
    for g, (o, m) in enumerate(zip(offs, lens)):
        if m == 0:
            continue
        v = x[o:o + m].double()
        want, mag = v @ w[g].T, v.abs() @ size[g].T
        bound = HALF[dtype] * want.abs() + (k / 32 + 16) * 2.0**-24 * mag + 2.0**-25
        err = (out[o:o + m].double() - want).abs()
        assert bool((err <= bound).all()), (g, m, float((err - bound).max()))
        written[o:o + m] = True
    return written


CASES = [  # n, k, group, rows of the groups
    (8, 128, 128, [1]),
    (16, 32, 32, [0, 1, 0]),
    (24, 160, 32, [3, 0, 16]),
    (64, 64, 64, [17, 1, 15, 0, 2]),
    (264, 192, 64, [33, 64, 65]),
    (512, 1024, 128, [1, 1, 0, 1, 1, 0, 0, 1]),
    (2880, 2880, 32, [8, 0, 5]),
    (1000, 896, 128, [100, 31]),
    (136, 2048, 64, [130, 0, 0, 7]),
    (4096, 7168, 128, [1, 2]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,k,group,lens", CASES)
def test_against_64_bits(pkg, dtype, zeros, n, k, group, lens):
    q, s, z = _weights(len(lens), n, k, group, dtype, zeros, n + k)
    w4 = pkg.pack_w4(q, s, z)
    w, size = _dense(q, s, z, group)
    x = torch.randn(sum(lens), k, device=DEV, generator=_gen(k)).to(dtype)
    offs = [sum(lens[:g]) for g in range(len(lens))]
    for group_m in (lens, torch.tensor(lens, dtype=torch.int64, device=DEV)):
        out = torch.full((sum(lens) * n + 64,), 3.0, dtype=dtype, device=DEV)
        got = pkg.grouped_gemm_w4(x, w4, group_m, out=out[:-64].view(sum(lens), n))
        assert bool(_check(got, x, w, size, offs, lens, dtype, k).all()) and bool((out[-64:] == 3).all())
    assert torch.equal(got, pkg.grouped_gemm_w4(x, w4, group_m))


def _ragged(b, rows, seed):
    """Rows of b groups that add up to `rows`: one group with many, some with none."""
    g = torch.Generator().manual_seed(seed)
    share = torch.rand(b, generator=g) ** 2
    share[seed % b] += 3.0
    share[(seed + 1) % b] = 0.0
    lens = (share / share.sum() * rows).int().tolist()
    lens[seed % b] += rows - sum(lens)
    return lens


# The kernel is chosen by the average rows and the number of workgroups: these reach every choice (the cases above
# have few workgroups).
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group,k", [(32, 160), (64, 448), (128, 640)])
@pytest.mark.parametrize("b,n,per", [(16, 264, 2), (16, 1048, 5), (32, 1048, 12), (32, 1000, 19), (32, 1032, 21), (32, 1016, 40)])
def test_every_instance(pkg, dtype, zeros, group, k, b, n, per):
    q, s, z = _weights(b, n, k, group, dtype, zeros, n + k + per)
    w4 = pkg.pack_w4(q, s, z)
    w, size = _dense(q, s, z, group)
    lens = _ragged(b, b * per, per)
    x = torch.randn(b * per, k, device=DEV, generator=_gen(k)).to(dtype)
    out = torch.full((b * per * n + 64,), 3.0, dtype=dtype, device=DEV)
    got = pkg.grouped_gemm_w4(x, w4, torch.tensor(lens, device=DEV), out=out[:-64].view(b * per, n))
    offs = [sum(lens[:g]) for g in range(b)]
    assert bool(_check(got, x, w, size, offs, lens, dtype, k).all()) and bool((out[-64:] == 3).all())
    assert torch.equal(got, pkg.grouped_gemm_w4(x, w4, torch.tensor(lens, device=DEV)))
    # rows elsewhere than back to back, in another order of the groups
    order = sorted(range(b), key=lambda g: (g * 7) % b)
    at, start = 3, [0] * (b + 1)
    for g in order:
        start[g], at = at, at + lens[g] + 1
    wide = torch.zeros(at, k, dtype=dtype, device=DEV)
    far = torch.full((at, n), 5.0, dtype=dtype, device=DEV)
    for g in range(b):
        wide[start[g]:start[g] + lens[g]] = x[offs[g]:offs[g] + lens[g]]
    pkg.grouped_gemm_w4(wide, w4, torch.tensor(lens, device=DEV), out=far, group_offs=torch.tensor(start, device=DEV))
    for g in range(b):
        assert torch.equal(far[start[g]:start[g] + lens[g]], got[offs[g]:offs[g] + lens[g]])
        assert bool((far[start[g] + lens[g]] == 5).all())


@pytest.mark.parametrize("b", [63, 64, 65, 200, 1000])
def test_many_groups_few_with_rows(pkg, b):
    n, k, group = 32, 128, 64
    lens = [0] * b
    for i, m in ((0, 1), (b // 2, 3), (b - 1, 2)):
        lens[i] = m
    q, s, z = _weights(b, n, k, group, torch.bfloat16, True, b)
    w4 = pkg.pack_w4(q, s, z)
    w, size = _dense(q, s, z, group)
    x = torch.randn(6, k, device=DEV, generator=_gen(b)).to(torch.bfloat16)
    got = pkg.grouped_gemm_w4(x, w4, torch.tensor(lens, device=DEV))
    offs = [sum(lens[:g]) for g in range(b)]
    assert bool(_check(got, x, w, size, offs, lens, torch.bfloat16, k).all())


# Pieces of 16 and 32 rows of many groups: full ones, ragged ones, groups without rows between them, few and many rows on average.
@pytest.mark.parametrize("gaps", [False, True])
@pytest.mark.parametrize("b,sizes", [(70, (0, 17, 1, 0, 33, 16)), (300, (5, 0, 32, 0, 0, 0, 65)), (330, (64, 31, 0, 15, 48)), (520, (0, 0, 0, 0, 47, 0, 1))])
def test_pieces_of_many_groups(pkg, b, sizes, gaps):
    n, k, group, dtype = 40, 160, 32, torch.float16
    lens = [sizes[(i * i // 3) % len(sizes)] for i in range(b)]
    offs = [sum(lens[:g]) + (g // 2 if gaps else 0) for g in range(b)]
    total = offs[-1] + lens[-1] + 1
    q, s, z = _weights(b, n, k, group, dtype, True, b)
    w4 = pkg.pack_w4(q, s, z)
    w, size = _dense(q, s, z, group)
    x = torch.randn(total, k, device=DEV, generator=_gen(b)).to(dtype)
    out = torch.full((total, n), 4.0, dtype=dtype, device=DEV)
    where = torch.tensor(offs + [total], device=DEV) if gaps else None
    pkg.grouped_gemm_w4(x, w4, torch.tensor(lens, device=DEV), out=out, group_offs=where)
    written = _check(out, x, w, size, offs, lens, dtype, k)
    assert bool((out[~written] == 4).all()) and int(written.sum()) == sum(lens)


def test_offsets_gaps_and_bad_sizes(pkg):
    """Rows between groups stay as they were; a group that does not lie inside x gets no work, the others do."""
    n, k, group, dtype = 48, 256, 128, torch.bfloat16
    lens, offs = [2, 5, 1, 4, -3, 2, 1 << 40], [3, 6, 12, 17, 2, 13, 0, 22]
    q, s, z = _weights(len(lens), n, k, group, dtype, False, 1)
    w4 = pkg.pack_w4(q, s, z)
    w, size = _dense(q, s, z, group)
    x = torch.randn(20, k, device=DEV, generator=_gen(7)).to(dtype)
    out = torch.full((20, n), 9.0, dtype=dtype, device=DEV)
    pkg.grouped_gemm_w4(x, w4, torch.tensor(lens, device=DEV), out=out, group_offs=torch.tensor(offs, device=DEV))
    good = [m if i in (0, 1, 2, 5) else 0 for i, m in enumerate(lens)]  # 3: 17 + 4 > 20
    written = _check(out, x, w, size, offs, good, dtype, k)
    assert bool((out[~written] == 9).all()) and int(written.sum()) == 10
    # offsets that overlap: more groups with rows than rows
    m = 8
    q, s, z = _weights(m, n, k, group, dtype, False, 2)
    w, size = _dense(q, s, z, group)
    o = pkg.grouped_gemm_w4(x[:1].contiguous(), pkg.pack_w4(q, s, z), torch.tensor([0] * (m - 1) + [1], device=DEV),
                            group_offs=torch.zeros(m + 1, dtype=torch.int64, device=DEV))
    _check(o, x[:1], w, size, [0] * m, [0] * (m - 1) + [1], dtype, k)


def test_values_that_do_not_mix(pkg):
    """A row of NaN or infinity stays in its own output row; weights past N and columns past K do not exist."""
    n, k, group, dtype = 40, 160, 32, torch.bfloat16
    lens = [18, 3]
    q, s, z = _weights(2, n, k, group, dtype, True, 3)
    w4 = pkg.pack_w4(q, s, z)
    x = torch.randn(21, k, device=DEV, generator=_gen(8)).to(dtype)
    clean = pkg.grouped_gemm_w4(x, w4, lens)
    x[4] = float("nan")
    x[19, 3] = float("inf")
    got = pkg.grouped_gemm_w4(x, w4, lens)
    rest = [i for i in range(21) if i not in (4, 19)]
    assert torch.equal(got[rest], clean[rest]) and bool(got[4].isnan().all()) and not bool(got[19].isfinite().all())
    # what lies in the padding of the storage does not reach a result
    p, sc, zr = w4.packed.clone(), w4.scales.clone(), w4.zeros.clone()
    sc[:, 2, :, 8:] = float("nan")  # rows 40-47
    zr[:, 2, :, 8:] = 255
    p[:, :, 1, :, 4:] = 0xff        # columns 160-255
    dirty = pkg.W4Weights(p, sc, zr, n, k, group)
    assert torch.equal(pkg.grouped_gemm_w4(x[:4].contiguous(), dirty, [4, 0]), got[:4])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantized_weights_are_near(pkg, dtype, zeros):
    """quantize_w4: each weight within half a step (and a clipped end's one step and a half of zero points' rounding)."""
    b, n, k, group = 2, 40, 256, 64
    w = torch.randn(b, n, k, device=DEV, generator=_gen(6)).to(dtype)
    w[0, 3] = 0
    w4 = pkg.quantize_w4(w, group, zeros)
    x = torch.eye(k, device=DEV, dtype=dtype)
    v = w.float().view(b, n, -1, group)
    step = ((v.amax(3).clamp(min=0) - v.amin(3).clamp(max=0)) / 15 if zeros else v.abs().amax(3) / 7.5).repeat_interleave(group, 2)
    for g in range(b):
        out = pkg.grouped_gemm_w4(x, w4, [k if i == g else 0 for i in range(b)]).float().t()
        assert bool(((out - w[g].float()).abs() <= step[g] * 1.02 + 1e-6).all())


def test_other_stream_and_graph(pkg):
    n, k, group = 512, 512, 128
    q, s, z = _weights(4, n, k, group, torch.bfloat16, True, 12)
    w4 = pkg.pack_w4(q, s, z)
    x = torch.randn(9, k, device=DEV, generator=_gen(2)).to(torch.bfloat16)
    lens = torch.tensor([4, 0, 3, 2], device=DEV)
    want = pkg.grouped_gemm_w4(x, w4, lens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = pkg.grouped_gemm_w4(x, w4, lens, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.grouped_gemm_w4(x, w4, lens)
    for sizes in ([9, 0, 0, 0], [0, 0, 0, 9], [1, 2, 3, 3]):
        lens.copy_(torch.tensor(sizes))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, pkg.grouped_gemm_w4(x, w4, lens))


def test_torch_level_refusals(pkg):
    q, s, z = _weights(2, 16, 128, 128, torch.bfloat16, False, 1)
    w4 = pkg.pack_w4(q, s, z)
    x = torch.zeros(4, 128, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        pkg.grouped_gemm_w4(x, w4, [4])
    with pytest.raises(ValueError):
        pkg.grouped_gemm_w4(x, w4, [5, -1])
    with pytest.raises(TypeError):
        pkg.grouped_gemm_w4(x.half(), w4, [4, 0])
    with pytest.raises(ValueError):
        pkg.grouped_gemm_w4(x[:, :64], w4, [4, 0])
    with pytest.raises(ValueError):
        pkg.grouped_gemm_w4(x, w4._replace(k=256), [4, 0])
    with pytest.raises(ValueError):
        pkg.grouped_gemm_w4(x, w4, [4, 0], group_offs=torch.zeros(3, dtype=torch.int64, device=DEV))
