"""The 4-bit products at the sizes that choose a kernel, in workgroups that take more than one piece of rows, and with
values near the end of the stated range. Bounds as in test_gpu_w4.py."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

import w4_cases  # noqa: E402
from test_gpu_w4 import DEV, _check, _dense, _gen, _ragged, _weights  # noqa: E402

FORMATS = [(32, 160), (64, 448), (128, 128), (128, 640)]  # weights a scale, k


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group,k", FORMATS)
@pytest.mark.parametrize("kernel,b,m,n", w4_cases.CHOICES)
def test_sizes_that_choose(pkg, dtype, zeros, group, k, kernel, b, m, n):
    q, s, z = _weights(b, n, k, group, dtype, zeros, n + k + m)
    w4 = pkg.pack_w4(q, s, z)
    w, size = _dense(q, s, z, group)
    lens = _ragged(b, m, m)
    x = torch.randn(m, k, device=DEV, generator=_gen(k)).to(dtype)
    out = torch.full((m * n + 64,), 3.0, dtype=dtype, device=DEV)
    got = pkg.grouped_gemm_w4(x, w4, torch.tensor(lens, device=DEV), out=out[:-64].view(m, n))
    offs = [sum(lens[:g]) for g in range(b)]
    assert bool(_check(got, x, w, size, offs, lens, dtype, k).all()) and bool((out[-64:] == 3).all())
    assert torch.equal(got, pkg.grouped_gemm_w4(x, w4, torch.tensor(lens, device=DEV)))


def _trips(kernel, b, m):
    """(rows, first rows, whether inside x) of groups whose pieces are about three times or more the grid's, and of which
    those inside x are the first of each trip of the workgroups."""
    lens, offs, good, at = [], [], [], 0
    if kernel == "rows":  # 40 groups of 680 rows: 40 + 680 / 32 = 61 pieces a trip
        for _ in range(b // 5):
            for rows in (33, 40):
                lens, offs, good, at = lens + [rows], offs + [at], good + [True], at + rows + 1
            lens, offs, good = lens + [m, m, 13 * 32], offs + [1, m - 1, m - 100], good + [False] * 3  # 22 + 22 + 13 pieces
    else:  # a row each: 32 + 32 / 16 = 34 pieces a trip
        for g in range(b):
            inside = g % 34 < 6 and at < m
            lens, offs, good = lens + [1], offs + [at if inside else m if g % 2 else -1], good + [inside]
            at += inside
    return lens, offs, good


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group,k", FORMATS)
@pytest.mark.parametrize("kernel,b,m,n", w4_cases.TRIPS)
def test_workgroups_that_come_back(pkg, dtype, zeros, group, k, kernel, b, m, n):
    """More pieces than the grid holds: a workgroup takes its next one after groups outside x and after its own."""
    lens, offs, good = _trips(kernel, b, m)
    rows = 32 if kernel == "rows" else 16
    grid = min(b, m) + m // rows
    pieces = [g for g, length in enumerate(lens) for _ in range(-(-length // rows))]
    trips = [p // grid for p, g in enumerate(pieces) if good[g]]
    assert len(lens) == b and max(trips) >= 4 and all(p % grid < 6 for p, g in enumerate(pieces) if good[g])
    q, s, z = _weights(b, n, k, group, dtype, zeros, n + k)
    w4 = pkg.pack_w4(q, s, z)
    w, size = _dense(q, s, z, group)
    x = torch.randn(m, k, device=DEV, generator=_gen(k)).to(dtype)
    out = torch.full((m, n), 9.0, dtype=dtype, device=DEV)
    pkg.grouped_gemm_w4(x, w4, torch.tensor(lens, device=DEV), out=out, group_offs=torch.tensor(offs + [0], device=DEV))
    written = _check(out, x, w, size, offs, [length if ok else 0 for length, ok in zip(lens, good)], dtype, k)
    assert bool((out[~written] == 9).all()) and int(written.sum()) == sum(length for length, ok in zip(lens, good) if ok)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("signs", ["one", "both"])
@pytest.mark.parametrize("b,m,n", [(2, 3, 64), (32, 1024, 904)])
def test_values_up_to_the_stated_limit(pkg, zeros, signs, b, m, n):
    """62 times the sum of |x| over a scale's k just below 3.4e38: the sums on the way stay finite."""
    k, group, dtype = 256, 128, torch.bfloat16
    q, s, z = _weights(b, n, k, group, dtype, zeros, 5)
    w4 = pkg.pack_w4(q, s, z)
    w, size = _dense(q, s, z, group)
    x = torch.full((m, k), 4.2e34, device=DEV)
    if signs == "both":
        x = torch.where(torch.rand(m, k, device=DEV, generator=_gen(3)) < 0.5, x, -x)
    x = x.to(dtype)
    assert float(x.double().abs().view(m, k // group, group).sum(2).max()) * 62 < 3.4e38
    lens = [m // b + (g < m % b) for g in range(b)]
    got = pkg.grouped_gemm_w4(x, w4, lens)
    assert bool(got.isfinite().all())
    assert bool(_check(got, x, w, size, [sum(lens[:g]) for g in range(b)], lens, dtype, k).all())
