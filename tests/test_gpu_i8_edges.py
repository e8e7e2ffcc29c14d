"""Refusals and limits of the int8 products that the device has to be there for."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
BF, I8 = torch.bfloat16, torch.int8


def test_columns_that_only_int8_rows_may_have(pkg):
    """K past 32768: int8 rows go through, and 16-bit ones, which cannot be rounded at that width, are refused in terms of
    this call."""
    k, lens = 32784, torch.tensor([1, 2], device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    x, w = (torch.randint(-128, 128, s, device=DEV, generator=g).to(I8) for s in ((3, k), (2, 16, k)))
    xs, ws = torch.full((3,), 2.0**-12, device=DEV), torch.full((2, 16), 2.0**-8, device=DEV)
    got = pkg.grouped_gemm_i8(x, pkg.I8Weights(w, ws), lens, xs)
    for row, group in ((0, 0), (1, 1), (2, 1)):
        want = (w[group].double() @ x[row].double()).float() * 2.0**-8 * 2.0**-12
        assert torch.equal(got[row], want.to(BF))
    with pytest.raises(pkg.GGError, match="K must be at most 32768 for x of 16 bits") as e:
        pkg.grouped_gemm_i8(x.to(BF), pkg.I8Weights(w, ws), lens)
    assert e.value.status == 1  # GG_ERR_UNSUPPORTED
