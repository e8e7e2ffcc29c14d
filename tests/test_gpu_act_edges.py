"""The gated activation's gradient at the ends of bf16's range, against its formula in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
BF = torch.bfloat16
HALF, TINY, E = 2.0**-8, 2.0**-134, 2.0**-23


@pytest.mark.parametrize("up", [3.38e38, -3.38e38, 2.0**127, 2.0**-120])
@pytest.mark.parametrize("grad", [1.5, 2.0**-1, 2.0**-20, -2.0**-60])
def test_gradient_of_the_largest_ups(pkg, up, grad):
    """silu's slope is up to 1.1: up times it is past float32 where the gradient, with a small grad_y, is not. The bounds
    are those of the sigmoid and four products in float32, (12 + 3 |v|)(1 + |v|) 2^-23, and half a unit of the stored value;
    past bf16's range the gradient is infinite."""
    n = 256
    v = torch.linspace(-20, 20, n, device=DEV).repeat(2, 1)
    gu = torch.cat([v, torch.full((2, n), up, device=DEV)], 1).to(BF)
    gy = torch.full((2, n), grad, device=DEV).to(BF)
    got = pkg.silu_product_backward(gy, gu).double()
    v, u = gu.double().chunk(2, dim=1)
    p, g = torch.sigmoid(v), gy.double()
    gate, rel = g * u * p * (1 + v * (1 - p)), (12 + 3 * v.abs()) * E
    for part, want, off in ((got[:, :n], gate, rel * (1 + v.abs()) * (g * u * p).abs()), (got[:, n:], g * v * p, rel * (g * v * p).abs())):
        within = want.abs() < 3.36e38  # bf16 holds 3.39e38
        assert not bool(part.isnan().any())
        assert bool(((part - want).abs() <= HALF * (want.abs() + off) + off + TINY)[within].all())
        assert bool((part[want.abs() > 3.42e38].abs() == float("inf")).all())
