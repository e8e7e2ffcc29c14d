"""The router's gradient where it is easily off."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("grad_loss", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("t,e,k", [(9, 8, 2), (70, 33, 4), (40, 256, 8), (20, 1000, 4)])
def test_padding_stays_zero_when_the_loss_overflows(pkg, renormalize, grad_loss, t, e, k):
    """A scaled loss that overflowed: rows of tokens that take no part are zero all the same (exactly)."""
    logits = torch.randn(t, e, device=DEV, generator=torch.Generator(device=DEV).manual_seed(e))
    mask = torch.arange(t, device=DEV) % 3 != 1
    logits[~mask] = float("nan")
    r = pkg.route(logits, k, mask, renormalize, True)
    got = pkg.route_backward(logits, r, torch.ones(t, k, device=DEV), torch.tensor(grad_loss, device=DEV))
    assert bool((got[~mask] == 0).all())
    assert bool((pkg.route_backward(logits, r, torch.ones(t, k, device=DEV))[~mask] == 0).all())
