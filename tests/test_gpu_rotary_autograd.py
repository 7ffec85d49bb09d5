"""Second derivatives and forward mode through the rotary kernels."""
import pytest
import torch
from torch.autograd import forward_ad

from jasper_b200 import paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_second_derivatives_and_forward_mode(cuda, layout):
    """Of sum(y^3) + sum(x^2), y the turned x: R^T diag(6 y) R d + 2 d."""
    g = torch.Generator(device="cuda").manual_seed(5)
    r = paged.Rotary(32, 24, layout=layout, scaling="yarn", factor=4.0, trained_length=2048)
    x = torch.randn(2, 13, 3, 32, generator=g, device="cuda", requires_grad=True)
    d = torch.randn(2, 13, 3, 32, generator=g, device="cuda")
    positions = torch.randint(0, 10_000, (13,), generator=g, device="cuda")
    y = r.apply(x, positions)
    first, = torch.autograd.grad((y ** 3).sum() + (x ** 2).sum(), x, create_graph=True)
    second, = torch.autograd.grad((first * d).sum(), x)
    with torch.no_grad():
        want = r.grad(6 * y * r.apply(d, positions), positions) + 2 * d
        # two products and a sum, in another order: each off by half a unit, 2^-24, of what it adds up
        size = r.grad((6 * y * r.apply(d, positions)).abs(), positions).abs().max() + 12 * y.abs().max() * d.abs().max()
        assert (second - want).abs().max() <= 8 * 2.0 ** -24 * size
        with forward_ad.dual_level():
            out = forward_ad.unpack_dual(r.apply(forward_ad.make_dual(x.detach(), d), positions))
            assert torch.equal(out.primal, y) and torch.equal(out.tangent, r.apply(d, positions))
