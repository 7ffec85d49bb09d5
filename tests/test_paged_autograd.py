"""Derivatives through rotary positions, of any order and in both modes.  The
kernel is stood in for by the same turn in 64 bits, which like it returns
tensors without a graph, so that no GPU is needed."""
import pytest
import torch
from torch.autograd import forward_ad

from jasper_b200 import paged
import paged_model


class StandIn:
    @staticmethod
    def rotary(x, positions, out, inverse, freq, head_dim, rot_dim, scale, interleaved):
        assert out is None
        flat = x.detach().reshape(-1, *x.shape[-2:])
        theta = [f / 2.0 ** 64 * 2 * torch.pi for f in freq.tolist()]
        where = positions.expand(x.shape[:-2]).reshape(-1)
        return paged_model.turned(flat, where, theta, rot_dim, "interleaved" if interleaved else "half", scale,
                                  -1 if inverse else 1).view(x.shape)


@pytest.fixture
def rotary(monkeypatch):
    monkeypatch.setattr(paged._lib, "paged_module", lambda: StandIn)
    return paged.Rotary(6, 4, layout="interleaved", scaling="yarn", factor=4.0, trained_length=64, device="cpu")


def inputs(*shape):
    g = torch.Generator().manual_seed(3)
    return torch.randn(*shape, dtype=torch.float64, generator=g).requires_grad_(), torch.arange(shape[-3]) * 3 + 1


@pytest.mark.parametrize("shape", [(3, 2, 6), (2, 3, 1, 6)])
def test_derivatives_against_differences(rotary, shape):
    x, p = inputs(*shape)
    for turn in (rotary.apply, rotary.grad):
        assert torch.autograd.gradcheck(lambda t: turn(t, p), x, check_forward_ad=True)
        assert torch.autograd.gradgradcheck(lambda t: turn(t, p) ** 3, x, check_fwd_over_rev=True)


def test_second_derivatives_beside_another_term(rotary):
    """sum(turn(x)^3) + sum(x^2): the Hessian is R^T diag(6 y) R + 2."""
    x, p = inputs(3, 2, 6)
    d = torch.randn(3, 2, 6, dtype=torch.float64, generator=torch.Generator().manual_seed(4))
    f = (rotary.apply(x, p) ** 3).sum() + (x ** 2).sum()
    g, = torch.autograd.grad(f, x, create_graph=True)
    h, = torch.autograd.grad((g * d).sum(), x)
    with torch.no_grad():
        want = rotary.grad(6 * rotary.apply(x, p) * rotary.apply(d, p), p) + 2 * d
    assert torch.allclose(h, want, rtol=1e-12, atol=1e-12)


def test_forward_mode_without_a_gradient(rotary):
    x, p = inputs(3, 2, 6)
    d = torch.ones(3, 2, 6, dtype=torch.float64)
    with torch.no_grad(), forward_ad.dual_level():
        y = rotary.apply(forward_ad.make_dual(x.detach(), d), p)
        assert torch.equal(forward_ad.unpack_dual(y).tangent, rotary.apply(d, p))


def test_function_transforms(rotary):
    x, p = inputs(3, 2, 6)
    d = torch.ones(3, 2, 6, dtype=torch.float64)
    loss = lambda t: (rotary.apply(t, p) ** 3).sum()
    x = x.detach()
    assert torch.allclose(torch.func.grad(loss)(x), rotary.grad(3 * rotary.apply(x, p) ** 2, p), rtol=1e-12)
    hv = torch.func.jvp(torch.func.grad(loss), (x,), (d,))[1]
    assert torch.allclose(hv, rotary.grad(6 * rotary.apply(x, p) * rotary.apply(d, p), p), rtol=1e-12)
