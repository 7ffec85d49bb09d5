"""What autograd sees of the paged cache's calls."""
import pytest
import torch
from torch.autograd import forward_ad

from jasper_b200 import paged

pytestmark = pytest.mark.gpu


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make():
    c = paged.PagedCache.allocate(1, 6, 4, 1, 8, 2, 3)
    c.extend(ints(0, 1), ints(5, 3))
    c.k.normal_(), c.v.normal_()
    return c, paged.Rotary(8)


def calls_into(c, r):
    """Each call that takes an output, as a function of it."""
    q = torch.randn(2, 2, 8, device="cuda").half()
    kv = torch.randn(2, 1, 8, device="cuda").half()
    return (lambda out: r.apply(q, ints(0, 3), out=out), lambda out: r.grad(q, ints(0, 3), out=out),
            lambda out: c.append(0, kv, kv, ints(0, 1), q=q, rotary=r, q_out=out), lambda out: c.attend(0, q, out=out))


def test_outputs_are_seen_to_change(cuda):
    c, r = make()
    for call in calls_into(c, r):
        out = torch.ones(2, 2, 8, device="cuda").half()
        w = torch.ones(2, 2, 8, device="cuda", requires_grad=True)
        y = (w * out).sum()                       # saves out
        version = out._version
        assert call(out) is out
        assert out._version > version
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        with torch.inference_mode():              # tensors without versions
            call(torch.empty(2, 2, 8, device="cuda").half())


def test_outputs_that_require_a_gradient(cuda):
    c, r = make()
    for call in calls_into(c, r):
        leaf = torch.zeros(2, 2, 8, device="cuda").half().requires_grad_()
        for out in (leaf, leaf * 1):
            with pytest.raises(ValueError, match="gradient"):
                call(out)
            with torch.no_grad():
                call(out)
        with forward_ad.dual_level(), pytest.raises(ValueError, match="gradient"):
            call(forward_ad.make_dual(leaf.detach(), torch.ones_like(leaf)))


def test_a_backward_pass_through_the_cache_raises(cuda):
    c, r = make()
    q = torch.randn(2, 2, 8, device="cuda").half().requires_grad_()
    kv = torch.randn(2, 1, 8, device="cuda").half()
    for call in (lambda: c.append(0, kv, kv, ints(0, 1), q=q, rotary=r), lambda: c.attend(0, q),
                 lambda: c.attend(0, q, return_lse=True)[0], lambda: c.attend(0, q, return_lse=True)[1],
                 lambda: c.attend(0, (q * 2).transpose(0, 1)[:, :1].contiguous().transpose(0, 1))):
        out = call()
        with pytest.raises(RuntimeError, match="not implemented"):
            (out.float().sum() + (q.float() ** 2).sum()).backward()
        with torch.no_grad():
            assert not call().requires_grad
        q.requires_grad_(False)
        assert torch.equal(call(), out) and not call().requires_grad
        with forward_ad.dual_level():
            plain, q = q, forward_ad.make_dual(q, torch.ones_like(q))
            with pytest.raises(ValueError, match="forward-mode"):
                call()
            q = plain
        q.requires_grad_()
