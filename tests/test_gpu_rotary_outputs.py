"""Outputs of the caller's, for batches: any whose batch and tokens can be
walked in one stride."""
import pytest
import torch

from jasper_b200 import paged

pytestmark = pytest.mark.gpu


def test_batches_into_views(cuda):
    r = paged.Rotary(8)
    g = torch.Generator(device="cuda").manual_seed(1)
    big = torch.randn(4, 5, 3, 8, generator=g, device="cuda")
    for view in (lambda t: t, lambda t: t[:, :1], lambda t: t[:, 2:3], lambda t: t[1:2], lambda t: t[1:2, 1:4],
                 lambda t: t[:, :1, 1:2], lambda t: t[::2, 4:], lambda t: t[:, :0], lambda t: t[:0]):
        store = big.clone()
        x = view(big).contiguous()
        positions = torch.arange(x.size(0) * x.size(1), device="cuda").view(x.shape[:2])
        want = r.apply(x, positions)
        out = view(store)
        assert r.apply(x, positions, out=out) is out
        assert torch.equal(out, want)
        out.copy_(x)
        assert torch.equal(store, big)                       # nothing beside it changed
        assert torch.equal(r.apply(out, positions, out=out), want)
    with pytest.raises(ValueError, match="one run"):
        r.apply(big[:, :2], torch.arange(2, device="cuda"), out=big[:, 2:4])
