"""Values near the end of bfloat16's range: the result is their weighted mean,
so as finite as they are."""
import pytest
import torch

from test_gpu_paged_attention import make, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [[1], [40], [17, 300], [9000, 40], [50] * 300])
@pytest.mark.parametrize("log2", [110, 120, 126])
def test_large_values_in_bfloat16(cuda, lengths, log2):
    """A power of two in every value is that power in every result: bit for bit
    what the same values scaled down give."""
    c = make(lengths, kv_heads=2, dim=64, dtype=torch.bfloat16, poison=False)
    c.v.clamp_(-1, 1)
    q = queries(len(lengths), 4, 64, torch.bfloat16)
    want = c.attend(0, q)
    c.v.mul_(2.0 ** log2)
    out = c.attend(0, q)
    assert out.isfinite().all()
    assert torch.equal(out.float() * 2.0 ** -log2, want.float())
