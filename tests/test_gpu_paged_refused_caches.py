"""Caches outside the kernels' limits can be made, and every call through the
Python boundary refuses them."""
import pytest
import torch

from jasper_b200 import paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv_heads,dim,page_size,message", [(0, 8, 4, "n_kv_heads"), (1, 0, 4, "head_dim"),
                                                            (1, 12, 4, "head_dim"), (1, 264, 4, "head_dim"),
                                                            (1, 8, 0, "page_size")])
def test_every_call_refuses(cuda, kv_heads, dim, page_size, message):
    c = paged.PagedCache.allocate(1, 4, page_size, kv_heads, dim, 2, 2)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv = torch.zeros(1, kv_heads, dim, dtype=torch.float16, device="cuda")
    q = torch.zeros(1, 2, dim, dtype=torch.float16, device="cuda")
    for call in (lambda: c.attend(0, q), lambda: c.attend(0, q[:, :0]), lambda: c.append(0, kv, kv, one),
                 lambda: c.extend(one, one), lambda: c.fork(one, one), lambda: c.free(one),
                 lambda: c.adopt(one, one[None]), lambda: c.compact(), lambda: c.copy_pages(one, one)):
        with pytest.raises(ValueError, match=message):
            call()
