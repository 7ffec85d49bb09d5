"""Infinite values that are attended to come out of the attention as such: every
weight is positive, so sum p v is infinite where v is, and NaN where values of
both signs or NaN meet.  All other elements keep their bits."""
import math

import pytest
import torch

from test_gpu_paged_attention import make, queries

pytestmark = pytest.mark.gpu


def place(c, row, token):
    return int(c.table[row, token // c.page_size]), token % c.page_size


def check(c, q, put, seen=lambda row, token: True, **kw):
    """`put`: (row, token, kv head, element, value).  `seen` says which of these
    tokens are attended to."""
    clean, clean_lse = c.attend(0, q, return_lse=True, **kw)
    assert clean.isfinite().all()
    add = torch.zeros(c.n_rows, c.n_kv_heads, c.head_dim)   # what infinities add to each sum of values
    for row, token, head, d, value in put:
        page, slot = place(c, row, token)
        c.v[0, page, slot, head, d] = value
        if seen(row, token):
            add[row, head, d] += value
    want = clean + add.to(c.dtype).cuda().repeat_interleave(q.size(1) // c.n_kv_heads, 1)
    out, lse = c.attend(0, q, return_lse=True, **kw)
    assert torch.equal(lse, clean_lse)
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))
    assert not want.isfinite().all() or not any(seen(row, token) for row, token, *_ in put)


def some(c, lengths, seed, heads, n=24):
    g = torch.Generator().manual_seed(seed)
    def r(k):
        return int(torch.randint(0, k, (1,), generator=g))
    held = [i for i, m in enumerate(lengths) if m]
    put = [(i := held[r(len(held))], r(lengths[i]), r(heads), r(c.head_dim), [math.inf, -math.inf][r(2)])
           for _ in range(n)]
    longest = max(range(len(lengths)), key=lengths.__getitem__)
    put += [(longest, 0, 0, 3, math.inf), (longest, lengths[longest] - 1, 0, 3, -math.inf),      # both: NaN
            (longest, lengths[longest] // 2, 0, 5, math.inf), (longest, 1 % lengths[longest], 0, 5, math.inf),
            (longest, lengths[longest] // 3, heads - 1, 6, math.nan)]
    return put


# clusters, shared blocks, equal parts (some rows in many parts, some in one), more rows' heads than
# workers, and more queries than a block lists
@pytest.mark.parametrize("lengths", [[40], [900], [17, 0, 300], [53 * i % 150 for i in range(200)],
                                     [20_000, 3], [1, 0, 2500, 0, 1, 9000, 17],
                                     [30 + 7 * i % 50 for i in range(900)] + [9000],
                                     [7 * i % 50 for i in range(1100)] + [3000]], ids=lambda n: f"{len(n)}x{max(n)}")
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_infinite_values(cuda, lengths, dtype):
    c = make(lengths, kv_heads=2, dim=64, dtype=dtype, poison=False)
    q = queries(len(lengths), 8, 64, dtype, factor=3.0)
    check(c, q, some(c, lengths, 1, 2))


@pytest.mark.parametrize("dim", [8, 40, 80, 96, 128, 256])
@pytest.mark.parametrize("group,page_size,layout", [(1, 16, "token"), (5, 7, "head"), (16, 32, "token"), (19, 24, "head")])
def test_heads_groups_and_pages(cuda, dim, group, page_size, layout):
    for lengths in ([70, 0, 33], [6000, 11]):
        c = make(lengths, kv_heads=1, dim=dim, dtype=torch.bfloat16, page_size=page_size, layout=layout, poison=False)
        check(c, queries(len(lengths), group, dim, torch.bfloat16), some(c, lengths, dim, 1))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("length", [64, 700, 20_000])
def test_small_weights(cuda, length, dtype):
    """A weight of e^-200 or less of the largest is zero in float32."""
    c = make([length], kv_heads=1, dim=64, dtype=dtype, poison=False)
    c.k.fill_(0.0)
    for token, k in ((0, 40.0), (length // 2, -40.0), (length - 1, 0.0)):
        page, slot = place(c, 0, token)
        c.k[0, page, slot] = k
    q = torch.ones(1, 3, 64, dtype=dtype, device="cuda")     # scores of 320, -320 and 0
    check(c, q, [(0, length // 2, 0, 9, math.inf), (0, length - 1, 0, 10, -math.inf), (0, 0, 0, 11, math.inf),
                 (0, 1, 0, 12, math.inf), (0, length // 2, 0, 12, -math.inf)])


def test_weights_that_are_exact(cuda):
    """Equal scores: weights are powers of two, without a second half."""
    for length in (1, 2, 16, 64, 5000):
        for dtype in (torch.float16, torch.bfloat16):
            c = make([length], kv_heads=1, dim=64, dtype=dtype, poison=False)
            check(c, torch.zeros(1, 2, 64, dtype=dtype, device="cuda"), [(0, length - 1, 0, 1, -math.inf)])


@pytest.mark.parametrize("lengths", [[64, 300], [9000, 40]])
def test_infinite_values_that_are_not_attended_to(cuda, lengths):
    """Masked, outside the window, or in pages that are not there."""
    g = torch.Generator().manual_seed(2)
    mask = torch.rand(2, 200, generator=g) < 0.5
    for kw, seen in ((dict(mask=mask.cuda()), lambda row, token: token >= 200 or bool(mask[row, token])),
                     (dict(window=21), lambda row, token: token >= lengths[row] - 21)):
        c = make(lengths, dim=64, poison=False)
        check(c, queries(2, 4, 64, torch.float16), some(c, lengths, 5, 2), seen, **kw)
