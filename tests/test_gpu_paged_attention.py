"""The attention of one token over the paged cache, against a plain
implementation in 64 bits.

Bounds, for unit u of the output's type (2^-11 for float16, 2^-8 for
bfloat16): rounding the result once costs u |out|; scores are float32 sums of
exact products, so each is off by at most 2 D 2^-24 times the sum of the
products' magnitudes, and a weight by that factor twice (its own and the
sum's); 2^-14 of the weighted magnitudes covers the exponentials, the rounding
of a weight to 16 bits or more, and the sums over tokens; 2^-24 is the step
of float16 below its normal range."""
import math

import pytest
import torch

from jasper_b200 import paged
import paged_model

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make(lengths, page_size=16, kv_heads=2, dim=64, dtype=torch.float16, layout="token", seed=0, spare=3,
         layers=1, poison=True):
    """A cache with rows of these lengths, pages in a random order; with
    `poison`, NaN wherever no token lies."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page_size) for n in lengths]
    n_pages, width = sum(held) + spare, max(max(held), 1) + 1
    c = paged.PagedCache.allocate(layers, n_pages, page_size, kv_heads, dim, len(lengths), width, dtype, layout)
    order = torch.randperm(n_pages, generator=g)
    table, at = torch.full((len(lengths), width), -1, dtype=torch.int32), 0
    valid = torch.zeros(n_pages, page_size, dtype=torch.bool)
    for r, n in enumerate(lengths):
        for j in range(held[r]):
            table[r, j] = order[at]
            valid[order[at], :min(page_size, n - j * page_size)] = True
            at += 1
    fill = math.nan if poison else 0.0
    for t in (c.k, c.v):
        x = torch.randn(t.shape, generator=g)
        x[:, ~valid] = fill
        t.copy_(x.to(dtype))
    c.table.copy_(table)
    c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    c.refs[order[:at].cuda()] = 1
    return c


def queries(n, heads, dim, dtype, seed=1, factor=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, dim, generator=g) * factor).to(dtype).cuda()


def check(c, q, out, lse, rows=None, scale=None, window=0, mask=None, layer=0):
    k, v = c.k[layer].cpu(), c.v[layer].cpu()
    table, lengths = c.table.cpu(), c.lengths.cpu().tolist()
    scale = c.head_dim ** -0.5 if scale is None else scale
    u, dim = UNIT[c.dtype], c.head_dim
    out, lse = out.cpu().double(), lse.cpu().double()
    for i in range(q.size(0)):
        r = i if rows is None else rows[i]
        length = lengths[r] if 0 <= r < c.n_rows else 0
        pages = table[r] if 0 <= r < c.n_rows else None
        want, want_lse, weight, reach = paged_model.attention(
            q[i].cpu(), k, v, pages, length, c.page_size, scale, window, None if mask is None else mask[i].tolist())
        score = 2 * dim * 2.0 ** -24 * reach
        bound = u * want.abs() + (2.0 ** -14 + 2 * score) * weight + 2.0 ** -24
        assert ((out[i] - want).abs() <= bound).all(), (i, float(((out[i] - want).abs() / bound).max()))
        none = want_lse == -math.inf
        assert (lse[i][none] == -math.inf).all() and (out[i][none] == 0).all()
        bound = score + 2.0 ** -18 * (1 + want_lse.abs())
        assert ((lse[i] - want_lse).abs() <= bound)[~none].all(), i


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("dim", [8, 64, 80, 128, 256])
def test_types_layouts_and_sizes_of_heads(cuda, dtype, layout, dim):
    c = make([1, 0, 33, 200, 16], dim=dim, dtype=dtype, layout=layout)
    q = queries(5, 6, dim, dtype)
    out, lse = c.attend(0, q, return_lse=True)
    check(c, q, out, lse)


@pytest.mark.parametrize("kv_heads,group", [(1, 1), (4, 1), (2, 2), (1, 5), (2, 7), (1, 8), (3, 16), (1, 17), (2, 33)])
def test_groups_of_query_heads(cuda, kv_heads, group):
    c = make([70, 5, 129], kv_heads=kv_heads, dim=64)
    q = queries(3, kv_heads * group, 64, torch.float16)
    out, lse = c.attend(0, q, return_lse=True)
    check(c, q, out, lse)


@pytest.mark.parametrize("page_size", [1, 3, 8, 16, 24, 64, 100, 256])
def test_pages_that_end_inside_a_tile(cuda, page_size):
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 300]
    c = make(lengths, page_size=page_size, dtype=torch.bfloat16)
    q = queries(len(lengths), 4, 64, torch.bfloat16)
    out, lse = c.attend(0, q, return_lse=True)
    check(c, q, out, lse)


@pytest.mark.parametrize("lengths", [[5000], [40_000, 3], [1, 0, 2500, 0, 1, 9000, 17], [700] * 60])
def test_long_and_ragged_rows(cuda, lengths):
    c = make(lengths, kv_heads=1, dim=64, spare=40)
    q = queries(len(lengths), 4, 64, torch.float16, factor=3.0)
    out, lse = c.attend(0, q, return_lse=True)
    check(c, q, out, lse)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [40, 64, 80, 128, 256])
@pytest.mark.parametrize("group,page_size", [(1, 16), (4, 7), (16, 16), (19, 24)])
def test_rows_in_several_parts(cuda, dtype, dim, group, page_size):
    """Long enough that a row's head is shared out, with its neighbours' ends
    in the same parts."""
    lengths = [13_000, 5, 0, 2900, 17]
    c = make(lengths, kv_heads=1, dim=dim, dtype=dtype, page_size=page_size, layout="head" if group == 4 else "token")
    q = queries(len(lengths), group, dim, dtype)
    g = torch.Generator().manual_seed(3)
    mask = torch.rand(len(lengths), 13_000, generator=g) < 0.7
    mask[0, 4000:6000] = False                       # whole parts with nothing to attend to
    out, lse = c.attend(0, q, mask=mask.cuda(), return_lse=True)
    check(c, q, out, lse, mask=mask)
    out, lse = c.attend(0, q, window=3001, return_lse=True)
    check(c, q, out, lse, window=3001)


def test_more_rows_and_heads_than_workers(cuda):
    """2800 rows' heads, one row much longer than the others."""
    lengths = [20 + (37 * i) % 90 for i in range(700)]
    lengths[333], lengths[334], lengths[699] = 9000, 0, 1500
    c = make(lengths, kv_heads=4, dim=64, page_size=16)
    q = queries(len(lengths), 8, 64, torch.float16)
    out, lse = c.attend(0, q, return_lse=True)
    check(c, q, out, lse)


@pytest.mark.parametrize("rows", [1, 8, 9, 16, 17, 37, 38, 74, 75])
def test_few_rows_in_clusters(cuda, rows):
    """Clusters of 8, 4, 2 and 1 blocks."""
    lengths = [(61 * i) % 180 for i in range(rows)]
    lengths[-1] = 900
    c = make(lengths, kv_heads=2, dim=64, dtype=torch.bfloat16)
    q = queries(rows, 6, 64, torch.bfloat16)
    out, lse = c.attend(0, q, return_lse=True)
    check(c, q, out, lse)


@pytest.mark.parametrize("rows,longest", [(75, 700), (148, 600), (149, 300), (296, 150), (297, 180), (600, 90)])
@pytest.mark.parametrize("dim,group", [(64, 3), (128, 16), (256, 2), (96, 9)])
def test_rows_that_share_blocks(cuda, rows, longest, dim, group):
    """All, four, two or one of a block's warps to a row's head; some rows are empty."""
    lengths = [(53 * i) % (longest + 1) for i in range(rows)]
    lengths[0] = longest
    c = make(lengths, kv_heads=1, dim=dim, page_size=32, dtype=torch.bfloat16)
    q = queries(rows, group, dim, torch.bfloat16)
    out, lse = c.attend(0, q, return_lse=True)
    check(c, q, out, lse)


@pytest.mark.parametrize("kv_heads", [1, 2])
def test_more_queries_than_a_block_lists(cuda, kv_heads):
    """Over 1024 rows of very different lengths, named in another order."""
    lengths = [(7 * i) % 50 for i in range(1100)]
    lengths[700], lengths[3], lengths[1099] = 3000, 700, 260
    c = make(lengths, kv_heads=kv_heads, dim=64, page_size=16)
    rows = torch.randperm(1100, generator=torch.Generator().manual_seed(11)).tolist() + [700, -5, 3]
    q = queries(len(rows), 2 * kv_heads, 64, torch.float16)
    out, lse = c.attend(0, q, torch.tensor(rows, dtype=torch.int32, device="cuda"), return_lse=True)
    check(c, q, out, lse, rows=rows)


def test_many_short_rows(cuda):
    lengths = [(7 * i) % 50 for i in range(1100)]
    c = make(lengths, kv_heads=1, dim=8, page_size=8)
    q = queries(len(lengths), 2, 8, torch.float16)
    out, lse = c.attend(0, q, return_lse=True)
    check(c, q, out, lse)


@pytest.mark.parametrize("window", [1, 5, 16, 40, 1000])
def test_window(cuda, window):
    c = make([1, 40, 41, 200, 0], dim=64)
    q = queries(5, 4, 64, torch.float16)
    out, lse = c.attend(0, q, window=window, return_lse=True)
    check(c, q, out, lse, window=window)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 65504.0])
def test_masked_tokens_may_hold_anything(cuda, value):
    lengths = [64, 50, 300, 17]
    c = make(lengths, dim=64)
    g = torch.Generator().manual_seed(7)
    mask = torch.rand(4, 250, generator=g) < 0.5  # covers part of the longest row
    mask[1] = False                               # leaves row 1 empty
    table = c.table.cpu()
    for r, n in enumerate(lengths):
        for t in range(n):
            if t < 250 and not mask[r, t]:
                c.k[0, table[r, t // 16], t % 16] = value
                c.v[0, table[r, t // 16], t % 16] = value
    q = queries(4, 4, 64, torch.float16)
    out, lse = c.attend(0, q, mask=mask.cuda(), return_lse=True)
    check(c, q, out, lse, mask=mask)
    assert (out[1] == 0).all()
    wide = torch.zeros(4, 777, dtype=torch.bool, device="cuda")[:, ::3][:, :250]  # strided: copied by the call
    wide[:] = mask.cuda()
    again = c.attend(0, q, mask=wide)
    assert torch.equal(out, again)
    one = mask[:1].expand(4, 250)                  # one mask for all rows
    out, lse = c.attend(0, q[:1].expand(4, 4, 64), torch.zeros(4, dtype=torch.int32, device="cuda"),
                        mask=one.cuda(), return_lse=True)
    assert all(torch.equal(out[0], out[i]) for i in range(4))


@pytest.mark.parametrize("lengths", [[40], [900], [20_000, 3]])
def test_nan_is_not_hidden(cuda, lengths):
    """NaN in a query, or in a key or value that is attended to, comes out; in
    the other heads and rows it does not."""
    c = make(lengths, kv_heads=2, dim=64, poison=False)
    q = queries(len(lengths), 4, 64, torch.float16)
    clean, clean_lse = c.attend(0, q, return_lse=True)
    bad = q.clone()
    bad[0, 1, 5] = math.nan
    out, lse = c.attend(0, bad, return_lse=True)
    assert out[0, 1].isnan().all() and lse[0, 1].isnan()
    keep = torch.ones_like(lse, dtype=torch.bool)
    keep[0, 1] = False
    assert torch.equal(out[keep], clean[keep]) and torch.equal(lse[keep], clean_lse[keep])
    page = c.table[0, (lengths[0] - 1) // 16].long()
    c.v[0, page, (lengths[0] - 1) % 16, 1, 7] = math.nan
    out, lse = c.attend(0, q, return_lse=True)
    assert out[0, 2:, 7].isnan().all() and torch.equal(lse, clean_lse)
    out[0, 2:, 7] = clean[0, 2:, 7]
    assert torch.equal(out, clean)
    c.k[0, page, (lengths[0] - 1) % 16, 0, 3] = math.inf
    out, lse = c.attend(0, q.abs(), return_lse=True)
    assert out[0, :2].isnan().all() and lse[0, :2].isnan().all()


def test_pages_that_are_not_there(cuda):
    c = make([100, 64, 48, 200], dim=64)
    c.table[0, 2] = -1
    c.table[1, :] = -1            # a row of absent pages
    c.table[2, 0] = 10 ** 6       # a number out of range: not there either
    c.table[3, 3:9] = -1
    q = queries(4, 4, 64, torch.float16)
    out, lse = c.attend(0, q, return_lse=True)
    c.table[2, 0] = -1
    check(c, q, out, lse)
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()


def test_rows_named_in_any_order(cuda):
    c = make([10, 90, 33], dim=64)
    rows = [2, 2, 0, -1, 1, 3, 0]
    q = queries(len(rows), 4, 64, torch.float16)
    out, lse = c.attend(0, q, torch.tensor(rows, dtype=torch.int32, device="cuda"), return_lse=True)
    check(c, q, out, lse, rows=rows)


def test_scores_far_apart_and_far_from_zero(cuda):
    """The running maximum moves late, and scores of +-1000 neither overflow
    nor lose the sum."""
    c = make([400], kv_heads=1, dim=64, poison=False)
    rising = torch.linspace(-8, 8, 400)[:, None] * torch.ones(64) / 8
    table = c.table.cpu()
    for t in range(400):
        c.k[0, table[0, t // 16], t % 16, 0] = rising[t].half().cuda()
    q = torch.ones(1, 2, 64, dtype=torch.float16, device="cuda") * 125
    q[:, 1] *= -1
    out, lse = c.attend(0, q, return_lse=True)
    check(c, q, out, lse)
    assert float(lse.abs().max()) > 900


def test_scale_layers_and_strides(cuda):
    c = make([77, 130], dim=64, layers=3)
    base = torch.randn(2, 11, 3, 64, generator=torch.Generator().manual_seed(5)).half().cuda()
    q = base[:, 1:9, 1]                           # strided rows and heads
    for layer in (0, 2):
        store = torch.zeros(2, 8, 128, dtype=torch.float16, device="cuda")
        out, lse = c.attend(layer, q, scale=0.3, return_lse=True, out=store[..., 64:])
        check(c, q, out, lse, scale=0.3, layer=layer)
        assert (store[..., :64] == 0).all()
    odd = torch.empty(2 * 8 * 64 + 1, dtype=torch.float16, device="cuda")[1:].view(2, 8, 64)
    odd.copy_(q)                                   # not on 16 bytes: copied by the call
    assert torch.equal(c.attend(0, odd), c.attend(0, q))


def test_zero_scale_is_the_mean(cuda):
    c = make([50], kv_heads=1, dim=64)
    out, lse = c.attend(0, queries(1, 1, 64, torch.float16), scale=0.0, return_lse=True)
    check(c, queries(1, 1, 64, torch.float16), out, lse, scale=0.0)


def test_offsets_past_32_bits(cuda):
    """A pool of over 2^32 bytes, keys and values each, read at both ends."""
    ps, heads, dim = 64, 8, 128
    n_pages = (2 ** 31 + 2 ** 28) // (ps * heads * dim)
    k, v = (torch.empty(1, n_pages, ps, heads, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(3)
    pages = [n_pages - 1, 0, n_pages - 7]
    for p in pages:
        for t in (k, v):
            t[0, p] = torch.randn(ps, heads, dim, generator=g).half().cuda()
    table = torch.tensor([pages], dtype=torch.int32, device="cuda")
    c = paged.PagedCache(k, v, table, torch.tensor([150], dtype=torch.int32, device="cuda"),
                         torch.zeros(n_pages, dtype=torch.int32, device="cuda"))
    q = queries(1, 8, dim, torch.float16)
    out, lse = c.attend(0, q, return_lse=True)
    c.refs[pages] = 1
    new = torch.randn(1, heads, dim, generator=g).half().cuda()
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.append(0, new, new, one, one + 149)
    assert torch.equal(k[0, pages[2], 149 - 128], new[0])
    c.copy_pages(torch.tensor([pages[0]], dtype=torch.int32, device="cuda"), one + 5)
    assert torch.equal(k[0, 5], k[0, pages[0]]) and torch.equal(v[0, 5], v[0, pages[0]])
    k[0, pages[2], 149 - 128], v[0, pages[2], 149 - 128] = math.nan, math.nan
    small_k, small_v = k[:, pages].cpu(), v[:, pages].cpu()
    want, want_lse, weight, reach = paged_model.attention(q[0].cpu(), small_k[0], small_v[0], torch.arange(3), 149,
                                                          ps, dim ** -0.5)
    got, got_lse = c.attend(0, q, return_lse=True)      # row 0 again, one token shorter
    c.lengths.fill_(149)
    got, got_lse = c.attend(0, q, return_lse=True)
    bound = 2.0 ** -11 * want.abs() + (2.0 ** -14 + 4 * dim * 2.0 ** -24 * reach) * weight + 2.0 ** -24
    assert ((got[0].cpu().double() - want).abs() <= bound).all()
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


def test_same_bits_on_every_call(cuda):
    """Parts are joined in order, not as they arrive."""
    c = make([30_000, 10, 5000], kv_heads=1, dim=128, dtype=torch.bfloat16)
    q = queries(3, 8, 128, torch.bfloat16)
    first = c.attend(0, q, return_lse=True)
    for _ in range(20):
        again = c.attend(0, q, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_other_streams_and_graphs(cuda):
    c = make([3000, 200], dim=64)
    q = queries(2, 4, 64, torch.float16)
    want = c.attend(0, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.attend(0, q)
        again = c.attend(0, q)
    other = c.attend(0, q)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(again, want) and torch.equal(other, want)
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.attend(0, q, out=out)
    for lengths in ([3000, 200], [17, 0], [2999, 1]):
        c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, c.attend(0, q))


def test_refusals(cuda):
    c = make([10, 20], dim=64, kv_heads=2)
    q = queries(2, 4, 64, torch.float16)
    for bad in (q.float(), q[:, :3], q[..., :32], q[0], q.cpu(), queries(3, 4, 64, torch.float16)):
        with pytest.raises(ValueError):
            c.attend(0, bad)
    for kw in ({"window": -1}, {"mask": torch.ones(2, 9)}, {"mask": torch.ones(3, 9, dtype=torch.bool, device="cuda")},
               {"rows": torch.zeros(2, dtype=torch.int64, device="cuda")},
               {"rows": torch.zeros(1, dtype=torch.int32, device="cuda")}, {"out": torch.empty(2, 4, 64)},
               {"scale": math.inf}):
        with pytest.raises(ValueError):
            c.attend(0, q, **kw)
    for layer in (1, -1):
        with pytest.raises(ValueError, match="layer"):
            c.attend(layer, q)
    assert c.attend(0, q[:0]).shape == (0, 4, 64)
