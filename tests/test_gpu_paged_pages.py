"""The paged cache's page operations against a plain model of the cache, bit
for bit: tables, lengths, holders, keys, values and the status word."""
import random

import numpy as np
import pytest
import torch

from jasper_b200 import _lib, paged
import paged_model

pytestmark = pytest.mark.gpu


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make(n_pages=40, page_size=4, rows=12, width=8, layers=2, kv_heads=2, dim=16, dtype=torch.float16,
         layout="token", seed=0):
    c = paged.PagedCache.allocate(layers, n_pages, page_size, kv_heads, dim, rows, width, dtype, layout)
    g = torch.Generator().manual_seed(seed)
    for t in (c.k, c.v):
        t.copy_(torch.randn(t.shape, generator=g).to(dtype))
    return c, paged_model.PlainCache(c)


def both(c, m, name, *args):
    r = getattr(c, name)(*(torch.as_tensor(np.ascontiguousarray(a, np.int32)).cuda() for a in args))
    want = getattr(m, name)(*(np.asarray(a, np.int32) for a in args))
    m.check_against(c)
    return r, want


@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_one_of_each(cuda, layout, dtype):
    c, m = make(layout=layout, dtype=dtype)
    both(c, m, "extend", [3, 0, 7], [9, 4, 1])
    both(c, m, "extend", [0, 3], [1, 0])
    both(c, m, "fork", [3, 3, 0, 7], [1, 2, 4, 5])
    both(c, m, "free", [3, 9])
    both(c, m, "adopt", [8, 9], [[6, -1, 0], [1, 1, 2]])
    r, want = both(c, m, "compact")
    np.testing.assert_array_equal(r.cpu().numpy(), want)
    both(c, m, "copy_pages", [0, 3], [20, 39])
    c.check()


@pytest.mark.parametrize("page_size,n_pages,rows,width", [(1, 30, 10, 9), (5, 70, 20, 6), (16, 12, 6, 3)])
def test_any_order_of_calls(cuda, page_size, n_pages, rows, width):
    """Random calls, sane and not, on small pools."""
    rng = random.Random(page_size)
    c, m = make(n_pages, page_size, rows, width, layers=1, kv_heads=1, dim=8)
    for step in range(120):
        some = [rng.randrange(-1, rows + 1) for _ in range(rng.randint(1, rows))]
        kind = rng.choice(["extend", "extend", "fork", "free", "adopt", "compact", "copy_pages"])
        if kind == "extend":
            both(c, m, kind, some, [rng.choice([0, 1, 1, rng.randint(-1, 2 * page_size * width // 3)]) for _ in some])
        elif kind == "fork":
            both(c, m, kind, some, [rng.randrange(-1, rows + 1) for _ in some])
        elif kind == "free":
            both(c, m, kind, some[:max(1, rows // 4)])
        elif kind == "adopt":
            w = rng.randint(1, width)
            pages = [[rng.choice([-1, rng.randrange(n_pages), n_pages + 3]) for _ in range(w)] for _ in some]
            both(c, m, kind, some, pages, [rng.randint(-1, w * page_size + 1) for _ in some])
        elif kind == "compact":
            r, want = both(c, m, kind)
            np.testing.assert_array_equal(r.cpu().numpy(), want)
        else:
            two = rng.sample(range(-1, n_pages + 1), 6)
            both(c, m, kind, two[:3], two[3:])
    with pytest.raises(_lib.JasperError) as e:
        c.check()
    assert ("free page" in str(e.value)) == bool(m.status & paged.EXHAUSTED)
    assert ("a row is" in str(e.value)) == bool(m.status & paged.BAD_ROW)
    assert ("a token" in str(e.value)) == bool(m.status & paged.BAD_TOKEN)
    c.check()  # cleared


def test_rows_are_served_in_order(cuda):
    c, m = make(n_pages=5, page_size=4, rows=6, width=8)
    both(c, m, "extend", [5, 2, 0, 1, 3], [8, 4, 12, 4, 0])  # 2 + 1, then 3 that are not there: 1 goes without too
    assert c.lengths.tolist() == [0, 0, 4, 0, 0, 8]
    both(c, m, "extend", [0, 1], [8, 1])
    both(c, m, "extend", [2], [1])
    both(c, m, "free", [0])
    both(c, m, "extend", [2], [5])
    assert sorted(c.table[c.table >= 0].tolist()) == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("n_pages", [1, 1023, 1024, 1025, 9000, 100_003, 300_000])
def test_pools_of_any_size(cuda, n_pages):
    """Free pages far apart, behind runs of held ones."""
    g = torch.Generator().manual_seed(n_pages)
    c = paged.PagedCache.allocate(1, n_pages, 2, 1, 8, 300, 4000)
    held = torch.rand(n_pages, generator=g) < 0.9
    held[: n_pages // 2] = True
    c.refs.copy_(held.int() * 3)
    free = torch.where(~held)[0].tolist()
    rows = torch.randperm(300, generator=g).int()
    tokens = torch.randint(0, 8, (300,), generator=g).int()
    tokens[5] = 2 * min(3999, len(free) // 3)
    c.extend(rows.cuda(), tokens.cuda())
    table, lengths = c.table.cpu(), c.lengths.cpu()
    upto, taken = 0, []
    for r, n in zip(rows.tolist(), tokens.tolist()):
        need = -(-n // 2)
        upto += need
        if need and upto > len(free):
            assert int(lengths[r]) == 0 and (table[r] == -1).all()
            continue
        assert int(lengths[r]) == n and table[r, :need].tolist() == free[upto - need:upto]
        taken += free[upto - need:upto]
    want = held.int() * 3
    want[taken] = 1
    assert torch.equal(c.refs.cpu(), want)
    remap = c.compact().cpu()
    live = int((want > 0).sum())
    assert (c.refs[:live] > 0).all() and (c.refs[live:] == 0).all()
    stay = (want > 0) & (torch.arange(n_pages) < live)
    assert torch.equal(remap[stay], torch.arange(n_pages).int()[stay])
    moved = torch.where((want > 0) & (torch.arange(n_pages) >= live))[0]
    holes = torch.where((want == 0) & (torch.arange(n_pages) < live))[0]
    assert torch.equal(remap[moved], holes.int())
    assert torch.equal(c.refs.cpu()[holes], want[moved])
    assert torch.equal(c.table.cpu()[table >= 0], remap[table[table >= 0].long()])


@pytest.mark.parametrize("rows,named,n_pages", [(9000, 1500, 9000), (3000, 2900, 5000), (12_000, 5000, 40_000)])
def test_many_rows(cuda, rows, named, n_pages):
    """More rows, in the table and in a call, than a block's shared memory keeps."""
    rng = np.random.default_rng(rows)
    c, m = make(n_pages, 2, rows, 9, layers=1, kv_heads=1, dim=8)
    order = rng.permutation(rows)[:named].astype(np.int32)
    order[5] = order[900]                                   # named twice: the first time counts
    both(c, m, "extend", order, rng.integers(0, 9, named))
    both(c, m, "extend", order[::-1], rng.integers(0, 3, named))
    children = np.setdiff1d(np.arange(rows), order)
    children = rng.permutation(children)[:min(named // 2, len(children))]
    parents = rng.choice(order, len(children))
    both(c, m, "fork", parents, children)
    both(c, m, "free", order[:named // 3])
    r, want = both(c, m, "compact")
    np.testing.assert_array_equal(r.cpu().numpy(), want)
    both(c, m, "adopt", order[:named // 3], rng.integers(-1, n_pages, (named // 3, 4)))


@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("kv_heads,dim,page_size", [(1, 8, 16), (3, 40, 7), (8, 128, 16)])
def test_fork_copies_the_filled_tokens_only(cuda, layout, kv_heads, dim, page_size):
    c, m = make(60, page_size, 20, 4, layers=3, kv_heads=kv_heads, dim=dim, layout=layout)
    both(c, m, "extend", range(6), [1, page_size - 1, page_size, page_size + 1, 2 * page_size + 3, 0])
    both(c, m, "fork", [0, 1, 2, 3, 4, 5, 4, 4], [10, 11, 12, 13, 14, 15, 16, 17])
    assert int(c.refs[c.table[4, 0]]) == 4 and int(c.refs[c.table[4, 2]]) == 1
    # a child goes on alone
    before = c.k[:, c.table[4, 2].long()].clone()
    new = torch.full((1, kv_heads, dim), 7.0, dtype=torch.float16, device="cuda")
    c.append(1, new, new, ints(14), ints(2 * page_size + 2))
    assert torch.equal(c.k[:, c.table[4, 2].long()], before)


def test_a_cache_inside_larger_tensors(cuda):
    """Strides of its own for layers, pages, tokens, heads and the table."""
    g = torch.Generator().manual_seed(9)
    big = torch.randn(2, 3, 33, 6, 5, 32, generator=g).half().cuda()
    k, v = big[0, :2, 1:31, 1:5, :3, 8:24], big[1, :2, 1:31, 1:5, :3, 8:24]
    table = torch.full((9, 20), -1, dtype=torch.int32, device="cuda")
    untouched = big.clone()
    c = paged.PagedCache(k, v, table[:, 3:9], torch.zeros(9, dtype=torch.int32, device="cuda"),
                         torch.zeros(30, dtype=torch.int32, device="cuda"))
    m = paged_model.PlainCache(c)
    both(c, m, "extend", [0, 1, 2], [24, 9, 3])
    both(c, m, "fork", [1, 2], [3, 4])
    both(c, m, "free", [0])
    both(c, m, "compact")
    both(c, m, "copy_pages", [1], [29])
    untouched[:, :2, 1:31, 1:5, :3, 8:24] = big[:, :2, 1:31, 1:5, :3, 8:24]
    assert torch.equal(big, untouched)
    assert (table[:, :3] == -1).all() and (table[:, 9:] == -1).all()


def test_graphs_and_streams(cuda):
    c, m = make()
    rows, tokens = ints(1, 2), ints(5, 3)
    c.extend(rows, tokens)
    m.extend([1, 2], [5, 3])
    graph = torch.cuda.CUDAGraph()
    children = ints(4, 5)
    with torch.cuda.graph(graph):
        c.free(children)
        c.fork(rows, children)
        c.compact()
    for _ in range(3):
        graph.replay()
        m.free([4, 5])
        m.fork([1, 2], [4, 5])
        m.compact()
        m.check_against(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.free(rows)
        c.extend(children, tokens)
    side.synchronize()
    m.free([1, 2])
    m.extend([4, 5], [5, 3])
    m.check_against(c)


def test_refusals(cuda):
    c, _ = make()
    for call in (lambda: c.extend(ints(1), ints(1, 2)), lambda: c.extend(ints(1).long(), ints(1)),
                 lambda: c.extend(ints(1).cpu(), ints(1)), lambda: c.free(torch.zeros(1, 1)),
                 lambda: c.fork(ints(1, 2), ints(3)), lambda: c.adopt(ints(1), ints(1)),
                 lambda: c.adopt(ints(1), torch.zeros(1, 9, dtype=torch.int32, device="cuda")),
                 lambda: c.adopt(ints(1), torch.zeros(2, 2, dtype=torch.int32, device="cuda")),
                 lambda: c.copy_pages(ints(1), ints(1, 2))):
        with pytest.raises(ValueError):
            call()
    empty = ints()
    c.extend(empty, empty), c.fork(empty, empty), c.free(empty), c.copy_pages(empty, empty)
    c.check()
    k, v, rest = c.k, c.v, (c.table, c.lengths, c.refs)
    for k1, v1, rest1 in ((k, v[:1], rest), (k.float(), v.float(), rest), (k, v.transpose(2, 3), rest),
                          (k.cpu(), v.cpu(), rest), (k, v, (c.table.long(), c.lengths, c.refs)),
                          (k, v, (c.table, c.lengths[:3], c.refs)), (k, v, (c.table, c.lengths, c.refs[:3])),
                          (k, v, (c.table, c.lengths.cpu(), c.refs))):
        with pytest.raises(ValueError):
            paged.PagedCache(k1, v1, *rest1)
    with pytest.raises(ValueError):
        paged.PagedCache.allocate(1, 4, 4, 1, 8, 2, 2, layout="page")
    odd = paged.PagedCache.allocate(1, 4, 4, 1, 12, 2, 2)  # 12 elements: no multiple of 16 bytes
    with pytest.raises(ValueError, match="head_dim"):
        odd.free(ints(0))
