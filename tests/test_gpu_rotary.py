"""Rotary positions, their gradient, and appending to the paged cache, against
plain implementations in 64 bits.

Bounds: the angle is a float32 of at most half a turn (off by 2^-25 of half a
turn, 1e-7), cosine and sine by two units more (2.4e-7), each product and sum
by one: 6e-7 of |a| + |b| times the factor; theta's own last bit times the
position is in both sides, twice; then the result is rounded to its type
once."""
import pytest
import torch

from jasper_b200 import paged
import paged_model

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SCALING = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
           dict(scaling="yarn", factor=8.0, trained_length=4096)]


def check(got, x, positions, rotary, sign=1):
    want = paged_model.turned(x, positions, rotary.theta, rotary.rot_dim, rotary.layout, rotary.scale, sign)
    reach = paged_model.turned(x.abs(), torch.zeros_like(positions), rotary.theta, rotary.rot_dim, rotary.layout,
                               rotary.scale)
    rot, half = rotary.rot_dim, rotary.rot_dim // 2
    pair = reach.clone()
    a, b = (slice(0, half), slice(half, rot)) if rotary.layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    pair[..., a] = pair[..., b] = reach[..., a] + reach[..., b]
    drift = positions.cpu().double().abs().max() * 2.0 ** -52
    bound = UNIT[x.dtype] * want.abs() + (6e-7 + drift) * pair + 2.0 ** -25
    off = (got.detach().cpu().double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())
    assert torch.equal(got[..., rot:], x[..., rot:])  # what is not rotated is copied


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (64, 32), (80, 20), (96, 6), (5, 2), (256, 256), (20, 20)])
def test_layouts_types_and_parts_of_heads(cuda, dtype, layout, dim, rot):
    r = paged.Rotary(dim, rot, layout=layout)
    g = torch.Generator().manual_seed(dim)
    for tokens, heads in ((1, 1), (37, 3), (2, 19)):
        x = torch.randn(tokens, heads, dim, generator=g).to(dtype).cuda()
        positions = torch.randint(0, 5000, (tokens,), generator=g).cuda()
        check(r.apply(x, positions), x, positions, r)
        check(r.grad(x, positions.int()), x, positions, r, sign=-1)


@pytest.mark.parametrize("scaling", SCALING, ids=lambda s: s.get("scaling", "none"))
def test_scaled_contexts_and_far_positions(cuda, scaling):
    r = paged.Rotary(64, layout="half", **scaling)
    x = torch.randn(9, 4, 64, generator=torch.Generator().manual_seed(1)).cuda()
    positions = torch.tensor([0, 1, -1, 4095, 131_072, 1_000_003, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31]).cuda()
    check(r.apply(x, positions), x, positions, r)
    check(r.apply(x, positions.int()), x, positions, r)
    far = torch.tensor([2 ** 40 + 12345] * 9).cuda()
    check(r.apply(x, far), x, far, r)


def test_strides_batches_and_in_place(cuda):
    g = torch.Generator().manual_seed(2)
    r = paged.Rotary(64)
    qkv = torch.randn(3, 40, 10, 64, generator=g).half().cuda()
    positions = torch.randint(0, 9000, (3, 40), generator=g).cuda()
    x = qkv[:, :, 2:7]
    flat = r.apply(qkv.flatten(0, 1)[:, 2:7], positions.flatten())
    check(flat, qkv.flatten(0, 1)[:, 2:7], positions.flatten(), r)
    assert torch.equal(r.apply(x, positions).flatten(0, 1), flat)
    assert torch.equal(r(x, positions[0])[0], flat[:40])               # one row of positions for all
    turned_view = x.transpose(0, 1).contiguous().transpose(0, 1)        # batch inside tokens
    assert torch.equal(r.apply(turned_view, positions).flatten(0, 1), flat)
    rest = qkv.clone()
    assert r.apply(x, positions, out=x).data_ptr() == x.data_ptr()
    assert torch.equal(x.flatten(0, 1), flat)
    rest[:, :, 2:7] = x
    assert torch.equal(qkv, rest)                                       # nothing beside it changed
    odd = torch.randn(40 * 3 * 64 + 1, generator=g).half().cuda()[1:].view(40, 3, 64)
    check(r.apply(odd, positions[0]), odd, positions[0], r)             # not on 16 bytes
    heads_first = torch.randn(5, 40, 64, generator=g).half().cuda().transpose(0, 1)
    check(r.apply(heads_first, positions[0]), heads_first, positions[0], r)
    assert r.apply(x[:0], positions[:0]).shape == x[:0].shape


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient(cuda, layout):
    """Through autograd: against the formula, and against differences of the
    loss (which is linear in x: no error of the step's own)."""
    g = torch.Generator().manual_seed(4)
    r = paged.Rotary(32, 24, layout=layout, scaling="yarn", factor=4.0, trained_length=2048)
    x = torch.randn(13, 3, 32, generator=g).cuda().requires_grad_()
    w = torch.randn(13, 3, 32, generator=g).cuda()
    positions = torch.randint(0, 10_000, (13,), generator=g).cuda()
    (r.apply(x, positions) * w).sum().backward()
    check(x.grad, w, positions, r, sign=-1)
    assert torch.equal(x.grad, r.grad(w, positions))
    for _ in range(5):
        d = torch.randn(13, 3, 32, generator=g).cuda()
        with torch.no_grad():
            up, down = r.apply(x + d, positions), r.apply(x - d, positions)
        slope = ((up.double() - down.double()) * w.double()).sum() / 2
        want = (x.grad.double() * d.double()).sum()
        size = (up.double().abs() * w.double().abs()).sum()  # float32 sums of x + d, and the turn's own 6e-7
        assert abs(slope - want) <= 2e-6 * size


def make_cache(lengths, page_size, kv_heads, dim, dtype, layout="token", layers=2):
    c = paged.PagedCache.allocate(layers, sum(-(-n // page_size) for n in lengths) + 2, page_size, kv_heads, dim,
                                  len(lengths), max(-(-n // page_size) for n in lengths) + 1, dtype, layout)
    c.extend(torch.arange(len(lengths), dtype=torch.int32, device="cuda"),
             torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    for t in (c.k, c.v):
        t.normal_()
    return c


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("dim,rot,page_size", [(64, 64, 16), (128, 32, 7), (80, 40, 1), (8, 2, 100)])
def test_append(cuda, dtype, layout, dim, rot, page_size):
    """A prompt's tokens, then one more of each row, with queries; the rest of
    the cache stays as it is."""
    g = torch.Generator().manual_seed(6)
    c = make_cache([50, 1, 21], page_size, 2, dim, dtype, layout)
    r = paged.Rotary(dim, rot, layout="interleaved" if layout == "head" else "half")
    for rows, index in (([0] * 50 + [2] * 20, list(range(50)) + list(range(20))), ([2, 0, 1], [20, 49, 0])):
        n = len(rows)
        qkv = torch.randn(n, 3 * 2 + 4, dim, generator=g).to(dtype).cuda()
        q, k, v = qkv.split([6, 2, 2], 1)
        before = c.k.clone(), c.v.clone()
        ri, ii = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in (rows, index))
        turned = c.append(1, k, v, ri, None if n == 3 else ii, q=q, rotary=r)  # n == 3: each row's last token
        check(turned, q, ii.long(), r)
        page = c.table[ri.long(), (ii // page_size).long()].long()
        slot = (ii % page_size).long()
        check(c.k[1, page, slot], k, ii.long(), r)
        assert torch.equal(c.v[1, page, slot], v)
        assert torch.equal(c.k[1, page, slot], r.apply(k, ii))  # the same bits as by apply()
        before[0][1, page, slot], before[1][1, page, slot] = c.k[1, page, slot], v
        assert torch.equal(c.k, before[0]) and torch.equal(c.v, before[1])
    c.check()
    # positions of their own, in place, and no rotation at all
    positions = torch.tensor([7, 70_000, 0], device="cuda")
    same = q.clone()
    assert c.append(0, k, v, ri, ii, q=same, rotary=r, positions=positions, q_out=same) is same
    check(same, q, positions, r)
    check(c.k[0, page, slot], k, positions, r)
    assert c.append(0, k, v, ri, ii) is None
    assert torch.equal(c.k[0, page, slot], k)


def test_append_where_there_is_no_place(cuda):
    c = make_cache([10, 4], 4, 1, 8, torch.float16, layers=1)
    c.table[0, 1] = -1
    before = c.k.clone(), c.v.clone()
    rows = torch.tensor([-1, 2, 0, 0, 0, 1], dtype=torch.int32, device="cuda")
    index = torch.tensor([0, 0, 5, -1, 400, 4], dtype=torch.int32, device="cuda")
    kv = torch.ones(6, 1, 8, dtype=torch.float16, device="cuda")
    q = c.append(0, kv, kv, rows, index, q=kv, rotary=paged.Rotary(8))
    assert torch.equal(c.k, before[0]) and torch.equal(c.v, before[1])
    check(q, kv, index.long(), paged.Rotary(8))  # queries are turned all the same
    with pytest.raises(RuntimeError, match="place"):
        c.check()


def test_graphs(cuda):
    c = make_cache([5, 9], 4, 1, 16, torch.float16, layers=1)
    r = paged.Rotary(16)
    rows, one = torch.arange(2, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    kv = torch.randn(2, 1, 16, generator=torch.Generator().manual_seed(8)).half().cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.append(0, kv, kv, rows, rotary=r)
    c.extend(rows, one)
    graph.replay()
    last = (c.lengths - 1).long()
    page = c.table[rows.long(), last // 4].long()
    assert torch.equal(c.k[0, page, last % 4], r.apply(kv, last))


def test_refusals(cuda):
    r = paged.Rotary(16)
    x, p = torch.zeros(3, 2, 16, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in ((x[0], p), (x[..., :8], p), (x.double(), p), (x, p[:2]), (x, p.float()), (x, p.cpu()), (x.cpu(), p)):
        with pytest.raises(ValueError):
            r.apply(*bad)
    with pytest.raises(ValueError):
        r.apply(x, p, out=x.half())
    with pytest.raises(ValueError, match="positions"):
        r.apply(x[None], p[:2])
    c = make_cache([5], 4, 2, 16, torch.float16)
    k = torch.zeros(1, 2, 16, dtype=torch.float16, device="cuda")
    rows = torch.zeros(1, dtype=torch.int32, device="cuda")
    for kw in ({"k": k.bfloat16()}, {"v": k[:, :1]}, {"rows": rows.long()}, {"q": k}, {"rotary": paged.Rotary(32)},
               {"index": torch.zeros(2, dtype=torch.int32, device="cuda")},
               {"rotary": r, "positions": rows.float()}):
        with pytest.raises(ValueError):
            c.append(0, **{"k": k, "v": k, "rows": rows, **kw})
    with pytest.raises(ValueError, match="layer"):
        c.append(2, k, k, rows)
