"""What a call of the paged cache must leave alone: tokens that were there
before, of the row itself and of rows that share its pages."""
import pytest
import torch

from jasper_b200 import paged

pytestmark = pytest.mark.gpu


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make(n_pages, rows, width, page_size=4, layers=2, kv_heads=1, dim=8, seed=0):
    c = paged.PagedCache.allocate(layers, n_pages, page_size, kv_heads, dim, rows, width)
    g = torch.Generator(device="cuda").manual_seed(seed)
    c.k.normal_(generator=g), c.v.normal_(generator=g)
    return c


def new_tokens(n, c, value=7.0):
    return torch.full((n, c.n_kv_heads, c.head_dim), value, dtype=c.dtype, device="cuda")


def append_everywhere(c, rows, index=None):
    kv = new_tokens(len(rows), c)
    for layer in range(c.n_layers):
        c.append(layer, kv, kv, rows, index)


def untouched(c, before, but=()):
    """Keys and values are as before, except for tokens (page, slot) of `but`."""
    for t, was in zip((c.k, c.v), before):
        same = (t == was).all(-1).all(-1).all(0)
        for page, slot in but:
            assert not same[page, slot]
            same[page, slot] = True
        assert same.all()


@pytest.mark.parametrize("length", [8, 7, 1])
def test_an_append_after_a_refused_extend_writes_nothing(cuda, length):
    """No free page is left: the row keeps its last token, in every layer; a
    row that got its room is served."""
    c = make(n_pages=3, rows=3, width=8)
    c.extend(ints(0, 1), ints(length, 4))
    spare = 3 - -(-length // 4) - 1
    before = c.k.clone(), c.v.clone()
    rows = ints(0, 1)
    c.extend(rows, ints(4 * spare + 5, 0))                  # row 0: more than there is
    assert c.lengths.tolist()[:2] == [length, 4]
    append_everywhere(c, ints(0))
    untouched(c, before)
    with pytest.raises(RuntimeError, match="free page.*place"):
        c.check()
    c.free(ints(1))
    c.extend(ints(0), ints(1))                              # now there is room
    append_everywhere(c, ints(0))
    page = int(c.table[0, length // 4])
    untouched(c, before, [(page, length % 4)])
    c.check()


def test_a_full_row_and_a_negative_extension(cuda):
    c = make(n_pages=9, rows=4, width=2)
    c.extend(ints(0, 1, 2), ints(8, 3, 5))
    before = c.k.clone(), c.v.clone()
    c.extend(ints(0, 1, 2, 2), ints(1, -1, 0, 1))           # full, no number, nothing wanted, named again
    assert c.lengths.tolist() == [8, 3, 5, 0]
    append_everywhere(c, ints(0, 1, 3))
    untouched(c, before)
    append_everywhere(c, ints(2))                           # asked for nothing: its last token is rewritten
    untouched(c, before, [(int(c.table[2, 1]), 0)])
    append_everywhere(c, ints(1), ints(2))                  # an index of the caller's own is followed
    untouched(c, before, [(int(c.table[2, 1]), 0), (int(c.table[1, 0]), 2)])


def test_a_shared_last_page_survives_a_refused_extend(cuda):
    """Rows that end in a whole page of another row, adopted or forked."""
    c = make(n_pages=2, rows=6, width=4)
    c.extend(ints(0), ints(8))
    c.adopt(ints(1, 2), c.table[:1, :2].expand(2, 2))
    c.fork(ints(0, 1), ints(3, 4))
    before = c.k.clone(), c.v.clone()
    rows = ints(0, 1, 2, 3, 4)
    c.extend(rows, torch.ones_like(rows))
    append_everywhere(c, rows)
    untouched(c, before)
    c.fork(ints(3), ints(5))                                # a copy of a refused row is no better off
    append_everywhere(c, ints(5))
    untouched(c, before)
    for name in ("free", "adopt", "fork"):                  # an emptied row begins anew
        c.free(ints(1, 2, 5))
        assert c.marks[[1, 2, 5]].tolist() == [0, 0, 0]
        if name == "adopt":
            c.adopt(ints(1), c.table[:1, :2])
        if name == "fork":
            c.marks[0] = 0
            c.fork(ints(0), ints(1))
        assert c.marks[1] == 0


@pytest.mark.parametrize("n", [3, 1500, 2600])
def test_refused_rows_of_long_lists(cuda, n):
    """Every other row of a long list is full; all parents' marks reach their
    children."""
    c = make(n_pages=2 * n, rows=2 * n, width=1, page_size=2, layers=1)
    rows = torch.arange(n, dtype=torch.int32, device="cuda")
    full = rows % 2 == 0
    c.extend(rows, torch.where(full, 2, 1).int())
    before = c.k.clone(), c.v.clone()
    c.extend(rows, torch.ones_like(rows))
    assert torch.equal(c.marks[:n] < 0, full) and (c.lengths[:n] == 2).all()
    c.fork(rows, rows + n)
    assert torch.equal(c.marks[n:] < 0, full) and (c.lengths[n:] == 2).all()
    kv = new_tokens(n, c)
    c.append(0, kv, kv, rows)
    written = torch.zeros(2 * n, 2, dtype=torch.bool, device="cuda")
    written[c.table[:n, 0][~full].long(), 1] = True
    assert torch.equal((c.k != before[0]).any(-1).any(-1)[0], written)


def test_marks_of_the_callers_own(cuda):
    c = make(n_pages=2, rows=2, width=2)
    marks = ints(0, -1)
    own = paged.PagedCache(c.k, c.v, c.table, c.lengths, c.refs, c.status, marks)
    own.extend(ints(0, 1), ints(4, 4))
    assert own.marks is marks and marks.tolist() == [0, 0]
    own.extend(ints(0, 1), ints(1, 1))
    assert (marks < 0).all()
    for bad in (marks[:1], marks.long(), marks.cpu(), ints(0, 0, 0, 0)[::2]):
        with pytest.raises(ValueError, match="marks"):
            paged.PagedCache(c.k, c.v, c.table, c.lengths, c.refs, c.status, bad)
