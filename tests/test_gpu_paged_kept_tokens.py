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


def rows_of(c, r, n):
    """Keys and values of the first n tokens of row r."""
    t = torch.arange(n, device="cuda")
    page = c.table[r][t // c.page_size].long()
    return c.k[:, page, t % c.page_size].clone(), c.v[:, page, t % c.page_size].clone()


@pytest.mark.parametrize("page_size,length", [(4, 6), (4, 1), (7, 13), (16, 20)])
def test_a_row_adopted_into_a_page_does_not_write_there(cuda, page_size, length):
    """Adopted, extended and appended to: the donor's tokens stay, and the donor
    goes on in its page; a fork of the row goes on behind what it adopted."""
    held = -(-length // page_size)
    c = make(n_pages=20, rows=8, width=6, page_size=page_size)
    c.extend(ints(0), ints(held * page_size - 1))            # its last page has a place left
    c.adopt(ints(1, 2), c.table[:1, :held].expand(2, held), ints(length, length))
    c.fork(ints(1), ints(3))
    before = c.k.clone(), c.v.clone()
    for step in range(held * page_size - length):            # up to the page's end
        c.extend(ints(1, 2), ints(1, 1))
        append_everywhere(c, ints(1, 2))
        append_everywhere(c, ints(1), ints(length + step))   # nor by index
    untouched(c, before)
    with pytest.raises(RuntimeError, match="place"):
        c.check()
    c.extend(ints(0), ints(1))
    append_everywhere(c, ints(0))
    last = [(int(c.table[0, held - 1]), page_size - 1)]
    untouched(c, before, last)
    c.extend(ints(1), ints(1))                               # a page of its own again
    append_everywhere(c, ints(1))
    untouched(c, before, last + [(int(c.table[1, held]), 0)])
    c.extend(ints(3), ints(1))                               # a fork: at once
    append_everywhere(c, ints(3))
    assert int(c.table[3, length // page_size]) != int(c.table[1, length // page_size])
    untouched(c, before, last + [(int(c.table[1, held]), 0), (int(c.table[3, length // page_size]), length % page_size)])
    assert all(torch.equal(a, b) for a, b in zip(rows_of(c, 3, length), rows_of(c, 0, length)))
    c.check()


@pytest.mark.parametrize("length,window", [(21, 0), (21, 9), (5, 0), (700, 0)])
@pytest.mark.parametrize("copies", [1, 40, 1100])
def test_the_rest_of_an_adopted_page_is_not_attended_to(cuda, length, window, copies):
    """The same result before the row grows past its adopted tokens, with and
    without a fork, as after it, wherever the donor's later tokens are: they are
    NaN here."""
    page_size, dim = 16, 64
    held = -(-length // page_size)
    c = paged.PagedCache.allocate(1, 200, page_size, 2, dim, 6, max(held + 3, 110))
    g = torch.Generator(device="cuda").manual_seed(length)
    c.extend(ints(0, 5), ints(held * page_size, 1700))
    c.k.normal_(generator=g), c.v.normal_(generator=g)
    page, slot = int(c.table[0, held - 1]), length % page_size
    c.k[:, page, slot:], c.v[:, page, slot:] = float("nan"), float("nan")
    c.adopt(ints(1), c.table[:1, :held], ints(length))
    q = torch.randn(1, 4, dim, generator=g, device="cuda").half().expand(copies + 1, 4, dim)
    rows = torch.full((copies + 1,), 1, dtype=torch.int32, device="cuda")
    rows[copies // 2] = 5                                    # a longer row among them
    at = torch.arange(copies + 1, device="cuda") != copies // 2

    def attend(r):
        out = c.attend(0, q, torch.where(rows == 1, r, rows).int(), return_lse=True, window=window)
        assert all(t[at].isfinite().all() for t in out)
        assert all(torch.equal(t[at], t[at][:1].expand_as(t[at])) for t in out if copies < 1000)
        return [t[at][0] for t in out]

    plain = attend(1)
    more = held * page_size - length
    c.extend(ints(1), ints(more))                            # to the page's end: nothing there is the row's
    if not window:
        assert all(torch.equal(a, b) for a, b in zip(attend(1), plain))
    c.fork(ints(1), ints(2))                                 # nor is it the fork's
    assert int(c.marks[2]) == length
    if not window:
        assert all(torch.equal(a, b) for a, b in zip(attend(2), plain))
    # behind the page the row goes on; it and its fork attend to the same
    c.extend(ints(1), ints(3))
    kv = torch.randn(3, 2, dim, generator=g, device="cuda").half()
    three = held * page_size + torch.arange(3, dtype=torch.int32, device="cuda")
    c.append(0, kv, kv, ints(1, 1, 1), three)
    c.fork(ints(1), ints(3))
    grown = attend(1)
    assert all(torch.equal(a, b) for a, b in zip(attend(3), grown))
    # the same tokens in pages that the row holds whole
    c.extend(ints(4), ints(length + 3))
    t = torch.arange(length + 3, device="cuda")
    source = torch.where(t < length, t, t - length + held * page_size)
    from_page, to_page = c.table[1][source // page_size].long(), c.table[4][t // page_size].long()
    for cache in (c.k, c.v):
        cache[:, to_page, t % page_size] = cache[:, from_page, source % page_size]
    if not window:
        for a, b in zip(attend(4), grown):                   # tokens in other tiles: other rounding
            assert (a.float() - b.float()).abs().max() <= 2 ** -9 * (1 + b.float().abs().max())
    c.check()


def test_an_emptied_row_forgets_where_it_was_adopted(cuda):
    c = make(n_pages=8, rows=4, width=4)
    c.extend(ints(0), ints(8))
    c.adopt(ints(1), c.table[:1, :2], ints(6))
    assert c.marks.tolist() == [0, 6, 0, 0]
    c.extend(ints(1), ints(1))
    assert c.marks.tolist() == [0, 6, 0, 0]
    c.extend(ints(1), ints(100))                             # refused
    assert c.marks[1] < 0
    c.fork(ints(1), ints(2))
    assert c.marks[1] == c.marks[2]
    c.free(ints(1, 2))
    c.adopt(ints(1), c.table[:1, :2], ints(4))               # whole pages, if fewer
    assert c.marks.tolist() == [0, 0, 0, 0]
    c.free(ints(1))
    c.marks[1] = 6
    c.extend(ints(1), ints(7))
    assert c.marks.tolist() == [0, 0, 0, 0]
    before = c.k.clone(), c.v.clone()
    append_everywhere(c, ints(1))
    untouched(c, before, [(int(c.table[1, 1]), 2)])


def test_forks_of_empty_rows_carry_no_mark(cuda):
    """A chain of pairs, each child the next one's parent: all but the first
    parent are empty, and only its child is a copy of a refused row."""
    n = 2500
    c = make(n_pages=2, rows=n + 1, width=1, page_size=2, layers=1)
    c.extend(ints(0), ints(2))
    every = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    c.extend(every, torch.full_like(every, 3))               # no row has place for so many
    assert (c.marks < 0).all() and c.lengths.sum() == 2
    c.fork(every[:-1], every[1:])
    assert c.lengths[:3].tolist() == [2, 2, 0] and (c.marks[:2] < 0).all() and (c.marks[2:] == 0).all()
