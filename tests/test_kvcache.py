"""The paged cache's bookkeeping without a GPU: which page each sequence holds through growth, forks, frees and
compaction, with the page copies recorded instead of run."""
import pytest
import torch

from basal_b200 import kvcache


@pytest.fixture
def moved(monkeypatch):
    got = []
    monkeypatch.setattr(kvcache.ops, "kv_copy_pages", lambda pools, src, dst: got.append((list(src), list(dst))))
    return got


def cache(pages=10, page_size=4, **kw):
    return kvcache.PagedKVCache(1, pages, 1, 64, page_size, device="cpu", **kw)


def consistent(c):
    held = {}
    for s, pages in c._of.items():
        assert len(pages) * c.page_size >= c.length(s) and len(set(pages)) == len(pages)
        for p in pages:
            held[p] = held.get(p, 0) + 1
    assert [held.get(p, 0) for p in range(c.pages)] == c._shares
    assert sorted(c._free) == [p for p in range(c.pages) if p not in held]


def test_grow_and_free(moved):
    c = cache()
    a, b = c.add(), c.add()
    c.grow([a, b], [4, 5])
    assert [len(c.pages_of(s)) for s in (a, b)] == [1, 2] and c.free_pages == 7
    c.grow([a])
    assert len(c.pages_of(a)) == 2 and c.length(a) == 5
    c.grow([a, b], 0)
    consistent(c)
    c.free(a)
    assert c.free_pages == 8 and not moved
    consistent(c)
    with pytest.raises(KeyError):
        c.grow([a])
    with pytest.raises(KeyError):
        c.fork(a)


def test_fork_copies_only_what_is_written(moved):
    c = cache()
    a = c.add()
    c.grow([a], 6)
    full, half = c.pages_of(a)
    b, d = c.fork(a), c.fork(a)
    assert c.free_pages == 8
    c.grow([a, b, d])  # three write the half-full page: two copies, the last keeps it
    assert moved == [([half, half], [c.pages_of(a)[1], c.pages_of(b)[1]])]
    assert c.pages_of(d) == [full, half] and c.pages_of(a)[0] == c.pages_of(b)[0] == full
    consistent(c)
    moved.clear()
    c.grow([a, b, d], 1)  # nobody shares what is written now
    assert not moved
    e = c.fork(a)  # at a page's end (8 tokens of 4): nothing to copy, a new page each
    c.grow([e, a])
    assert not moved and c.pages_of(e)[:2] == c.pages_of(a)[:2] and c.pages_of(e)[2] != c.pages_of(a)[2]
    consistent(c)


def test_a_shared_page_is_copied_when_one_of_its_holders_writes(moved):
    c = cache()
    a = c.add()
    c.grow([a], 2)
    b = c.fork(a)
    c.grow([a])
    assert moved == [(c.pages_of(b), c.pages_of(a))]
    c.free(a)
    moved.clear()
    c.grow([b])
    assert not moved
    consistent(c)


def test_out_of_pages_changes_nothing(moved):
    c = cache(pages=3)
    a = c.add()
    c.grow([a], 10)
    b = c.fork(a)
    before = (c.pages_of(a), c.length(a), c.free_pages)
    for n in (1, 3):  # b would need a copy; a copy and a page
        with pytest.raises(MemoryError):
            c.grow([b], n)
    with pytest.raises(MemoryError):
        c.grow([a, b])
    assert before == (c.pages_of(a), c.length(a), c.free_pages) and not moved
    consistent(c)


def test_refusals(moved):
    c = cache()
    a = c.add()
    for bad in (lambda: c.grow([a, a]), lambda: c.grow([a], -1), lambda: c.grow([a], [1, 2]), lambda: cache(pages=0),
                lambda: kvcache.PagedKVCache(1, 4, 1, 96, device="cpu"), lambda: cache(dtype=torch.float32)):
        with pytest.raises(ValueError):
            bad()
    assert c.length(a) == 0


def test_compact(moved):
    c = cache()
    s = [c.add() for _ in range(4)]
    for x in s:
        c.grow([x], 8)
    t = c.fork(s[3])
    c.free(s[0])
    c.free(s[2])
    assert c.compact() == 4
    (src, dst), = moved
    assert not set(src) & set(dst) and max(dst) < 4 and min(src) >= 4
    assert c.pages_of(t) == c.pages_of(s[3]) and max(c.pages_of(t) + c.pages_of(s[1])) < 4
    consistent(c)
    moved.clear()
    assert c.compact() == 4 and not moved
    c.grow([t])
    consistent(c)


def test_batch(moved):
    c = cache()
    a, b, e = c.add(), c.add(), c.add()
    c.grow([a], 9)
    c.grow([b, a], [2, 1])
    got = c.batch([b, e, a])
    assert got.table.tolist() == [c.pages_of(b) + [-1, -1], [-1] * 3, c.pages_of(a)]
    assert got.lengths.tolist() == [2, 0, 10] and got.start.tolist() == [0, 0, 9] and got.count.tolist() == [2, 0, 1]
    assert c.batch([]).table.shape == (0, 1)


def test_batches_follow_every_change(moved):
    """The table of a batch after growth, a copied page, a compaction and a freed sequence is the sequences' pages."""
    c = cache(pages=12)

    def same(*seqs):
        got = c.batch(seqs)
        for r, s in enumerate(seqs):
            pages = c.pages_of(s)
            assert got.table[r].tolist() == pages + [-1] * (got.table.shape[1] - len(pages))
        assert got.lengths.tolist() == [c.length(s) for s in seqs]

    a, b = c.add(), c.add()
    c.grow([a, b], [6, 9])
    same(a, b)
    c.grow([a], 3)
    same(b, a)
    d = c.fork(a)
    same(a, b, d)
    c.grow([d, a])          # d writes a copy of the shared last page
    same(a, b, d)
    c.free(b)
    same(d, a)
    c.compact()
    same(a, d)
    c.grow([a], 5)
    same(a, d)


def test_a_batch_brings_only_what_the_last_grow_made_room_for(moved):
    """A grown, an ungrown and a forked sequence in one batch: an append with it writes the grown one's tokens and no
    other position, so no shared page and no token that was appended before."""
    c = cache()
    a, b = c.add(), c.add()
    c.grow([a, b], 2)
    f = c.fork(b)
    got = c.batch([b, f])               # forked since: its page is shared
    assert got.count.tolist() == [0, 0] and got.start.tolist() == got.lengths.tolist() == [2, 2]
    c.grow([a])
    got = c.batch([a, b, f])
    assert got.count.tolist() == [1, 0, 0] and got.start.tolist() == [2, 2, 2] and got.lengths.tolist() == [3, 2, 2]
    c.grow([b, f], [3, 0])
    got = c.batch([a, b, f])
    assert got.count.tolist() == [0, 3, 0] and got.start.tolist() == [3, 2, 2] and got.lengths.tolist() == [3, 5, 2]
    c.compact()                          # pages move, tokens stay to be appended
    assert c.batch([b]).count.tolist() == [3]
    c.free(b)
    with pytest.raises(MemoryError):
        c.grow([a], 100)
    assert c.batch([a, f]).count.tolist() == [0, 0]
    consistent(c)


def test_a_copy_that_is_refused_changes_nothing(monkeypatch):
    c = cache()
    a = c.add()
    c.grow([a], 6)
    b = c.fork(a)
    before = (c.pages_of(a), c.pages_of(b), c.length(b), c.free_pages, c.batch([a, b]).table.tolist())

    def fails(*a):
        raise RuntimeError("no copy")

    monkeypatch.setattr(kvcache.ops, "kv_copy_pages", fails)
    with pytest.raises(RuntimeError):
        c.grow([b], 5)
    assert before == (c.pages_of(a), c.pages_of(b), c.length(b), c.free_pages, c.batch([a, b]).table.tolist())
    consistent(c)


def test_no_batch_inside_a_captured_graph(moved, monkeypatch):
    """A graph would replay the copy from host memory that is used for something else by then."""
    c = cache()
    a = c.add()
    c.grow([a], 2)
    c.device = torch.device("cuda")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="capture"):
        c.batch([a])


def test_an_append_of_fewer_tokens_than_there_is_room_for(moved, monkeypatch):
    """The positions behind them would be read as they were allocated; rows of uneven counts, padded, are fine."""
    wrote = []
    monkeypatch.setattr(kvcache.ops, "kv_append", lambda *a: wrote.append(a))
    c = cache()
    a, b = c.add(), c.add()
    c.grow([a, b], [3, 2])
    x = torch.zeros(2, 3, 1, 64)
    with pytest.raises(ValueError, match="3"):
        c.append(0, c.batch([a, b]), x[:, :2], x[:, :2])
    assert not wrote
    c.append(0, c.batch([a, b]), x, x)
    c.append(0, c.batch([b]), x[:1, :2], x[:1, :2])
    assert len(wrote) == 2
