"""Which page belongs to whom: forks, copies on write, truncation, compaction, and calls that do not fit."""
import random

import pytest

from antares_b200.kv_cache import CacheFull, PagedKV8Cache, PagePool


class Model:
    """What every sequence should read: page contents as rows, copied as the pool says."""

    def __init__(self, pages, page_rows, max_seqs=8, max_pages=8):
        self.pool = PagePool(pages, page_rows, max_seqs, max_pages)
        self.page = [[None] * page_rows for _ in range(pages)]
        self.want = {}

    def copy(self, pairs):
        src, dst = {a for a, _ in pairs}, [b for _, b in pairs]
        assert len(set(dst)) == len(dst) and not src & set(dst)   # what ops.kv_copy_pages asks for
        for a, b in pairs:
            self.page[b] = list(self.page[a])

    def write(self, seqs, n, mark):
        self.copy(self.pool.reserve({s: n for s in seqs}))
        R = self.pool.page_rows
        for s in seqs:
            for i in range(n):
                p = self.pool.rows[s] + i
                page = self.pool.held[s][p // R]
                assert self.pool.users[page] == 1
                self.page[page][p % R] = (s, mark, i)
                self.want[s].append((s, mark, i))
            self.pool.advance(s, n)

    def check(self):
        R, used = self.pool.page_rows, {}
        for s, rows in self.want.items():
            assert self.pool.rows[s] == len(rows)
            assert [self.page[self.pool.held[s][p // R]][p % R] for p in range(len(rows))] == rows
            for p in self.pool.held[s]:
                used[p] = used.get(p, 0) + 1
        assert [used.get(p, 0) for p in range(self.pool.pages)] == self.pool.users
        assert sorted(self.pool._free) == [p for p in range(self.pool.pages) if p not in used]


@pytest.mark.parametrize("seed", range(6))
def test_any_order_of_calls(seed):
    rng = random.Random(seed)
    m = Model(40, rng.choice([1, 4, 16]))
    for t in range(400):
        seqs = sorted(m.want)
        what = rng.choice(["add", "write", "write", "write", "fork", "free", "truncate", "compact", "reserve"])
        try:
            if what == "add":
                m.want[m.pool.add()] = []
            elif what == "compact":
                m.copy(m.pool.compact())
                used = sum(1 for u in m.pool.users if u)
                assert all(m.pool.users[:used]) and not any(m.pool.users[used:])
            elif seqs:
                s = rng.choice(seqs)
                if what == "write":
                    m.write(rng.sample(seqs, rng.randrange(1, len(seqs) + 1)), rng.randrange(0, 9), t)
                elif what == "reserve":   # room that is not used before something else happens
                    m.copy(m.pool.reserve({s: rng.randrange(20)}))
                elif what == "fork":
                    m.want[m.pool.fork(s)] = list(m.want[s])
                elif what == "free":
                    m.pool.free(s)
                    del m.want[s]
                else:
                    n = rng.randrange(len(m.want[s]) + 1)
                    m.pool.truncate(s, n)
                    del m.want[s][n:]
        except CacheFull:
            pass   # nothing has changed
        m.check()


def test_the_last_writer_keeps_the_page():
    m = Model(10, 16)
    a = m.pool.add()
    m.want[a] = []
    m.write([a], 5, 0)
    b, c = m.pool.fork(a), m.pool.fork(a)
    m.want[b], m.want[c] = list(m.want[a]), list(m.want[a])
    assert m.pool.free_pages == 9
    m.write([a, b, c], 1, 1)
    m.check()
    assert m.pool.free_pages == 7
    # full pages stay shared
    m.write([a], 10, 2)
    d = m.pool.fork(a)
    m.want[d] = list(m.want[a])
    assert m.pool.reserve({d: 1}) == [] and m.pool.users[m.pool.held[d][0]] == 2


def test_forks_of_room_that_is_reserved_but_not_written():
    """Pages of rows to come are shared by a fork like any other; whoever writes first gets pages of its own, nothing to copy."""
    for rows in (0, 16, 20):
        m = Model(12, 16)
        a = m.pool.add()
        m.want[a] = []
        m.write([a], rows, 0)
        m.copy(m.pool.reserve({a: 36}))
        b = m.pool.fork(a)
        m.want[b] = list(m.want[a])
        copies = m.pool.reserve({a: 36})
        assert len(copies) == (rows % 16 > 0)
        m.copy(copies)
        m.write([a], 36, 1)
        m.write([b], 36, 2)
        m.check()


def test_what_does_not_fit_changes_nothing():
    pool = PagePool(4, 16, 2, 3)
    a, b = pool.add(), pool.add()
    with pytest.raises(CacheFull, match="sequences"):
        pool.add()
    with pytest.raises(CacheFull, match="more than its 3 pages"):
        pool.reserve({a: 49})
    with pytest.raises(CacheFull, match="needed"):
        pool.reserve({a: 48, b: 20})
    assert pool.free_pages == 4 and pool.held == {a: [], b: []}
    pool.reserve({a: 48})
    pool.advance(a, 48)
    with pytest.raises(ValueError):
        pool.advance(a, 1)
    with pytest.raises(ValueError):
        pool.truncate(a, 49)
    with pytest.raises(ValueError):
        pool.reserve({a: -1})
    for f in (pool.free, pool.fork):
        with pytest.raises(KeyError):
            f(7)
    with pytest.raises(KeyError):
        pool.reserve({7: 1})
    with pytest.raises(ValueError):
        PagePool(0, 16, 1, 1)
    with pytest.raises(ValueError, match="power of two"):
        PagedKV8Cache(1, 4, 2, page_rows=24, device="cpu")


def test_batches_on_the_host():
    c = PagedKV8Cache(2, 6, 2, page_rows=16, max_seqs=3, max_seq=48, device="cpu")
    a, b = c.add(), c.add()
    c.pool.reserve({a: 20, b: 3})
    c.advance(a, 20)
    table, pos0 = c.batch([b, a])
    assert table.shape == (2, 3) and pos0.tolist() == [0, 20] and table[1, :2].tolist() == c.pool.held[a]
    assert table[0, 1:].tolist() == [-1, -1] and table[1, 2] == -1
    with pytest.raises(ValueError, match="once"):
        c.batch([a, a])
    assert len(c.layer(1)) == 4 and c.layer(1)[2].shape == (6, 2, 1)
