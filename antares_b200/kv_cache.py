"""Pages of the 8-bit KV cache for many sequences: which page holds what (host), and the tensors that ops.kv8_* work on.

A sequence is a list of pages; pages are shared between forks until one of them writes (copy on write), freed when the last
user is gone, and moved together by compact().  The book-keeping (PagePool) is plain Python and touches no GPU; the copies
that it asks for are one ops.kv_copy_pages over every layer, in stream order with the launches around it.
"""
import heapq

import torch

from . import ops


class CacheFull(RuntimeError):
    """Fewer free pages, sequence slots or table columns than a call needs; nothing has been changed."""


class PagePool:
    """Pages 0 .. pages - 1 of page_rows rows, up to max_seqs sequences of up to max_pages pages each."""

    def __init__(self, pages, page_rows, max_seqs, max_pages):
        if pages < 1 or page_rows < 1 or max_seqs < 1 or max_pages < 1:
            raise ValueError("a pool needs at least one page, row, sequence and column")
        self.pages, self.page_rows, self.max_seqs, self.max_pages = pages, page_rows, max_seqs, max_pages
        self.users = [0] * pages            # sequences that a page belongs to
        self._free = list(range(pages))     # a heap: the lowest page first, so that little is left to compact
        self._slots = list(range(max_seqs))
        self.held = {}                      # sequence -> its pages
        self.rows = {}                      # sequence -> rows in use

    @property
    def free_pages(self):
        return len(self._free)

    def _known(self, seq):
        if seq not in self.held:
            raise KeyError("no sequence %r" % (seq,))

    def add(self):
        """A new, empty sequence."""
        if not self._slots:
            raise CacheFull("all %d sequences are in use" % self.max_seqs)
        seq = heapq.heappop(self._slots)
        self.held[seq], self.rows[seq] = [], 0
        return seq

    def fork(self, seq):
        """A sequence with the same rows.  Nothing is copied: whichever writes into a shared page first gets its own (reserve).  Rows
        that were reserved and not written are shared as well: reserve again before they are."""
        self._known(seq)
        new = self.add()
        self.held[new], self.rows[new] = list(self.held[seq]), self.rows[seq]
        for p in self.held[seq]:
            self.users[p] += 1
        return new

    def _drop(self, page):
        self.users[page] -= 1
        if self.users[page] == 0:
            heapq.heappush(self._free, page)

    def free(self, seq):
        self._known(seq)
        for p in self.held.pop(seq):
            self._drop(p)
        del self.rows[seq]
        heapq.heappush(self._slots, seq)

    def truncate(self, seq, rows):
        """Keeps the first rows only (drafted tokens that were not accepted)."""
        self._known(seq)
        if not 0 <= rows <= self.rows[seq]:
            raise ValueError("sequence %d has %d rows, not %d" % (seq, self.rows[seq], rows))
        keep = -(-rows // self.page_rows)
        for p in self.held[seq][keep:]:
            self._drop(p)
        del self.held[seq][keep:]
        self.rows[seq] = rows

    def reserve(self, need):
        """Makes room for need[seq] more rows of each sequence: new pages, and own ones in place of those that are shared and will
        be written.  Returns the (source, destination) pages to copy before anything is written: those partly filled."""
        fresh, own = {}, {}
        users = {}
        for seq, n in need.items():
            self._known(seq)
            if n < 0:
                raise ValueError("rows to reserve must not be negative, got %d" % n)
            have, end = len(self.held[seq]), self.rows[seq] + n
            want = -(-end // self.page_rows)
            if want > self.max_pages:
                raise CacheFull("sequence %d: %d rows are more than its %d pages hold" % (seq, end, self.max_pages))
            fresh[seq] = max(0, want - have)
            for at in range(self.rows[seq] // self.page_rows, min(have, want) if n else 0):
                page = self.held[seq][at]
                left = users.setdefault(page, self.users[page])
                if left > 1:   # the last one of those that write keeps the page
                    own[seq, at] = self.rows[seq] > at * self.page_rows
                    users[page] = left - 1
        total = sum(fresh.values()) + len(own)
        if total > len(self._free):
            raise CacheFull("%d pages are needed, %d are free" % (total, len(self._free)))
        copies = []
        for (seq, at), filled in own.items():
            new, old = heapq.heappop(self._free), self.held[seq][at]
            if filled:
                copies.append((old, new))
            self.users[new] = 1
            self.held[seq][at] = new
            self._drop(old)
        for seq, n in fresh.items():
            for _ in range(n):
                p = heapq.heappop(self._free)
                self.users[p] = 1
                self.held[seq].append(p)
        return copies

    def advance(self, seq, rows):
        """Rows that have been written (reserve() made room for them)."""
        self._known(seq)
        end = self.rows[seq] + rows
        if rows < 0 or end > len(self.held[seq]) * self.page_rows:
            raise ValueError("sequence %d has room for %d rows, not %d" % (seq, len(self.held[seq]) * self.page_rows, end))
        self.rows[seq] = end

    def compact(self):
        """Moves the pages in use to the lowest numbers.  Returns the (source, destination) pages to copy."""
        used = sum(1 for u in self.users if u)
        holes = [p for p in range(used) if not self.users[p]]
        moves = dict(zip([p for p in range(used, self.pages) if self.users[p]], holes))
        for old, new in moves.items():
            self.users[new], self.users[old] = self.users[old], 0
        for pages in self.held.values():
            pages[:] = [moves.get(p, p) for p in pages]
        self._free = list(range(used, self.pages))
        return list(moves.items())


class PagedKV8Cache:
    """The 8-bit cache of a model's layers.  layer(l) is what the ops.kv8_* calls take, batch(seqs) their page table and
    positions (columns without a page hold -1: rows that were not reserved are not written, and kernel_status says so).  A
    serving step: reserve({seq: rows}), then per layer kv8_step or kv8_append + kv8_attention, then advance().  max_seq: the rows a
    sequence may get to (None: all pages' rows).  It is what a batch's table has room for, and kernels are chosen by that: a
    server that knows its longest request says so."""

    def __init__(self, layers, pages, kv_heads, page_rows=64, max_seqs=64, max_seq=None, device="cuda"):
        if page_rows < 16 or page_rows & (page_rows - 1):
            raise ValueError("page_rows must be a power of two from 16, got %d" % page_rows)
        max_pages = pages if max_seq is None else -(-max_seq // page_rows)
        self.pool = PagePool(pages, page_rows, max_seqs, max_pages)
        z = lambda *shape, dt: torch.zeros(*shape, dtype=dt, device=device)  # noqa: E731
        self.k, self.v = (z(layers, pages, kv_heads, page_rows, 128, dt=torch.int8) for _ in range(2))
        self.k_scale, self.v_scale = (z(layers, pages, kv_heads, page_rows // 16, dt=torch.float32) for _ in range(2))
        self._layers = [(self.k[i], self.v[i], self.k_scale[i], self.v_scale[i]) for i in range(layers)]

    def layer(self, i):
        return self._layers[i]

    def _copy(self, pairs):
        if pairs:
            ops.kv_copy_pages([self.k, self.v, self.k_scale, self.v_scale], [a for a, _ in pairs], [b for _, b in pairs])

    def add(self):
        return self.pool.add()

    def fork(self, seq):
        return self.pool.fork(seq)

    def free(self, seq):
        self.pool.free(seq)

    def truncate(self, seq, rows):
        self.pool.truncate(seq, rows)

    def advance(self, seq, rows):
        self.pool.advance(seq, rows)

    def rows(self, seq):
        return self.pool.rows[seq]

    def reserve(self, need):
        self._copy(self.pool.reserve(need))

    def compact(self):
        moves = self.pool.compact()
        self._copy(moves)
        return len(moves)

    def batch(self, seqs):
        """(page_table int32 [len(seqs), max_pages], pos0 int32 [len(seqs)]) on the device: where the sequences' next rows go."""
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is in a batch once, got %r" % (list(seqs),))
        n, width, device = len(seqs), self.pool.max_pages, self.k.device
        if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("batch() is not captured: it uploads what the host knows now (call it before, and copy its result where the captured calls read)")
        # one upload, from pinned memory that torch keeps until the copy has run: nothing waits for the GPU
        host = torch.full((n * (width + 1),), -1, dtype=torch.int32, pin_memory=device.type == "cuda")
        table = host[:n * width].view(n, width)
        for i, s in enumerate(seqs):
            pages = self.pool.held[s]
            table[i, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        host[n * width:] = torch.tensor([self.pool.rows[s] for s in seqs], dtype=torch.int32)
        both = host.to(device, non_blocking=True)
        return both[:n * width].view(n, width), both[n * width:]
