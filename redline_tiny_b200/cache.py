"""The pages of an 8-bit cache of keys and values, and the sequences that live in them.

`PagedKV` owns a pool (ops.KVPool) and keeps its books on the host: which pages a sequence has, how many sequences share a
page, which are free. Forking a sequence copies nothing; a page that several sequences share is copied when one of them
first writes into it, all such copies of a step in one launch. Batches carry the page tables and lengths in device memory
at fixed addresses, so a captured decode step follows them when it is replayed.

    kv = PagedKV(layers=36, pages=4096, kv_heads=8)
    a = kv.new()
    batch = kv.batch([a])
    batch.extend([len(prompt)])                 # pages for the new tokens; raises (and changes nothing) without room
    ops.kv_append(kv.pool, layer, k, v, *batch.args)
    o = ops.kv_attention(q, kv.pool, layer, *batch.args)
    b = kv.fork(a)                              # b continues where a stands
    kv.free(a)
"""

import heapq

import torch

from . import ops


def _not_captured(what):
    """The books move on the host when the call is made, not when a captured graph is replayed."""
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} keeps books on the host and cannot be captured into a graph")


class OutOfPages(RuntimeError):
    """The pool has fewer free pages than a step needs; nothing was changed."""


class PagedKV:
    def __init__(self, layers, pages, kv_heads, page=64, device="cuda"):
        self.pool = ops.KVPool.empty(layers, pages, kv_heads, page, device)
        self.page = page
        self.refs = [0] * pages            # sequences that hold the page
        self._free = list(range(pages))    # a heap: the lowest page is taken first
        self._seqs = {}                    # sequence -> its pages in order
        self._len = {}
        self._next = 0
        self._version = 0                  # grows when any sequence's pages or length change
        self._stamp = {}                   # sequence -> the version of its last change: what a batch's tables go by

    # -- books ------------------------------------------------------------------------------------------------------
    def new(self):
        """An empty sequence."""
        s = self._next
        self._next += 1
        self._seqs[s], self._len[s], self._stamp[s] = [], 0, self._version
        return s

    def fork(self, seq):
        """A sequence that continues where `seq` stands, sharing all its pages."""
        length, pages = self.length(seq), self._seqs[seq]
        s = self.new()
        self._seqs[s], self._len[s] = list(pages), length
        for p in pages:
            self.refs[p] += 1
        return s

    def free(self, seq):
        """Give up a sequence; pages that no other sequence holds are free again."""
        self.length(seq)
        self._release(self._seqs.pop(seq))
        del self._len[seq], self._stamp[seq]
        self._version += 1

    def truncate(self, seq, length):
        """Forget the tokens from position `length` on."""
        if not 0 <= length <= self.length(seq):
            raise ValueError(f"sequence {seq} has {self._len[seq]} tokens")
        pages, keep = self._seqs[seq], -(-length // self.page)
        self._release(pages[keep:])
        del pages[keep:]
        if length != self._len[seq]:
            self._len[seq] = length
            self._changed([seq])

    def _changed(self, seqs):
        self._version += 1
        for s in seqs:
            self._stamp[s] = self._version

    def _release(self, pages):
        for p in pages:
            self.refs[p] -= 1
            if self.refs[p] == 0:
                heapq.heappush(self._free, p)

    def length(self, seq):
        if seq not in self._len:
            raise ValueError(f"no sequence {seq} in this cache")
        return self._len[seq]

    def pages(self, seq):
        return tuple(self._seqs[seq])

    @property
    def free_pages(self):
        return len(self._free)

    # -- steps ------------------------------------------------------------------------------------------------------
    def batch(self, seqs, max_pages=None):
        """A batch of up to 1024 different sequences; `max_pages` bounds the pages of each (default: the whole pool). Attention
        over short contexts is faster where that bound is at most 6144 tokens (777 keys: 5.6 against 7.0 us)."""
        return Batch(self, seqs, max_pages or len(self.refs))

    def _plan(self, seqs, counts):
        """What room for counts[i] more tokens of seqs[i] takes, with nothing changed: per sequence (the page that its tail
        moves to or None, new pages), and the (page, its private copy) pairs to copy first."""
        fresh, shared = 0, {}
        for s, n in zip(seqs, counts):
            if n < 0:
                raise ValueError(f"{n} new tokens")
            have, pages = self._len[s], self._seqs[s]
            fresh += -(-(have + n) // self.page) - len(pages)
            if n and have % self.page and self.refs[pages[-1]] > 1:   # the page it continues in is shared
                p = pages[-1]
                shared[p] = shared.get(p, 0) + 1
        # the last holder of a page keeps it when every holder writes into it
        copies_needed = sum(min(c, self.refs[p] - 1) for p, c in shared.items())
        if fresh + copies_needed > len(self._free):
            raise OutOfPages(f"{fresh + copies_needed} pages needed, {len(self._free)} free")
        take = iter(heapq.nsmallest(fresh + copies_needed, self._free))
        holders, moves, copies = {}, [], []
        for s, n in zip(seqs, counts):
            have, pages, tail = self._len[s], self._seqs[s], None
            if n and have % self.page:
                p = pages[-1]
                left = holders.get(p, self.refs[p])
                if left > 1:
                    holders[p], tail = left - 1, next(take)
                    copies.append((p, tail))
            moves.append((tail, [next(take) for _ in range(-(-(have + n) // self.page) - len(pages))]))
        return moves, copies

    def _commit(self, seqs, counts, moves):
        for s, n, (tail, more) in zip(seqs, counts, moves):
            pages = self._seqs[s]
            if tail is not None:
                self.refs[pages[-1]] -= 1
                pages[-1] = tail
            pages += more
            for p in more if tail is None else [tail, *more]:
                self.refs[p] = 1
                heapq.heappop(self._free)          # (the plan took the lowest)
            self._len[s] += n
        self._changed([s for s, n in zip(seqs, counts) if n])

    def compact(self):
        """Move the live pages to the front of the pool, so that its tail can be given back (resize). Returns the number
        of pages moved. A batch whose pages moved follows at its next `extend` (of no tokens, if need be), not before."""
        _not_captured("compact")
        live = [p for p, r in enumerate(self.refs) if r]
        n = len(live)
        to = dict(zip([p for p in live if p >= n], [p for p in range(n) if not self.refs[p]]))
        if to:
            ops.kv_copy_pages(self.pool, list(to.keys()), list(to.values()))
            for p, q in to.items():
                self.refs[q], self.refs[p] = self.refs[p], 0
            self._changed([s for s, pages in self._seqs.items() if any(p in to for p in pages)])
            for pages in self._seqs.values():
                pages[:] = [to.get(p, p) for p in pages]
            self._free = list(range(n, len(self.refs)))
        return len(to)

    def resize(self, pages):
        """A pool of `pages` pages (compacted first when that drops any). The old pool's memory is given up: steps captured
        before must not be replayed."""
        _not_captured("resize")
        if pages < len(self.refs):
            if pages < sum(1 for r in self.refs if r):
                raise OutOfPages(f"{sum(1 for r in self.refs if r)} pages are in use")
            self.compact()
        old, n = self.pool, min(pages, len(self.refs))
        self.pool = ops.KVPool.empty(old.layers, pages, old.kv_heads, old.page, old.k.device)
        for a, b in zip((self.pool.k, self.pool.v, self.pool.k_exp, self.pool.v_exp),
                        (old.k, old.v, old.k_exp, old.v_exp)):
            a[:, :n].copy_(b[:, :n])
        self.refs = self.refs[:pages] + [0] * (pages - len(self.refs))
        self._free = [p for p, r in enumerate(self.refs) if not r]


class Batch:
    """Sequences that take steps together. `args` = (table, kv_len, q_start): the device arrays that ops.kv_append and
    ops.kv_attention take, at addresses that never change. They hold what the last `extend` left: once a sequence's pages
    or length have changed otherwise (another batch's extend, truncate, free, compact), `args` raises until the next. A
    captured step reads the arrays as they are when it is replayed: extend comes before each replay."""

    def __init__(self, kv, seqs, max_pages):
        self.kv, self.seqs = kv, list(seqs)
        if len(set(self.seqs)) != len(self.seqs):
            raise ValueError("a sequence appears twice in a batch")
        if len(self.seqs) > ops.KV_SEQUENCES:     # (the kernels' limit, before the books depend on it)
            raise ValueError(f"{len(self.seqs)} sequences in a batch (at most {ops.KV_SEQUENCES})")
        if max_pages < 1 or max_pages * kv.page > ops.KV_TOKENS:
            raise ValueError(f"{max_pages} pages a sequence (1 to {ops.KV_TOKENS // kv.page})")
        for s in self.seqs:
            kv.length(s)
        B, self.width = len(self.seqs), int(max_pages)
        dev = kv.pool.k.device
        self._meta = torch.full((B * self.width + 2 * B + 1,), -1, dtype=torch.int32, device=dev)
        self._meta[B * self.width:] = 0
        self._written = [[] for _ in self.seqs]      # what the device tables hold
        self._lens, self._starts, self._rows = [0] * B, [0] * (B + 1), 0
        self._version, self._stamps = kv._version, [kv._stamp[s] for s in self.seqs]
        self.table = self._meta[:B * self.width].view(B, self.width)
        self.kv_len = self._meta[B * self.width:B * self.width + B]
        self.q_start = self._meta[B * self.width + B:]

    @property
    def args(self):
        if self._version != self.kv._version:
            for s, t in zip(self.seqs, self._stamps):
                if self.kv._stamp.get(s) != t:
                    raise RuntimeError(f"the pages or the length of sequence {s} have moved since this batch's last extend")
            self._version = self.kv._version
        return self.table, self.kv_len, self.q_start

    @property
    def rows(self):
        """New tokens of the last extend."""
        return self._rows

    def extend(self, counts):
        """Make room for counts[i] new tokens of each sequence and point the device arrays at them: pages are taken,
        shared pages that will be written are copied. Raises OutOfPages where the pool is full; an extend that raises leaves
        the cache's books as they were."""
        _not_captured("extend")
        counts = list(counts)
        kv, B = self.kv, len(self.seqs)
        if len(counts) != B:
            raise ValueError(f"{len(counts)} counts for {B} sequences")
        for s, n in zip(self.seqs, counts):
            need = -(-(kv.length(s) + n) // kv.page)
            if need > len(kv.refs):
                raise OutOfPages(f"sequence {s} needs {need} pages of a pool of {len(kv.refs)}")
            if need > self.width:
                raise ValueError(f"sequence {s} would need more than the batch's {self.width} pages a sequence")
        moves, copies = kv._plan(self.seqs, counts)
        # the device first, the books when all its calls have been taken
        if copies:
            ops.kv_copy_pages(kv.pool, [a for a, _ in copies], [b for _, b in copies])
        entries, current, lens, starts = self._entries(counts, moves)
        if entries:
            try:
                ops.kv_set(self._meta, entries)
            except Exception:
                self._forget()
                raise
        kv._commit(self.seqs, counts, moves)
        for b, (tail, more) in enumerate(moves):
            row = self._written[b]
            if not current[b]:
                row[:] = kv._seqs[self.seqs[b]]
            else:
                if tail is not None:
                    row[-1] = tail
                if more:
                    row += more
        self._lens, self._starts, self._rows = lens, starts, starts[-1]
        self._version, self._stamps = kv._version, [kv._stamp[s] for s in self.seqs]

    def _forget(self):
        """What the device arrays hold is not known: `args` raises, and the next extend writes them whole."""
        B = len(self.seqs)
        self._written, self._lens, self._starts = [[] for _ in range(B)], [None] * B, [None] * (B + 1)
        self._version, self._stamps = None, [None] * B

    def _entries(self, counts, moves):
        """The entries of the device arrays that the planned step changes, and the lengths and row ranges that follow."""
        kv, W, at, new, current, lens, starts = self.kv, self.width, 0, {}, [], [], [0]
        for s, n, (tail, more), have, stamp in zip(self.seqs, counts, moves, self._written, self._stamps):
            pages = kv._seqs[s]
            k = len(pages)
            same = stamp == kv._stamp[s] and len(have) == k          # the row holds the sequence's pages
            if not same:
                new.update((at + i, p) for i, p in enumerate(pages) if i >= len(have) or have[i] != p)
            if tail is not None:
                new[at + k - 1] = tail
            for i, p in enumerate(more, at + k):
                new[i] = p
            at += W
            current.append(same)
            lens.append(kv._len[s] + n)
            starts.append(starts[-1] + n)
        new.update((at + i, v) for i, (v, old) in enumerate(zip(lens + starts, self._lens + self._starts)) if v != old)
        return new, current, lens, starts
