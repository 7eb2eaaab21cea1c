"""Which pages of a paged cache belong to whom: the host's book beside bonsai_b200_pages (include/bonsai_b200_ext.h).

A sequence's positions lie in pages of 64.  A fork shares every page of the sequence that it continues; the page that a sequence is about
to write to and does not have to itself is replaced by a copy first.  The book says which pages to copy (`pages_copy`); it
touches no device memory, and nothing happens to it when a call is refused.
"""
from bonsai_b200 import PAGE_POSITIONS


class NoRoom(RuntimeError):
    """There are not as many free pages as asked for.  The book is as it was."""


class PageBook:
    def __init__(self, n_pages):
        if n_pages <= 0:
            raise ValueError("a pool has pages")
        self.users = [0] * n_pages                      # sequences that hold the page
        self._free = list(range(n_pages - 1, -1, -1))
        self._seqs = {}                                 # name -> [pages, positions]
        self._next = 0

    # ---- what there is
    @property
    def free_pages(self):
        return len(self._free)

    def pages(self, seq):
        return list(self._seqs[seq][0])

    def length(self, seq):
        return self._seqs[seq][1]

    def tables(self, seqs, stride=None):
        """(table rows filled up with 0, lengths) of the sequences, as lists of ints."""
        stride = stride or max([1] + [len(self._seqs[s][0]) for s in seqs])
        rows = [self._seqs[s][0] for s in seqs]
        if any(len(r) > stride for r in rows):
            raise ValueError("a sequence has more pages than the table's rows")
        return [r + [0] * (stride - len(r)) for r in rows], [self._seqs[s][1] for s in seqs]

    # ---- what changes it
    def new(self):
        """An empty sequence's name."""
        self._next += 1
        self._seqs[self._next] = [[], 0]
        return self._next

    def extend(self, seq, n_tok):
        """Room for n_tok more positions.  Returns the copies (source pages, destination pages) to be made before anything is appended."""
        if n_tok < 0:
            raise ValueError("truncate() shortens a sequence")
        pages, length = self._seqs[seq]
        if n_tok == 0:
            return [], []
        shared = bool(length % PAGE_POSITIONS) and self.users[pages[length // PAGE_POSITIONS]] > 1
        need = -(-(length + n_tok) // PAGE_POSITIONS) - len(pages)
        if need + shared > len(self._free):
            raise NoRoom(f"{need + shared} pages asked for, {len(self._free)} free")
        src, dst = [], []
        if shared:
            at = length // PAGE_POSITIONS
            src, dst = [pages[at]], [self._take()]
            self._drop(pages[at])
            pages[at] = dst[0]
        pages += [self._take() for _ in range(need)]
        self._seqs[seq][1] = length + n_tok
        return src, dst

    def fork(self, seq):
        """A sequence that continues this one, every page shared."""
        pages, length = self._seqs[seq]
        other = self.new()
        for p in pages:
            self.users[p] += 1
        self._seqs[other] = [list(pages), length]
        return other

    def truncate(self, seq, length):
        """Forgets the positions from `length` on (drafted tokens that were not taken)."""
        pages, now = self._seqs[seq]
        if not 0 <= length <= now:
            raise ValueError(f"the sequence has {now} positions")
        keep = -(-length // PAGE_POSITIONS)
        for p in pages[keep:]:
            self._drop(p)
        self._seqs[seq] = [pages[:keep], length]

    def free(self, seq):
        self.truncate(seq, 0)
        del self._seqs[seq]

    def compact(self):
        """Moves the pages in use to the front of the pool.  Returns the copies to be made before the next call that uses the cache; no page is both a source and
        a destination."""
        used = sorted(p for p, n in enumerate(self.users) if n)
        src = [p for p in used if p >= len(used)]
        dst = sorted(self._free)[:len(src)]
        to = dict(zip(src, dst))
        for s, d in to.items():
            self.users[d], self.users[s] = self.users[s], 0
        for entry in self._seqs.values():
            entry[0] = [to.get(p, p) for p in entry[0]]
        self._free = list(range(len(self.users) - 1, len(used) - 1, -1))
        return src, dst

    def _take(self):
        p = self._free.pop()
        self.users[p] = 1
        return p

    def _drop(self, p):
        self.users[p] -= 1
        if self.users[p] == 0:
            self._free.append(p)
