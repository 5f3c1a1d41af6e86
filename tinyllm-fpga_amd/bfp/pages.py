"""The pages of paged caches that share their tables: which are held, how
often, and their copies (include/bfp.h: struct bfp_pages).

    pool = PagePool([cache, ...])                  # a model's layers, and their PageBounds
    pool.reserve(batch)                            # pages for the batch's new rows, before append
    tables, lens = pool.fork(pages, lens, parents)     # branches: whole pages shared, the last one copied
    pool.free(tables)                              # given up
    live = pool.compact(pages, tables)             # the held pages become 0 .. live - 1

All of it runs on the device, in the order of the current stream, with no
copy to the host, so it can be captured into a graph.  Free pages are given
lowest number first, in the order of the tables' entries.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _rows
from ._lib import PageArrayC, PagesC, PageTableC, lib

_copy, _reserve, _fork, _free, _compact = (
    _rows.Entry(f"bfp_pages_{name}_d") for name in ("copy", "reserve", "fork", "free", "compact"))


class PagePool(_rows.Fixed):
    """Who holds the pages of `caches` (Fp4Cache and PageBounds objects of the
    same n_pages and page, on one GPU; one alone may stand for a list).
    refs (n_pages), int32 on the device: how many table entries hold each page
    -- zeros, or what a program passes and keeps.  short (1), int32: how many
    pages were asked for and not there, over all calls."""

    def __init__(self, caches, refs=None):
        caches = tuple(caches) if isinstance(caches, (list, tuple)) else (caches,)
        if not caches:
            raise ValueError("a pool needs a cache")
        first = caches[0]
        for c in caches:
            if (c.n_pages, c.page, c.device) != (first.n_pages, first.page, first.device):
                raise ValueError(f"a cache has {c.n_pages} pages of {c.page} tokens on {c.device}, the first "
                                 f"{first.n_pages} of {first.page} on {first.device}")
        self.caches, self.n_pages, self.page, self.device = caches, first.n_pages, first.page, first.device
        if refs is None:
            refs = torch.zeros(self.n_pages, dtype=torch.int32, device=self.device)
        else:
            _rows.ints(refs, "refs", self.device, self.n_pages)
        self.refs, self.short = refs, torch.zeros(1, dtype=torch.int32, device=self.device)
        arrays = [a for c in caches for a in c._page_arrays()]
        self._arrays = (PageArrayC * len(arrays))(*arrays)
        self._made = PagesC(refs.data_ptr(), self.short.data_ptr(), self._arrays, self.n_pages, self.page, len(arrays))
        self._c = C.byref(self._made)
        self._size = lib().bfp_pages_work(self._c, 0)

    def _table(self, t, what):
        if t.dim() != 2 or t.shape[1] < 1 or t.dtype != torch.int32 or not t.is_contiguous() or t.device != self.device:
            raise ValueError(f"{what} must be a contiguous int32 tensor (sequences, width) on {self.device}")
        return t.data_ptr(), t.shape[0], t.shape[1]

    def _work(self, work, n=0):
        """Scratch for n children: its address and size (and itself, to live until the call is made)."""
        size = self._size + 8 * n
        if work is None:
            work = torch.empty(size, dtype=torch.uint8, device=self.device)
        else:
            size = _rows.scratch(work, self.device)
        return work, work.data_ptr(), size

    def work(self, n=0):
        """Scratch bytes fork() needs for n children, and the other calls for 0."""
        return lib().bfp_pages_work(self._c, _rows.c_int(n, "n"))

    def copy(self, src, dst):
        """Page src[i] of every cache to page dst[i] (int32 vectors).  No page
        may be in dst twice, or in both; a pair with a page outside the pool
        copies nothing."""
        n = src.shape[0] if src.dim() == 1 else -1
        s, d = (_rows.ints(t, what, self.device, n) for t, what in ((src, "src"), (dst, "dst")))
        if n:
            _copy(self.device, self._c, s, d, n)

    def reserve(self, batch, work=None):
        """A page for every entry of batch.pages that the batch's new rows lie
        in and that holds none (is outside [0, n_pages)): before append.  An
        entry for which none is left becomes -1, and its rows have no slot:
        once they have been appended the sequence is given up, or goes on
        from its last whole page (a page that the entry is given later does
        not hold them, but whatever was there).
        A page that another entry holds too is not replaced: fork a sequence
        that is cut back into one before it goes on."""
        if batch.device != self.device:
            raise ValueError(f"the batch is on {batch.device}, the pool on {self.device}")
        keep, p, size = self._work(work)
        _reserve(self.device, self._c, batch._c(None), p, size)

    def fork(self, pages, lens, parents, out=None, work=None):
        """Branches: row i of the result goes on from sequence parents[i] of
        pages (sequences, width), of which lens tokens are cached.  Whole pages
        are shared; the page in which the tokens end is copied to one of its
        own, in every cache.  Entries past those are -1.  Where no page was
        left for the copy, its entry is -1 and the branch's length ends with
        the whole pages.  A parent that does not exist gives an empty row.
        Returns (pages, lens), new tensors or `out`'s, whose pages are not
        given up first: free() them before."""
        p, n_seq, width = self._table(pages, "pages")
        ln = _rows.ints(lens, "lens", self.device, n_seq)
        n = parents.shape[0] if parents.dim() == 1 else -1
        pa = _rows.ints(parents, "parents", self.device, n)
        if out is None:
            out = (torch.empty((n, width), dtype=torch.int32, device=self.device),
                   torch.empty((n,), dtype=torch.int32, device=self.device))
        op, rows, out_width = self._table(out[0], "out's pages")
        if rows != n:
            raise ValueError(f"out has {rows} rows for {n} parents")
        ol = _rows.ints(out[1], "out's lens", self.device, n)
        if n:
            keep, w, size = self._work(work, n)
            _fork(self.device, self._c, p, ln, n_seq, width, pa, n, op, ol, out_width, w, size)
        return out

    def free(self, pages):
        """Give up what a table (sequences, width) holds, or a contiguous part
        of one (pages[b:b + 1]): its entries become -1."""
        p, n, width = self._table(pages, "pages")
        if n:
            _free(self.device, self._c, p, n * width)

    def compact(self, *tables, work=None):
        """Move the held pages into the lowest ones and rewrite `tables` (at
        most 16: all that hold any; entries with a free page become -1).
        Returns the held pages' number, an int32 tensor (1) on the device:
        pages from there on are free."""
        ts = (PageTableC * max(len(tables), 1))()
        for i, t in enumerate(tables):
            p, n, width = self._table(t, f"table {i}")
            ts[i] = PageTableC(p, n * width)
        live = torch.empty(1, dtype=torch.int32, device=self.device)
        keep, w, size = self._work(work)
        _compact(self.device, self._c, ts, len(tables), live.data_ptr(), w, size)
        return live
