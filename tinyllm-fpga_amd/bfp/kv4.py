"""The paged key/value cache in 4 bits and the attention over it, on device
tensors (include/bfp.h: struct bfp_kv4, struct bfp_kv4_batch).

    cache = Fp4Cache(n_pages, page=64, heads=3, hd=64)
    batch = Batch(pages, start, lens, max_q=1, max_len=2048)
    q = cache.append(batch, k, v, table, q=q)      # rotate, write the new tokens
    out = cache.attend(batch, q)                   # rows x query heads x hd

Rows are tensors (rows, heads, hd) in float32, bfloat16 or float16, or pairs
(m, e) of 16-bit tiles as the matvecs leave them.  Calls are queued on the
current stream of the cache's device, make no copies to the host and check
only what the host knows: page numbers and lengths are bounded on the device.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _rows
from ._lib import Kv4BatchC, Kv4C, lib
from .rotary import check_table

TILE = 16
_append, _read, _attend = (_rows.Entry(f"bfp_kv4_{name}_d") for name in ("append", "read", "attn"))


def _window(n):
    return _rows.c_int(n, "window", -1 - _rows.MAX_INT)   # negative ones are the entry point's to refuse


class Batch(_rows.Fixed):
    """Which rows belong to which sequence, and where they are cached: row
    start[b] + i of the row arrays is a new token of sequence b, the last of
    them at position lens[b] - 1; position p lies in page pages[b, p // page].
    pages (sequences, width), start (sequences + 1) and lens are int32 tensors
    on the device; they are read when a call runs, so a program may write new
    values into them (batch.lens += 1, but not put other tensors in their
    place).  max_q: the most new rows a sequence has; max_len: the longest
    sequence (0: the table's width), which only chooses how the work is
    split."""

    def __init__(self, pages, start, lens, max_q, max_len=0):
        if pages.dim() != 2 or pages.shape[1] < 1:
            raise ValueError(f"pages has shape {tuple(pages.shape)}, not (sequences, width)")
        n = pages.shape[0]
        for t, what, shape in ((pages, "pages", tuple(pages.shape)), (start, "start", (n + 1,)), (lens, "lens", (n,))):
            if tuple(t.shape) != shape or t.dtype != torch.int32 or not t.is_contiguous() or t.device != pages.device \
                    or not t.is_cuda:
                raise ValueError(f"{what} must be a contiguous int32 tensor {shape} on one GPU")
        self.pages, self.start, self.lens = pages, start, lens
        self.max_q, self.max_len = _rows.c_int(max_q, "max_q"), _rows.c_int(max_len, "max_len")
        self.device = pages.device
        self._made = (-1, None)

    def _c(self, n_rows):
        """The struct for row arrays of n_rows (this object keeps the tensors
        it points to)."""
        n, c = self._made
        if n != n_rows:
            if not 0 <= n_rows <= _rows.MAX_ROWS:
                raise ValueError(f"{n_rows} rows")
            c = Kv4BatchC(self.pages.data_ptr(), self.start.data_ptr(), self.lens.data_ptr(), self.pages.shape[0],
                          n_rows, self.pages.shape[1], self.max_q, self.max_len)
            self._made = (n_rows, c)
        return C.byref(c)


class Fp4Cache(_rows.Fixed):
    """n_pages pages of `page` tokens of `heads` KV heads, hd wide, at 4.5
    bits a value.  Which sequence has which page is the program's to say
    (Batch.pages)."""

    def __init__(self, n_pages, page, heads, hd, device=None):
        if n_pages < 1 or heads < 1 or hd < TILE or hd % TILE:
            raise ValueError(f"n_pages={n_pages}, heads={heads}, hd={hd} (a multiple of {TILE})")
        device = torch.device("cuda" if device is None else device)
        shape = (n_pages, heads, hd // TILE, page)
        new = lambda *n: torch.zeros(*shape, *n, dtype=torch.uint8, device=device)  # noqa: E731
        self._set(new(TILE // 2), new(), new(TILE // 2), new())

    @classmethod
    def from_buffers(cls, k, k_exp, v, v_exp):
        """A cache over existing memory: k, v uint8 (n_pages, heads, hd/16,
        page, 8), k_exp, v_exp uint8 (n_pages, heads, hd/16, page)."""
        self = cls.__new__(cls)
        self._set(k, k_exp, v, v_exp)
        return self

    def _set(self, k, k_exp, v, v_exp):
        if k.dim() != 5 or k.shape[4] != TILE // 2:
            raise ValueError(f"k has shape {tuple(k.shape)}, not (n_pages, heads, hd/16, page, 8)")
        for t, what, shape in ((k, "k", k.shape), (v, "v", k.shape), (k_exp, "k_exp", k.shape[:4]),
                               (v_exp, "v_exp", k.shape[:4])):
            if t.shape != shape or t.dtype != torch.uint8 or not t.is_contiguous() or not t.is_cuda \
                    or t.device != k.device:
                raise ValueError(f"{what} must be a contiguous uint8 tensor {tuple(shape)} on one GPU")
        n_pages, heads, tiles, page, _ = k.shape
        if page not in (16, 32, 64, 128, 256) or tiles > 16:
            raise ValueError(f"page={page} must be 16, 32, 64, 128 or 256, and hd={tiles * TILE} at most 256")
        self.k, self.k_exp, self.v, self.v_exp = k, k_exp, v, v_exp
        self.n_pages, self.heads, self.hd, self.page = n_pages, heads, tiles * TILE, page
        self.device = k.device
        self._scale = 1.0 / math.sqrt(self.hd)
        self._made = Kv4C(k.data_ptr(), k_exp.data_ptr(), v.data_ptr(), v_exp.data_ptr(), n_pages, page, heads, self.hd)
        self._c = C.byref(self._made)

    def _values(self, batch, x, what):
        """x's values, checked against the batch and the head width."""
        if batch.device != self.device:
            raise ValueError(f"the batch is on {batch.device}, the cache on {self.device}")
        t = _rows.values_of(x, what)
        if t.shape[2] != self.hd:
            raise ValueError(f"{what} has shape {tuple(t.shape)}, not (rows, heads, {self.hd})")
        return t

    def append(self, batch, k, v, table=None, interleaved=False, pos=None, q=None, q_out=None):
        """Write the batch's new k and v (rows, heads, hd) into their slots,
        k rotated by rotary.rope_table's `table` (None: as it is) at its
        position in the cache, or at pos (int32 per row).  q (rows, query
        heads, hd): queries to rotate in the same launch; returned, in q_out
        or a new tensor of q's type (float32 for tiles) whose rows outside
        every sequence are undefined.  A row whose position is negative, or
        whose page is not one of the cache's, writes nothing, and its
        rotated query is zero.  q_out may be q."""
        dev = self.device
        kt, vt = self._values(batch, k, "k"), self._values(batch, v, "v")
        n = kt.shape[0]
        if kt.shape[1] != self.heads or vt.shape != kt.shape:
            raise ValueError(f"k {tuple(kt.shape)} and v {tuple(vt.shape)} must both be (rows, {self.heads}, {self.hd})")
        kr, vr = _rows.rows(k, "k", dev), _rows.rows(v, "v", dev)
        qb = ob = None
        if q is not None:
            qt = self._values(batch, q, "q")
            if qt.shape[0] != n:
                raise ValueError(f"q has {qt.shape[0]} rows, k {n}")
            qr = _rows.rows(q, "q", dev)
            if q_out is None:
                q_out, qo = _rows.new(q, qt, None)
            elif type(q_out) is tuple or q_out.shape != qt.shape:
                raise ValueError(f"q_out must be a tensor {tuple(qt.shape)}")
            else:
                qo = _rows.rows(q_out, "q_out", dev)
            qb, ob = C.byref(qr), C.byref(qo)
        elif q_out is not None:
            raise ValueError("q_out without q")
        tp, n_pos, rot = None, 0, 0
        if table is not None:
            n_pos, rot = check_table(table, dev)
            tp = table.data_ptr()
        p = _rows.ints(pos, "pos", dev, n) if pos is not None else None
        if n:
            _append(dev, self._c, batch._c(n), C.byref(kr), C.byref(vr), qb, ob, p, tp, n_pos, rot,
                    1 if interleaved else 0)
        return q_out

    def read(self, batch, n_rows=None, dtype=None, k=None, v=None):
        """The cached values of the batch's rows (what append wrote for
        them): n_rows rows of new tensors (n_rows, heads, hd) of dtype
        (float32), whose rows outside every sequence are undefined, or into
        k and v (either may be left out).  A row without a slot gives
        zeros."""
        if k is None and v is None:
            if n_rows is None:
                raise ValueError("read needs n_rows, or tensors to read into")
            k, kr = _rows.empty(int(n_rows), self.heads, self.hd, dtype, self.device)
            v, vr = _rows.empty(int(n_rows), self.heads, self.hd, dtype, self.device)
            if batch.device != self.device:
                raise ValueError(f"the batch is on {batch.device}, the cache on {self.device}")
            if n_rows:
                _read(self.device, self._c, batch._c(int(n_rows)), C.byref(kr), C.byref(vr))
            return k, v
        n, rs = None if n_rows is None else int(n_rows), []
        for x, what in ((k, "k"), (v, "v")):
            if x is None:
                rs.append(None)
                continue
            t = self._values(batch, x, what)
            if t.shape[1] != self.heads or n not in (None, t.shape[0]):
                raise ValueError(f"{what} has shape {tuple(t.shape)}, not ({'rows' if n is None else n}, {self.heads}, {self.hd})")
            if dtype is not None and t.dtype != dtype:
                raise ValueError(f"{what} is not of {dtype}")
            n = t.shape[0]
            rs.append(C.byref(_rows.rows(x, what, self.device)))
        if n:
            _read(self.device, self._c, batch._c(n), *rs)
        return k, v

    def attend(self, batch, q, scale=None, window=0, out=None, dtype=None, work=None):
        """softmax(scale q k^T) v of every row of q (rows, query heads, hd)
        over its sequence's cached tokens up to its own, the last `window` of
        them (0: all).  scale: 1/sqrt(hd) by default.  Query heads share KV
        heads in groups of neighbours.  Returns out -- a tensor, or a pair
        (m, e) of 16-bit tiles -- or a new tensor of dtype (q's; float32 for
        tiles) whose rows outside every sequence are undefined.  A row that
        sees nothing is zero; tiles hold a NaN as -2^127.  Probabilities are
        carried to at least the result's precision: bfloat16 calls of many
        rows round them to bfloat16, dtype=torch.float32 keeps them whole.
        work: uint8 scratch of attend_work() bytes (allocated per call
        otherwise)."""
        dev = self.device
        t, qr, out, orow = self._attend_rows(batch, q, out, dtype)
        n = t.shape[0]
        if n == 0:
            return out
        b, qb, ob, window = batch._c(n), C.byref(qr), C.byref(orow), _window(window)
        if work is None:
            size = lib().bfp_kv4_attn_work(self._c, b, qb, ob, window)
            if size:
                work = torch.empty(size, dtype=torch.uint8, device=dev)
        elif work.device != dev or not work.is_contiguous():
            raise ValueError(f"work must be a contiguous tensor on {dev}")
        else:
            size = work.numel() * work.element_size()
        _attend(dev, self._c, b, qb, ob, self._scale if scale is None else float(scale), window,
                work.data_ptr() if work is not None else None, size)
        return out

    def _attend_rows(self, batch, q, out, dtype, make=True):
        t = self._values(batch, q, "q")
        heads = t.shape[1]
        if heads % self.heads or not heads:
            raise ValueError(f"{heads} query heads for {self.heads} KV heads")
        qr = _rows.rows(q, "q", self.device)
        if out is None:
            out, orow = _rows.new(q, t, dtype) if make else _rows.like(q, t, dtype)
        else:
            if self._values(batch, out, "out").shape != t.shape:
                raise ValueError(f"out must be {tuple(t.shape)}")
            if dtype is not None and (type(out) is tuple or out.dtype != dtype):
                raise ValueError(f"out is not of {dtype}")
            orow = _rows.rows(out, "out", self.device)
        return t, qr, out, orow

    def attend_work(self, batch, q, out=None, dtype=None, window=0):
        """Scratch bytes attend() needs for such a call."""
        t, qr, _, orow = self._attend_rows(batch, q, out, dtype, make=False)
        orow.p = orow.p or 16   # the size depends on no address
        return lib().bfp_kv4_attn_work(self._c, batch._c(t.shape[0]), C.byref(qr), C.byref(orow), _window(window))
