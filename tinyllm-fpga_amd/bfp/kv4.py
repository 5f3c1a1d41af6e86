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

from . import _rows
from ._dev import _torch
from ._lib import Kv4BatchC, Kv4C, call, lib
from .rotary import check_table

TILE = 16


class Batch:
    """Which rows belong to which sequence, and where they are cached: row
    start[b] + i of the row arrays is a new token of sequence b, the last of
    them at position lens[b] - 1; position p lies in page pages[b, p // page].
    pages (sequences, width), start (sequences + 1) and lens are int32 tensors
    on the device; they are read when a call runs, so a program may write new
    values into them.  max_q: the most new rows a sequence has; max_len: the
    longest sequence (0: the table's width), which only chooses how the work
    is split."""

    def __init__(self, pages, start, lens, max_q, max_len=0):
        if pages.dim() != 2 or pages.shape[1] < 1:
            raise ValueError(f"pages has shape {tuple(pages.shape)}, not (sequences, width)")
        n = pages.shape[0]
        torch = _torch()
        for t, what, shape in ((pages, "pages", tuple(pages.shape)), (start, "start", (n + 1,)), (lens, "lens", (n,))):
            if tuple(t.shape) != shape or t.dtype != torch.int32 or not t.is_contiguous() or t.device != pages.device \
                    or not t.is_cuda:
                raise ValueError(f"{what} must be a contiguous int32 tensor {shape} on one GPU")
        if max_q < 0 or max_len < 0:
            raise ValueError(f"max_q={max_q}, max_len={max_len}")
        self.pages, self.start, self.lens = pages, start, lens
        self.max_q, self.max_len = int(max_q), int(max_len)
        self.device = pages.device

    def _c(self, n_rows):
        return Kv4BatchC(self.pages.data_ptr(), self.start.data_ptr(), self.lens.data_ptr(), self.pages.shape[0],
                         n_rows, self.pages.shape[1], self.max_q, self.max_len)


class Fp4Cache:
    """n_pages pages of `page` tokens of `heads` KV heads, hd wide, at 4.5
    bits a value.  Which sequence has which page is the program's to say
    (Batch.pages)."""

    def __init__(self, n_pages, page, heads, hd, device=None):
        torch = _torch()
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
        torch = _torch()
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
        self._c = Kv4C(k.data_ptr(), k_exp.data_ptr(), v.data_ptr(), v_exp.data_ptr(), n_pages, page, heads, self.hd)

    def _check(self, batch, shape, what, heads=None):
        if batch.device != self.device:
            raise ValueError(f"the batch is on {batch.device}, the cache on {self.device}")
        want = (self.heads if heads is None else heads, self.hd)
        if len(shape) != 3 or shape[1:] != want:
            raise ValueError(f"{what} has shape {shape}, not (rows, {want[0]}, {want[1]})")

    def append(self, batch, k, v, table=None, interleaved=False, pos=None, q=None, q_out=None):
        """Write the batch's new k and v (rows, heads, hd) into their slots,
        k rotated by rotary.rope_table's `table` (None: as it is) at its
        position in the cache, or at pos (int32 per row).  q (rows, query
        heads, hd): queries to rotate in the same launch; returned, in q_out
        or a new tensor of q's type (float32 for tiles) whose rows outside
        every sequence are undefined.  A row whose position is negative, or
        whose page is not one of the cache's, writes nothing, and its
        rotated query is zero."""
        kr, vr = _rows.rows(k, "k", self.device), _rows.rows(v, "v", self.device)
        shape = _rows.shape_of(k)
        self._check(batch, shape, "k")
        if _rows.shape_of(v) != shape:
            raise ValueError(f"k {shape} and v {_rows.shape_of(v)} differ")
        n = shape[0]
        qr = qo = None
        if q is not None:
            qr = _rows.rows(q, "q", self.device)
            qs = _rows.shape_of(q)
            if qs[0] != n or qs[2] != self.hd:
                raise ValueError(f"q has shape {qs}, not ({n}, heads, {self.hd})")
            if q_out is None:
                torch = _torch()
                q_out = torch.empty(qs, dtype=torch.float32 if isinstance(q, tuple) else q.dtype, device=self.device)
            elif _rows.shape_of(q_out) != qs:
                raise ValueError(f"q_out has shape {_rows.shape_of(q_out)}, not {qs}")
            qo = _rows.rows(q_out, "q_out", self.device)
        elif q_out is not None:
            raise ValueError("q_out without q")
        n_pos, rot = check_table(table, self.device) if table is not None else (0, 0)
        p = _rows.ints(pos, "pos", self.device, n) if pos is not None else None
        if n == 0:
            return q_out
        with _rows.on(self.device):
            call("bfp_kv4_append_d", C.byref(self._c), C.byref(batch._c(n)), C.byref(kr), C.byref(vr),
                 C.byref(qr) if qr is not None else None, C.byref(qo) if qo is not None else None, p,
                 table.data_ptr() if table is not None else None, n_pos, rot, 1 if interleaved else 0,
                 _rows.stream_of(self.device))
        return q_out

    def read(self, batch, n_rows=None, dtype=None, k=None, v=None):
        """The cached values of the batch's rows (what append wrote for
        them): n_rows rows of new tensors (n_rows, heads, hd) of dtype
        (float32), whose rows outside every sequence are undefined, or into
        k and v (either may be left out).  A row without a slot gives
        zeros."""
        torch = _torch()
        if k is None and v is None:
            if n_rows is None:
                raise ValueError("read needs n_rows, or tensors to read into")
            k, v = torch.empty(2, int(n_rows), self.heads, self.hd, dtype=dtype or torch.float32, device=self.device)
        n = (k if k is not None else v).shape[0]
        rs = []
        for t, what in ((k, "k"), (v, "v")):
            rs.append(None if t is None else _rows.rows(t, what, self.device))
            if t is not None:
                self._check(batch, _rows.shape_of(t), what)
                if t.shape[0] != n:
                    raise ValueError(f"k has {n} rows, v {t.shape[0]}")
        if n:
            with _rows.on(self.device):
                call("bfp_kv4_read_d", C.byref(self._c), C.byref(batch._c(n)),
                     *(None if r is None else C.byref(r) for r in rs), _rows.stream_of(self.device))
        return k, v

    def attend(self, batch, q, scale=None, window=0, out=None, dtype=None, work=None):
        """softmax(scale q k^T) v of every row of q (rows, query heads, hd)
        over its sequence's cached tokens up to its own, the last `window` of
        them (0: all).  scale: 1/sqrt(hd) by default.  Query heads share KV
        heads in groups of neighbours.  Returns out -- a tensor, or a pair
        (m, e) of 16-bit tiles -- or a new tensor of dtype (q's; float32 for
        tiles) whose rows outside every sequence are undefined.  A row that
        sees nothing is zero.  work: uint8 scratch of attend_work() bytes
        (allocated per call otherwise)."""
        torch = _torch()
        qr = _rows.rows(q, "q", self.device)
        shape = _rows.shape_of(q)
        self._check(batch, shape, "q", shape[1])
        if shape[1] % self.heads:
            raise ValueError(f"{shape[1]} query heads for {self.heads} KV heads")
        if out is None:
            out = torch.empty(shape, dtype=dtype or (torch.float32 if isinstance(q, tuple) else q.dtype),
                              device=self.device)
        elif _rows.shape_of(out) != shape:
            raise ValueError(f"out has shape {_rows.shape_of(out)}, not {shape}")
        orow = _rows.rows(out, "out", self.device)
        if shape[0] == 0:
            return out
        b = batch._c(shape[0])
        with _rows.on(self.device):
            if work is None:
                n = lib().bfp_kv4_attn_work(C.byref(self._c), C.byref(b), C.byref(qr), C.byref(orow), int(window))
                work = torch.empty(n, dtype=torch.uint8, device=self.device) if n else None
            elif work.device != self.device or not work.is_contiguous():
                raise ValueError(f"work must be a contiguous tensor on {self.device}")
            call("bfp_kv4_attn_d", C.byref(self._c), C.byref(b), C.byref(qr), C.byref(orow),
                 1.0 / math.sqrt(self.hd) if scale is None else float(scale), int(window),
                 work.data_ptr() if work is not None else None,
                 work.numel() * work.element_size() if work is not None else 0, _rows.stream_of(self.device))
        return out

    def attend_work(self, batch, q, out=None, dtype=None, window=0):
        """Scratch bytes attend() needs for such a call."""
        torch = _torch()
        qr = _rows.rows(q, "q", self.device)
        orow = _rows.rows(out if out is not None else torch.empty(
            _rows.shape_of(q), dtype=dtype or (torch.float32 if isinstance(q, tuple) else q.dtype),
            device=self.device), "out", self.device)
        return lib().bfp_kv4_attn_work(C.byref(self._c), C.byref(batch._c(_rows.shape_of(q)[0])), C.byref(qr),
                                       C.byref(orow), int(window))
