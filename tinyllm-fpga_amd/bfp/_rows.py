"""Rows of heads on the device: torch tensors (rows, heads, hd), or pairs
(m, e) of 16-bit tiles, as the C entry points take them (struct bfp_rows).

A decode step makes these calls once a layer, so what a call costs on the
host is part of its latency: the checks read each tensor property once, and
the stream is taken as the raw handle (0.1 us; the Stream object costs 1.8).
"""
from __future__ import annotations

import torch

from ._dev import _torch as _need_gpu
from ._lib import RowsC, check, lib

TILE = 16
F32, BF16, F16, TILES = range(4)
TYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}

_current_device = torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
if _raw_stream is None:
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream


def values_of(x, what: str):
    """The tensor that holds x's values (a pair's mantissas)."""
    t = x[0] if type(x) is tuple and len(x) == 2 else x
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{what} must be a tensor (rows, heads, hd) or a pair (m, e) of them")
    return t


def rows(x, what: str, device) -> RowsC:
    """The RowsC of x, which has passed values_of; ValueError where it is not
    rows of heads on `device`.  The struct holds no reference: x has to live
    until the call is made."""
    if type(x) is tuple:
        return _tiles(x, what, device)
    kind = TYPES.get(x.dtype)
    if kind is None:
        raise ValueError(f"{what} has type {x.dtype}: float32, bfloat16, float16, or a pair (m, e) of "
                         "int16 mantissas and int8 exponents")
    if x.device != device:
        raise ValueError(f"{what} is on {x.device}, not on {device}")
    rs, hs, ds = x.stride()
    if ds != 1 and x.shape[2] > 1:
        raise ValueError(f"{what}: the values of a head must be contiguous")
    return RowsC(x.data_ptr(), None, kind, x.shape[1], rs, hs)


def _tiles(x, what, device):
    t, e = x
    n, heads, hd = t.shape
    if not isinstance(e, torch.Tensor) or t.dtype != torch.int16 or e.dtype != torch.int8 or t.device != device \
            or e.device != device:
        raise ValueError(f"{what}: tiles are int16 mantissas and int8 exponents on {device}")
    if hd % TILE or tuple(e.shape) != (n, heads, hd // TILE):
        raise ValueError(f"{what}: mantissas {tuple(t.shape)} and exponents {tuple(e.shape)} do not match")
    (rs, hs, ds), (ers, ehs, eds) = t.stride(), e.stride()
    if (ds != 1 and hd > 1) or (eds != 1 and hd > TILE):
        raise ValueError(f"{what}: the values of a head must be contiguous")
    if (n > 1 and ers * TILE != rs) or (heads > 1 and ehs * TILE != hs):
        raise ValueError(f"{what}: the exponents' strides {(ers, ehs)} are not a sixteenth of the "
                         f"mantissas' {(rs, hs)}")
    # strides that are never used (one row, one head) need not be multiples of a tile
    return RowsC(t.data_ptr(), e.data_ptr(), TILES, heads, rs if n > 1 else heads * hd, hs if heads > 1 else hd)


def like(x, t, dtype):
    """Results of dtype for x, whose values are t (None: x's type; float32
    for tiles), that lie nowhere yet: the type, and the RowsC of contiguous
    ones without their address."""
    if dtype is None:
        dtype = t.dtype if t is x else torch.float32
    elif dtype not in TYPES:
        raise ValueError(f"results are float32, bfloat16 or float16, not {dtype}")
    _, heads, hd = t.shape
    return dtype, RowsC(None, None, TYPES[dtype], heads, heads * hd, hd)


def new(x, t, dtype):
    """A contiguous tensor of the shape of x's values t: of dtype, or x's
    (float32 for tiles) -> it and its RowsC."""
    dtype, r = like(x, t, dtype)
    y = torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)   # 0.6 us less than empty
    r.p = y.data_ptr()
    return y, r


def empty(n, heads, hd, dtype, device):
    """New rows of dtype (float32) -> the tensor and its RowsC."""
    dtype = torch.float32 if dtype is None else dtype
    if dtype not in TYPES:
        raise ValueError(f"results are float32, bfloat16 or float16, not {dtype}")
    y = torch.empty((n, heads, hd), dtype=dtype, device=device)
    return y, RowsC(y.data_ptr(), None, TYPES[dtype], heads, heads * hd, hd)


def ints(t, what: str, device, n):
    """A contiguous int32 vector of n on `device` -> its pointer."""
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous() or t.shape != (n,):
        raise ValueError(f"{what} must be a contiguous int32 tensor ({n},) on {device}")
    return t.data_ptr()


def gpu_of(t, what):
    """The device of a tensor that has to be on a GPU."""
    if not t.is_cuda:
        _need_gpu()
        raise ValueError(f"{what} is on {t.device}, not on a GPU")
    return t.device


MAX_INT = MAX_ROWS = 0x7fffffff   # the entry points count rows in int


def c_int(n, what: str, least=0, most=MAX_INT):
    """n as an int of the entry points: ctypes would take the lowest bits of
    a larger one."""
    n = int(n)
    if not least <= n <= most:
        raise ValueError(f"{what}={n}")
    return n


class Fixed:
    """An object whose C struct is made once: its tensors are written into,
    never replaced (an in-place form, x.lens += 1, assigns the tensor it has
    written into: no other object)."""

    def __setattr__(self, name, value):
        if name in self.__dict__ and name[0] != "_" and self.__dict__[name] is not value:
            raise AttributeError(f"{type(self).__name__}.{name} cannot be replaced: write into it, or make a new object")
        object.__setattr__(self, name, value)

    def __delattr__(self, name):
        if name[0] != "_":
            raise AttributeError(f"{type(self).__name__}.{name} cannot be taken away")
        object.__delattr__(self, name)


class Entry:
    """A stream-ordered entry point: called with the device its tensors are
    on, and its arguments without the stream.  The C entry points launch on
    the current device, so that is switched where it is another."""

    def __init__(self, name):
        self.name, self.f = name, None

    def __call__(self, device, *args):
        if self.f is None:
            self.f = getattr(lib(), self.name)
        index = device.index
        if _current_device() == index:
            rc = self.f(*args, _raw_stream(index))
        else:
            with torch.cuda.device(device):
                rc = self.f(*args, _raw_stream(index))
        if rc:
            check(self.name, rc)
