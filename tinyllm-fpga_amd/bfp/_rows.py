"""Rows of heads on the device: torch tensors (rows, heads, hd), or pairs
(m, e) of 16-bit tiles, as the C entry points take them (struct bfp_rows)."""
from __future__ import annotations

from contextlib import nullcontext

from ._dev import _torch
from ._lib import RowsC

TILE = 16
F32, BF16, F16, TILES = range(4)
_TYPES = {}


def types():
    """{torch dtype: enum bfp_type}."""
    if not _TYPES:
        torch = _torch()
        _TYPES.update({torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16})
    return _TYPES


def device_of(x):
    return (x[0] if isinstance(x, tuple) else x).device


def shape_of(x):
    return tuple((x[0] if isinstance(x, tuple) else x).shape)


def rows(x, what: str, device=None) -> RowsC:
    """The RowsC of x; ValueError where x is not rows of heads.  The struct
    holds no reference: x has to live until the call is made."""
    pair = isinstance(x, tuple)
    if pair and len(x) != 2:
        raise ValueError(f"{what}: tiles are a pair (m, e)")
    t = x[0] if pair else x
    if not hasattr(t, "data_ptr") or t.dim() != 3:
        raise ValueError(f"{what} must be a tensor (rows, heads, hd) or a pair (m, e) of them")
    if t.device.type != "cuda" or (device is not None and t.device != device):
        raise ValueError(f"{what} is on {t.device}, not on {device if device is not None else 'a GPU'}")
    n, heads, hd = t.shape
    if hd > 1 and t.stride(2) != 1:
        raise ValueError(f"{what}: the values of a head must be contiguous")
    if not pair:
        kind = types().get(t.dtype)
        if kind is None:
            raise ValueError(f"{what} has type {t.dtype}: float32, bfloat16, float16, or a pair (m, e) of "
                             "int16 mantissas and int8 exponents")
        return RowsC(t.data_ptr(), None, kind, heads, t.stride(0), t.stride(1))
    torch, e = _torch(), x[1]
    if t.dtype != torch.int16 or e.dtype != torch.int8 or e.device != t.device:
        raise ValueError(f"{what}: tiles are int16 mantissas and int8 exponents on one device")
    if hd % TILE or tuple(e.shape) != (n, heads, hd // TILE):
        raise ValueError(f"{what}: mantissas {tuple(t.shape)} and exponents {tuple(e.shape)} do not match")
    if hd > TILE and e.stride(2) != 1:
        raise ValueError(f"{what}: the exponents of a head must be contiguous")
    rs, hs = t.stride(0), t.stride(1)
    if (n > 1 and e.stride(0) * TILE != rs) or (heads > 1 and e.stride(1) * TILE != hs):
        raise ValueError(f"{what}: the exponents' strides {e.stride()[:2]} are not a sixteenth of the "
                         f"mantissas' {(rs, hs)}")
    # strides that are never used (one row, one head) need not be multiples of a tile
    return RowsC(t.data_ptr(), e.data_ptr(), TILES, heads, rs if n > 1 else heads * hd, hs if heads > 1 else hd)


def ints(t, what: str, device, n=None):
    """A contiguous int32 vector on `device` -> its pointer."""
    if t.device != device or t.dtype != _torch().int32 or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor on {device}")
    if n is not None and tuple(t.shape) != (n,):
        raise ValueError(f"{what} has shape {tuple(t.shape)}, not ({n},)")
    return t.data_ptr()


def on(device):
    """The context in which calls for tensors on `device` are made: the C
    entry points launch on the current device."""
    torch = _torch()
    return nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def stream_of(device) -> int:
    return _torch().cuda.current_stream(device).cuda_stream
