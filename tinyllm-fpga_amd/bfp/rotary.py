"""Rotary positions on device tensors, beside ``api.rope_fp`` (one 64-wide
head, one position, float64): the angles of scaled contexts, and the
rotation of rows of heads in either pairing.

Tensors in and out stay on the device; every call is queued on the current
stream of their device and can be captured into a graph.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _rows
from ._lib import call

_table, _rope = _rows.Entry("bfp_rope_table_d"), _rows.Entry("bfp_rope_d")
SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "parts": 3, "bands": 4}


def rope_freqs(rot, base=10000.0, scaling="none", factor=1.0, orig_ctx=0):
    """The rot/2 angles per position (float64, host) and the factor on cos
    and sin.  scaling: how a context `factor` times as long as the trained
    `orig_ctx` gets its angles --
      "none"    base^(-2j/rot)
      "linear"  divided by factor
      "ntk"     base * factor^(rot/(rot-2))
      "parts"   pairs that turn more than 32 times over orig_ctx stay, those
                below one turn are divided, linear in the pair's index
                between; cos and sin grow by 0.1 ln(factor) + 1
      "bands"   above 4 turns stay, below 1 divided, linear in the turns"""
    if scaling not in SCALINGS:
        raise ValueError(f"scaling {scaling!r}: one of {', '.join(SCALINGS)}")
    rot, orig_ctx = (_rows.c_int(x, what, -1 - _rows.MAX_INT) for x, what in ((rot, "rot"), (orig_ctx, "orig_ctx")))
    inv, mscale = (C.c_double * max(rot // 2, 1))(), C.c_double()
    call("bfp_rope_freqs", rot, float(base), SCALINGS[scaling], float(factor), orig_ctx, inv, C.byref(mscale))
    return np.frombuffer(inv, np.float64), mscale.value


def _address(a):
    try:   # a third of the time a.ctypes.data takes
        return C.addressof(C.c_char.from_buffer(a))
    except (TypeError, ValueError, BufferError):   # not writable, or empty
        return a.ctypes.data


def rope_table(inv_freq, n_pos, mscale=1.0, first=0, out=None):
    """(cos, sin) of positions first .. first + n_pos - 1: float32 (n_pos,
    len(inv_freq), 2) on the current device (out: such a tensor to fill)."""
    inv = inv_freq
    if type(inv) is not np.ndarray or inv.dtype != np.float64 or inv.ndim != 1 or not inv.flags.c_contiguous:
        inv = np.ascontiguousarray(np.asarray(inv_freq, np.float64).reshape(-1))
    shape = (_rows.c_int(n_pos, "n_pos"), inv.size, 2)
    first = _rows.c_int(first, "first", -1 << 63, (1 << 63) - 1)
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device="cuda")
    elif tuple(out.shape) != shape or out.dtype != torch.float32 or not out.is_contiguous() or not out.is_cuda:
        raise ValueError(f"out must be a contiguous float32 tensor {shape} on a GPU")
    if shape[0]:
        _table(out.device, _address(inv), inv.size, float(mscale), first, shape[0], out.data_ptr())
    return out


def check_table(table, device):
    """n_pos and rot of a rope_table."""
    shape = table.shape
    if len(shape) != 3 or shape[2] != 2 or table.dtype != torch.float32 or not table.is_contiguous() \
            or table.device != device:
        raise ValueError(f"the table must be rope_table's: contiguous float32 (positions, pairs, 2) on {device}")
    return shape[0], 2 * shape[1]


def rope(x, pos, table, interleaved=False, out=None, dtype=None):
    """Rotate the first 2 * table.shape[1] values of every head of x (rows,
    heads, hd) -- or of 16-bit tiles (m, e) -- by table[pos[row]], and copy
    the rest.  Pairs are values (j, j + rot/2), as rope_fp has them, or with
    interleaved (2j, 2j + 1).  A row whose position is not in the table gets
    NaN there.  Returns `out` (may be x), or a new tensor of `dtype` (x's;
    float32 for tiles)."""
    t = _rows.values_of(x, "x")
    device = _rows.gpu_of(t, "x")
    xr = _rows.rows(x, "x", device)
    n, _, hd = t.shape
    if out is None:
        out, yr = _rows.new(x, t, dtype)
    elif type(out) is tuple or out.shape != t.shape or (dtype is not None and out.dtype != dtype):
        raise ValueError(f"out must be a tensor {tuple(t.shape)}" + (f" of {dtype}" if dtype else ""))
    else:
        yr = _rows.rows(out, "out", device)
    if n > _rows.MAX_ROWS:
        raise ValueError(f"{n} rows")
    n_pos, rot = check_table(table, device)
    p = _rows.ints(pos, "pos", device, n)
    if n:
        _rope(device, C.byref(xr), n, hd, p, table.data_ptr(), n_pos, rot, 1 if interleaved else 0, C.byref(yr))
    return out
