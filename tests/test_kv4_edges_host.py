"""The ends of what the rotary and 4-bit-cache entry points take, on the CPU:
what they refuse at their own checks, and what they do not."""
import ctypes as C

import numpy as np
import pytest

from test_kv4_host import _batch, _cache, _lib, _refused, _rows


def test_in_place_forms_put_back_the_same_object():
    """t.lens += 1 writes into the tensor and then assigns it: no other
    object, so nothing to refuse; another one is."""
    import torch
    from bfp._rows import Fixed

    class Thing(Fixed):
        def __init__(self, lens):
            self.lens = lens
    lens = torch.tensor([3, 4])
    t = Thing(lens)
    t.lens += 1
    t.lens *= 2
    assert t.lens is lens and lens.tolist() == [8, 10]
    with pytest.raises(AttributeError):
        t.lens = t.lens + 1
    assert t.lens is lens and lens.tolist() == [8, 10]


OVERLAP = [  # heads, hd, rows, row stride, head stride, whether two rows share a value
    (2, 64, 4, 128, 64, False), (2, 64, 4, 64, 64, True), (2, 64, 4, 127, 64, True), (2, 64, 4, 64, 256, False),   # heads before rows
    (2, 64, 4, 64, 255, True), (3, 64, 2, 320, 128, False), (3, 64, 2, 192, 128, False), (3, 64, 2, 128, 192, False),
    (3, 64, 3, 128, 192, False), (3, 64, 3, 127, 192, True), (2, 64, 1, 0, 64, False), (1, 64, 5, 64, 0, False), (1, 64, 5, 63, 0, True), (1, 64, 1, 0, 0, False),
    (9, 16, 1000, 144, 16, False), (9, 16, 1000, 143, 16, True), (9, 16, 1000, 16, 16000, False), (9, 16, 1000, 16, 15999, True)]


@pytest.mark.parametrize("case", OVERLAP, ids=str)
def test_results_that_lie_on_each_other(case):
    """Against a set of all values' places.  What passes this check is
    refused by a later one: nothing is launched."""
    heads, hd, n, rs, hs, shared = case
    seen = (np.arange(n)[:, None, None] * rs + np.arange(heads)[:, None] * hs + np.arange(hd)).reshape(-1)
    assert (len(np.unique(seen)) < len(seen)) == shared
    L = _lib()
    y = L.RowsC(1 << 30, None, 0, heads, rs, hs)
    x = L.RowsC(1 << 20, None, 0, heads, heads * hd, hd)
    msg = _refused(L, "bfp_rope_d", C.byref(x), n, hd, 4096, 4096, 16, hd + 2, 0, C.byref(y), None)
    assert ("overlap" in msg) == shared and ("rot" in msg) != shared, msg
    c, b = _cache(L, heads=heads, hd=hd), _batch(L, n_rows=n)
    msg = _refused(L, "bfp_kv4_attn_d", C.byref(c), C.byref(b), C.byref(x), C.byref(y), 1.0, -1, None, 0, None)
    assert ("overlap" in msg) == shared and ("window" in msg) != shared, msg


def test_strides_whose_product_leaves_64_bits():
    L = _lib()
    for rs, hs in ((1 << 62, 64), (64, 1 << 62), (1 << 60, 1 << 60)):
        x = L.RowsC(1 << 20, None, 0, 9, rs, hs)
        assert "too large" in _refused(L, "bfp_rope_d", C.byref(x), 4, 64, 4096, 4096, 16, 66, 0, C.byref(x), None)


def test_strides_that_nothing_uses():
    """One row, or one head: what its stride is does not matter.  The calls
    are refused for what follows."""
    L = _lib()
    c, b = C.byref(_cache(L, heads=1)), C.byref(_batch(L, n_rows=1))
    for kind, e in ((0, None), (1, None), (3, 4096)):
        r = L.RowsC(4096, e, kind, 1, 131, 3)
        free = L.RowsC(1 << 30, None, 1, 1, 131, 3)
        assert "window" in _refused(L, "bfp_kv4_attn_d", c, b, C.byref(r), C.byref(free), 1.0, -1, None, 0, None)
        assert "rot" in _refused(L, "bfp_kv4_append_d", c, b, C.byref(r), C.byref(r), None, None, None, 4096, 16, 66, 0, None)
        assert "rot" in _refused(L, "bfp_rope_d", C.byref(r), 1, 64, 4096, 4096, 16, 66, 0, C.byref(free), None)
    two = C.byref(_batch(L, n_rows=2))
    r = L.RowsC(4096, None, 1, 1, 131, 3)
    assert "strides" in _refused(L, "bfp_kv4_attn_d", c, two, C.byref(r), C.byref(L.RowsC(1 << 30, None, 1, 1, 64, 64)), 1.0, 0, None, 0, None)
