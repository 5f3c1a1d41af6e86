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


def test_what_a_struct_points_to_cannot_be_taken_away():
    """Else another object could take its name, while the struct points to
    the first one's memory."""
    from bfp._rows import Fixed

    class Thing(Fixed):
        def __init__(self):
            self.lens, self._n = [1], 2
    t = Thing()
    with pytest.raises(AttributeError):
        del t.lens
    del t._n
    assert t.lens == [1]


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


def _places(p, size, n, heads, hd, rs, hs):
    at = p + size * (np.arange(n)[:, None, None] * rs + np.arange(heads)[:, None] * hs + np.arange(hd))
    return set((at.reshape(-1, 1) + np.arange(size)).reshape(-1).tolist())


#  q_out's and k's first byte past 2^20, type (0: 4 bytes, 1: 2), heads, row stride, head stride; rows
BETWEEN = [
    ((0, 1, 4, 384, 64), (512, 1, 1, 384, 64), 5),              # joined rows q | k
    ((512, 1, 4, 384, 64), (0, 1, 4, 384, 64), 5),              # q runs into the next row's k
    ((0, 1, 4, 384, 64), (384, 1, 1, 384, 64), 5),              # k is one of q's heads
    ((0, 1, 4, 384, 64), (384, 1, 1, 320, 64), 5),              # other rows
    ((0, 1, 2, 768, 384), (128, 1, 2, 768, 384), 5),            # q, k and v side by side within a group
    ((0, 1, 2, 768, 384), (64, 1, 2, 768, 384), 5),
    ((0, 1, 2, 768, 384), (896, 1, 1, 768, 64), 5),             # between two groups' q
    ((0, 1, 2, 768, 384), (704, 1, 1, 768, 64), 5),
    ((0, 1, 4, 384, 64), (5 * 768, 1, 1, 384, 64), 5),          # behind the last row
    ((0, 1, 4, 384, 64), (4 * 768 + 256, 1, 1, 384, 64), 5),
    ((0, 0, 4, 384, 64), (1024, 0, 1, 384, 64), 5),
    ((0, 0, 4, 384, 64), (0, 1, 1, 384, 64), 5),                # another type's rows in the same place
    ((0, 1, 4, 384, 64), (512, 1, 1, 9999, 7), 1),              # one row, one head: strides that nothing uses
    ((0, 1, 4, 384, 64), (496, 1, 1, 9999, 7), 1),
    ((0, 1, 4, 64, 320), (4 * 640, 1, 1, 64, 64), 5),           # heads before rows
    ((0, 1, 4, 64, 320), (2 * 640, 1, 1, 64, 64), 5)]


@pytest.mark.parametrize("a,b,n", BETWEEN)
def test_results_that_lie_on_operands(a, b, n):
    """Against sets of bytes; the calls stop there or at a later check."""
    shared = bool(_places(a[0], 2 if a[1] else 4, n, a[2], 64, *a[3:]) & _places(b[0], 2 if b[1] else 4, n, b[2], 64, *b[3:]))
    L = _lib()
    make = lambda x: L.RowsC((1 << 20) + x[0], None, x[1], x[2], x[3], x[4])  # noqa: E731
    free = L.RowsC(1 << 30, None, 1, b[2], 1 << 12, 64)
    cache = C.byref(_cache(L, heads=b[2]))
    batch = C.byref(_batch(L, n_rows=n))
    for k, v in ((make(b), free), (free, make(b))):
        q = make(a)
        msg = _refused(L, "bfp_kv4_append_d", cache, batch, C.byref(k), C.byref(v), C.byref(q), C.byref(q), None, 4096, 16, 66, 0, None)
        assert ("q_out" in msg) == shared and ("rot" in msg) != shared, msg


def test_results_over_their_own_rows():
    """In place means the same place: not shifted, not in another stride or
    size of value."""
    L = _lib()
    x = L.RowsC(1 << 20, None, 1, 3, 192, 64)
    other = [L.RowsC((1 << 20) + 16, None, 1, 3, 192, 64), L.RowsC(1 << 20, None, 1, 3, 256, 64), L.RowsC(1 << 20, None, 0, 3, 192, 64),
             L.RowsC((1 << 20) + 384, None, 1, 3, 192, 64)]
    apart = [x, L.RowsC(1 << 20, None, 2, 3, 192, 64), L.RowsC((1 << 20) + 4 * 384, None, 1, 3, 192, 64), L.RowsC(1 << 24, None, 0, 3, 192, 64)]
    c, b = C.byref(_cache(L, heads=1)), C.byref(_batch(L, n_rows=4))
    kv = C.byref(L.RowsC(1 << 30, None, 1, 1, 64, 64))
    for y in other + apart:
        shared = any(y is o for o in other)
        msg = _refused(L, "bfp_rope_d", C.byref(x), 4, 64, 4096, 4096, 16, 66, 0, C.byref(y), None)
        assert ("y lies" in msg) == shared and ("rot" in msg) != shared, msg
        msg = _refused(L, "bfp_kv4_attn_d", c, b, C.byref(x), C.byref(y), 1.0, -1, None, 0, None)
        assert ("out lies" in msg) == shared and ("window" in msg) != shared, msg
        msg = _refused(L, "bfp_kv4_append_d", c, b, kv, kv, C.byref(x), C.byref(y), None, 4096, 16, 66, 0, None)
        assert ("q_out lies" in msg) == shared and ("rot" in msg) != shared, msg


def test_tiles_over_their_own_rows():
    L = _lib()
    q = L.RowsC(1 << 20, 1 << 21, 3, 3, 192, 64)
    c, b = C.byref(_cache(L, heads=1)), C.byref(_batch(L, n_rows=4))
    for out, shared in ((q, False), (L.RowsC(1 << 22, 1 << 23, 3, 3, 192, 64), False), (L.RowsC(1 << 20, 1 << 23, 3, 3, 192, 64), False),
                        (L.RowsC(1 << 22, 1 << 21, 3, 3, 192, 64), False), (L.RowsC(1 << 22, (1 << 21) + 4, 3, 3, 192, 64), True),
                        (L.RowsC(1 << 22, 1 << 20, 3, 3, 192, 64), True), (L.RowsC(1 << 22, (1 << 21) + 48, 3, 3, 192, 64), False)):
        msg = _refused(L, "bfp_kv4_attn_d", c, b, C.byref(q), C.byref(out), 1.0, -1, None, 0, None)
        assert ("out lies" in msg) == shared and ("window" in msg) != shared, msg


def test_keys_and_values_read_into_the_same_place():
    L = _lib()
    c, b = C.byref(_cache(L)), C.byref(_batch(L))
    k = L.RowsC(1 << 20, None, 1, 2, 128, 64)
    for v in (k, L.RowsC((1 << 20) + 128, None, 1, 2, 128, 64)):
        assert "v lies" in _refused(L, "bfp_kv4_read_d", c, b, C.byref(k), C.byref(v), None)


def test_numbers_that_an_int_does_not_hold():
    """They do not come back from the other end."""
    import torch
    from bfp import rotary
    inv, _ = rotary.rope_freqs(4)
    for bad in (2 ** 31, 2 ** 32 + 4, 2 ** 64 + 4, -2 ** 32 + 4):
        for call in (lambda: rotary.rope_freqs(bad), lambda: rotary.rope_freqs(64, 1e4, "parts", 4.0, bad),
                     lambda: rotary.rope_table(inv, bad, out=torch.zeros(4, 2, 2))):
            with pytest.raises(ValueError):
                call()
    for first in (2 ** 64, -2 ** 64 + 1, 2 ** 63):
        with pytest.raises(ValueError):
            rotary.rope_table(inv, 4, first=first, out=torch.zeros(4, 2, 2))


def test_positions_past_64_bits():
    L = _lib()
    inv = np.zeros(4)
    for first, n in ((2 ** 63 - 1, 1), (2 ** 63 - 5, 100), (2 ** 31, 1), (2 ** 31 - 1, 2)):
        assert "first" in _refused(L, "bfp_rope_table_d", inv.ctypes.data, 4, 1.0, first, n, 4096, None)


def test_positions_that_are_not_aligned():
    L = _lib()
    x = L.RowsC(1 << 20, None, 0, 1, 64, 64)
    assert "pos" in _refused(L, "bfp_rope_d", C.byref(x), 4, 64, 4098, 4096, 16, 64, 0, C.byref(x), None)


def test_scales_past_float32():
    L = _lib()
    c, b = C.byref(_cache(L)), C.byref(_batch(L))
    r = C.byref(_rows(L))
    for scale in (1e300, -1e300, 3e38, float("inf"), float("nan")):
        assert "scale" in _refused(L, "bfp_kv4_attn_d", c, b, r, r, scale, 0, None, 0, None)


def test_scratch_does_not_grow_with_rows_that_no_sequence_has():
    """Row arrays that hold room for more: the scratch is the sequences'."""
    L = _lib()
    for news, heads, width in ((64, 4, 4000), (1, 3, 4000), (300, 4, 1000), (500, 1, 4000)):
        c, r = C.byref(_cache(L, heads=1)), _rows(L, heads=heads)
        sizes = [L.lib().bfp_kv4_attn_work(c, C.byref(_batch(L, n_seq=1, n_rows=n, width=width, max_q=news)), C.byref(r), C.byref(r), 0)
                 for n in (news, 4 * news, 1 << 20)]
        assert sizes[0] > 0 and len(set(sizes)) == 1, sizes


def test_positions_past_31_bits():
    """A table of pages for more positions than an int counts."""
    L = _lib()
    r = _rows(L)
    for width, page in ((1 << 23, 256), ((1 << 27) - 1, 16), ((1 << 31) - 1, 16)):
        c, b = C.byref(_cache(L, page=page)), C.byref(_batch(L, width=width))
        k = C.byref(r)
        assert "positions" in _refused(L, "bfp_kv4_append_d", c, b, k, k, None, None, None, None, 0, 0, 0, None)
        assert "positions" in _refused(L, "bfp_kv4_read_d", c, b, k, None, None)
        assert "positions" in _refused(L, "bfp_kv4_attn_d", c, b, k, k, 1.0, 0, None, 0, None)
    c, b = C.byref(_cache(L, page=256)), C.byref(_batch(L, width=(1 << 23) - 256, max_q=0))
    assert L.lib().bfp_kv4_attn_d(c, b, C.byref(r), C.byref(r), 1.0, 0, None, 0, None) == 0
