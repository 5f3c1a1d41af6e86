"""What the bounds', the choice's and the listed pages' entry points refuse, on
the CPU: every call has to stop at a check."""
import ctypes as C

import pytest

from test_kv4_host import BAD_BATCH, BAD_CACHE, BAD_ROWS, _batch, _cache, _lib, _refused, _rows

WORK, BIG = 1 << 22, 1 << 30


def _calls(L, c, b, q, o):
    c, b, q, o = (C.byref(x) for x in (c, b, q, o))
    return [("bfp_kv4_bounds_d", c, b, 8192, None),
            ("bfp_kv4_select_d", c, b, 8192, q, 2, 1, 1, 4096, WORK, BIG, None),
            ("bfp_kv4_attn_picks_d", c, b, 4096, 2, q, o, 1.0, WORK, BIG, None)]


@pytest.mark.parametrize("cache,batch", [(c, {}) for c in BAD_CACHE] + [({}, b) for b in BAD_BATCH])
def test_refuses_bad_caches_and_batches(cache, batch):
    L = _lib()
    c, b, r = _cache(L, **cache), _batch(L, **batch), _rows(L)
    for name, *args in _calls(L, c, b, r, r):
        _refused(L, name, *args)
    R = C.byref(r)
    assert L.lib().bfp_kv4_select_work(C.byref(c), C.byref(b), R) == 0
    assert L.lib().bfp_kv4_attn_picks_work(C.byref(c), C.byref(b), 2, R, R) == 0


@pytest.mark.parametrize("bad", BAD_ROWS)
def test_refuses_bad_rows(bad):
    L = _lib()
    c, b, good, r = _cache(L), _batch(L), _rows(L), _rows(L, **bad)
    for name, *args in _calls(L, c, b, r, good)[1:]:
        _refused(L, name, *args)


def test_refuses_bad_calls():
    L = _lib()
    c, b, r = C.byref(_cache(L)), C.byref(_batch(L)), C.byref(_rows(L))
    wide = C.byref(_batch(L, width=16385))
    sel = lambda n=2, first=1, last=1, bounds=8192, picks=4096, work=WORK, size=BIG, batch=b: _refused(  # noqa: E731
        L, "bfp_kv4_select_d", c, batch, bounds, r, n, first, last, picks, work, size, None)
    for kw in (dict(n=0), dict(n=-1), dict(n=1 << 28), dict(first=-1), dict(last=0), dict(last=-1), dict(first=2), dict(last=2),
               dict(first=2 ** 31 - 1), dict(last=2 ** 31 - 1), dict(bounds=None), dict(bounds=8200), dict(picks=None), dict(picks=4098),
               dict(work=None), dict(work=WORK + 8), dict(size=8), dict(batch=wide)):
        sel(**kw)
    _refused(L, "bfp_kv4_bounds_d", c, b, None, None)
    _refused(L, "bfp_kv4_bounds_d", c, b, 8194, None)
    att = lambda n=2, picks=8192, scale=1.0: _refused(L, "bfp_kv4_attn_picks_d", c, b, picks, n, r, r, scale, WORK, BIG, None)  # noqa: E731
    for kw in (dict(n=0), dict(n=-3), dict(n=1 << 28), dict(picks=None), dict(picks=8193), dict(scale=float("inf")), dict(scale=float("nan"))):
        att(**kw)
    long_list = C.byref(_cache(L, n_pages=4096))
    one = C.byref(_batch(L, n_seq=1, n_rows=1, width=2000))
    n = L.lib().bfp_kv4_attn_picks_work(long_list, one, 2000, r, r)
    assert n > 0
    for work, size in ((None, n), (WORK, n - 1), (WORK + 4, n)):
        assert str(n) in _refused(L, "bfp_kv4_attn_picks_d", long_list, one, 4096, 2000, r, r, 1.0, work, size, None)


def test_nothing_to_do_is_no_error():
    L = _lib()
    c, r = C.byref(_cache(L)), C.byref(_rows(L))
    for kw in (dict(n_seq=0), dict(max_q=0), dict(n_rows=0)):
        b = C.byref(_batch(L, **kw))
        assert L.lib().bfp_kv4_bounds_d(c, b, 8192, None) == 0
        assert L.lib().bfp_kv4_select_d(c, b, 8192, r, 2, 1, 1, None, None, 0, None) == 0
        assert L.lib().bfp_kv4_attn_picks_d(c, b, None, 2, r, r, 1.0, None, 0, None) == 0


def test_scratch_is_bounded():
    """Scores of many rows go in pieces."""
    L = _lib()
    c = C.byref(_cache(L, heads=8))
    r = C.byref(_rows(L, heads=8, rs=512))
    for rows, width in ((1 << 20, 16000), (100, 10), (5, 16384)):
        n = L.lib().bfp_kv4_select_work(c, C.byref(_batch(L, n_seq=1, n_rows=rows, max_q=rows, width=width)), r)
        assert 0 < n <= 1 << 28
