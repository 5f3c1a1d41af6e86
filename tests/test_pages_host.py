"""What the page pool's entry points refuse, on the CPU: nothing may be
launched here, so every call has to stop at a check."""
import ctypes as C

import pytest


def _lib():
    from bfp import _lib
    return _lib


def _pool(L, pages=((1 << 20, 1536),), **kw):
    a = (L.PageArrayC * max(len(pages), 1))(*(L.PageArrayC(*x) for x in pages))
    d = dict(refs=4096, n_short=8192, arrays=a, n_pages=8, page=16, n_arrays=len(pages))
    d.update(kw)
    p = L.PagesC(**d)
    p._keep = a
    return p


def _batch(L, **kw):
    d = dict(pages=16384, start=20480, len=24576, n_seq=2, n_rows=4, width=3, max_q=1, max_len=0)
    d.update(kw)
    return L.Kv4BatchC(**d)


def _refused(L, name, *args):
    rc = getattr(L.lib(), name)(*args)
    assert rc == -22, (name, rc)
    return L.lib().bfp_last_error().decode()


WORK, BIG = 1 << 22, 1 << 20


def _calls(L, p):
    b = C.byref(_batch(L))
    P = C.byref(p)
    t = (L.PageTableC * 1)(L.PageTableC(16384, 6))
    return [("bfp_pages_copy_d", P, 32768, 40960, 2, None),
            ("bfp_pages_reserve_d", P, b, WORK, BIG, None),
            ("bfp_pages_fork_d", P, 16384, 20480, 2, 3, 24576, 2, 28672, 32768, 3, WORK, BIG, None),
            ("bfp_pages_free_d", P, 16384, 6, None),
            ("bfp_pages_compact_d", P, t, 1, 28672, WORK, BIG, None)]


@pytest.mark.parametrize("bad", [dict(refs=None), dict(refs=4100), dict(n_short=8193), dict(n_pages=0), dict(n_pages=-1),
                                 dict(n_pages=(1 << 28) + 1), dict(page=8), dict(page=48), dict(page=512), dict(n_arrays=-1),
                                 dict(arrays=None, n_arrays=1), dict(a=((None, 16),)), dict(a=((1 << 20, 24),)), dict(a=((1 << 20, 0),)),
                                 dict(a=(((1 << 20) + 8, 16),)), dict(a=((1 << 20, 16), (1 << 20, 1 << 33)))], ids=str)
def test_refuses_bad_pools(bad):
    L = _lib()
    bad = dict(bad)
    p = _pool(L, bad.pop("a")) if "a" in bad else _pool(L, **bad)
    for name, *args in _calls(L, p):
        _refused(L, name, *args)
    assert L.lib().bfp_pages_work(C.byref(p), 4) == 0


def test_refuses_bad_calls():
    L = _lib()
    p = C.byref(_pool(L))
    t = (L.PageTableC * 17)(*(L.PageTableC((1 << 24) + 4096 * i, 6) for i in range(17)))
    copy = lambda *a: _refused(L, "bfp_pages_copy_d", p, *a, None)  # noqa: E731
    copy(None, 40960, 2), copy(32768, None, 2), copy(32770, 40960, 2), copy(32768, 40960, -1)
    reserve = lambda work=WORK, size=BIG, **kw: _refused(L, "bfp_pages_reserve_d", p, C.byref(_batch(L, **kw)), work, size, None)  # noqa: E731
    for kw in (dict(pages=None), dict(start=None), dict(len=None), dict(n_seq=-1), dict(n_seq=65536), dict(width=0),
               dict(max_q=-1), dict(width=1 << 28), dict(pages=4100), dict(start=16388), dict(len=16384)):
        reserve(**kw)
    reserve(work=None), reserve(work=WORK + 8), reserve(size=16)
    good = dict(pages=16384, len=20480, n_seq=2, width=3, parents=24576, n=2, out=28672, out_len=32768, out_width=3, work=WORK, size=BIG)
    fork = lambda **kw: _refused(L, "bfp_pages_fork_d", p, *{**good, **kw}.values(), None)  # noqa: E731
    for kw in (dict(pages=None), dict(len=None), dict(parents=None), dict(out=None), dict(out_len=None), dict(n_seq=-1), dict(n=-1),
               dict(width=0), dict(out_width=0), dict(width=1 << 28), dict(out=16384), dict(out=16404), dict(out_len=28676), dict(out=24572),
               dict(out=4096), dict(work=None), dict(work=WORK + 4), dict(size=16), dict(pages=16386)):
        fork(**kw)
    assert "lies on" in fork(out=16388)
    free = lambda *a: _refused(L, "bfp_pages_free_d", p, *a, None)  # noqa: E731
    free(None, 6), free(16385, 6), free(16384, -1), free(4100, 6)
    compact = lambda tables, n, live=28672, work=WORK, size=BIG: _refused(  # noqa: E731
        L, "bfp_pages_compact_d", p, tables, n, live, work, size, None)
    compact(t, 17), compact(t, -1), compact(None, 1), compact(t, 1, live=None), compact(t, 1, work=None), compact(t, 1, size=16)
    compact(t, 1, live=(1 << 24) + 8)
    assert "lies on" in compact((L.PageTableC * 2)(L.PageTableC(16384, 6), L.PageTableC(16400, 6)), 2)


def test_nothing_to_do_is_no_error():
    L = _lib()
    p = C.byref(_pool(L))
    lib = L.lib()
    assert lib.bfp_pages_copy_d(p, None, None, 0, None) == 0
    for kw in (dict(n_seq=0), dict(max_q=0), dict(n_rows=0)):
        assert lib.bfp_pages_reserve_d(p, C.byref(_batch(L, **kw)), None, 0, None) == 0
    assert lib.bfp_pages_fork_d(p, 16384, 20480, 2, 3, None, 0, None, None, 3, None, 0, None) == 0
    assert lib.bfp_pages_free_d(p, None, 0, None) == 0


def test_work_grows_with_pages_and_children():
    L = _lib()
    size = lambda n_pages, n: L.lib().bfp_pages_work(C.byref(_pool(L, n_pages=n_pages)), n)  # noqa: E731
    assert size(8, 10) == size(8, 0) + 80 and size(100000, 0) > size(8, 0) > 0
    assert L.lib().bfp_pages_work(C.byref(_pool(L)), -1) == 0
