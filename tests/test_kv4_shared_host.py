"""What the attention over shared prefixes refuses, on the CPU: every call has
to stop at a check."""
import ctypes as C

import pytest

from test_kv4_host import BAD_BATCH, BAD_CACHE, BAD_ROWS, _batch, _cache, _lib, _refused, _rows

WORK, BIG = 1 << 22, 1 << 30


def _shared(L, **kw):
    d = dict(pages=4096, start=4096, len=4096, n_groups=2, width=3, max_rows=0, max_len=0)
    d.update(kw)
    return L.Kv4SharedC(**d)


def _call(L, cache=None, batch=None, shared=None, q=None, out=None, scale=1.0, window=0, work=WORK, size=BIG):
    good = (_cache(L), _batch(L), _shared(L), _rows(L), _rows(L))
    a = [C.byref(x or y) for x, y in zip((cache, batch, shared, q, out), good)]
    return "bfp_kv4_attn_shared_d", *a, scale, window, work, size, None


@pytest.mark.parametrize("bad", [dict(pages=None), dict(start=None), dict(len=None), dict(pages=4098), dict(start=4097), dict(len=4099),
                                 dict(n_groups=0), dict(n_groups=-1), dict(n_groups=65536), dict(width=0), dict(max_rows=-1), dict(max_len=-1),
                                 dict(width=1 << 28)], ids=str)
def test_refuses_bad_groups(bad):
    L = _lib()
    _refused(L, *_call(L, shared=_shared(L, **bad)))
    r = C.byref(_rows(L))
    assert L.lib().bfp_kv4_attn_shared_work(C.byref(_cache(L)), C.byref(_batch(L)), C.byref(_shared(L, **bad)), r, r, 0) == 0


def test_refuses_no_groups():
    L = _lib()
    r = C.byref(_rows(L))
    _refused(L, "bfp_kv4_attn_shared_d", C.byref(_cache(L)), C.byref(_batch(L)), None, r, r, 1.0, 0, WORK, BIG, None)


@pytest.mark.parametrize("cache,batch", [(c, {}) for c in BAD_CACHE] + [({}, b) for b in BAD_BATCH])
def test_refuses_bad_caches_and_batches(cache, batch):
    L = _lib()
    _refused(L, *_call(L, cache=_cache(L, **cache), batch=_batch(L, **batch)))


@pytest.mark.parametrize("bad", BAD_ROWS)
def test_refuses_bad_rows(bad):
    L = _lib()
    _refused(L, *_call(L, q=_rows(L, **bad)))


def test_refuses_bad_calls():
    L = _lib()
    for kw in (dict(scale=float("nan")), dict(window=-1), dict(q=_rows(L, heads=3)), dict(work=None), dict(work=WORK + 8), dict(size=64),
               dict(out=_rows(L, p=4096 + 64))):
        _refused(L, *_call(L, **kw))
    many = _batch(L, n_rows=2 ** 31 - 1)
    assert "too many" in _refused(L, *_call(L, cache=_cache(L, heads=1), batch=many, q=_rows(L, heads=8, rs=512), out=_rows(L, heads=8, rs=512)))
    many = _batch(L, n_rows=1 << 23, max_q=1 << 23)     # a thread for each lane of the join
    assert "too many" in _refused(L, *_call(L, cache=_cache(L, heads=1), batch=many, q=_rows(L, heads=8, rs=512), out=_rows(L, heads=8, rs=512)))


def test_nothing_to_do_is_no_error():
    L = _lib()
    for kw in (dict(n_seq=0), dict(max_q=0), dict(n_rows=0)):
        name, *args = _call(L, batch=_batch(L, **kw), work=None, size=0)
        assert getattr(L.lib(), name)(*args) == 0
