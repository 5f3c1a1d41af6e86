"""The scratch of the attention over shared prefixes, on the CPU: about what its
rows' unfinished sums take, however many splits fewer rows would have."""
import ctypes as C

import pytest

from test_kv4_host import _batch, _cache, _lib, _rows
from test_kv4_shared_host import _shared

PIECES = 65536      # rows of all workgroups that share a prefix: 512 of 128, 256 of 256


def _work(L, seqs, new, groups, prefix, heads, hq, hd, page=64, rows=None, hints=True, own=512, kind=0):
    rows = seqs * new if rows is None else rows
    cache = _cache(L, n_pages=4096, page=page, heads=heads, hd=hd)
    batch = _batch(L, n_seq=seqs, n_rows=rows, width=(prefix + new + own) // page + 1, max_q=new, max_len=prefix + new + own if hints else 0)
    shared = _shared(L, n_groups=groups, width=prefix // page + 1, max_rows=-(-seqs // groups) * new if hints else 0, max_len=prefix if hints else 0)
    q = _rows(L, type=kind, heads=hq, rs=hq * hd, hs=hd)
    n = L.lib().bfp_kv4_attn_shared_work(C.byref(cache), C.byref(batch), C.byref(shared), C.byref(q), C.byref(q), 0)
    assert n > 0, L.lib().bfp_last_error()
    return n


@pytest.mark.parametrize("hints", [True, False])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("seqs,new,groups,prefix", [(16, 512, 1, 8192), (64, 512, 1, 16384), (8, 1024, 1, 16384), (64, 1, 1, 16384), (21, 17, 3, 65536),
                                                    (1, 16000, 1, 16384), (66, 20, 66, 500), (130, 40, 130, 3000), (5, 1, 1, 304), (256, 64, 8, 2048)])
@pytest.mark.parametrize("heads,hq,hd", [(8, 32, 128), (3, 9, 64), (1, 8, 256)])
def test_scratch_of_many_rows(seqs, new, groups, prefix, heads, hq, hd, kind, hints):
    L = _lib()
    rows = seqs * new * hq
    # a place for each row of a whole prefix (and a workgroup's padding a group and head), or of all pieces; the
    # rest's rows, or their splits; what few rows' workgroups keep for themselves (768 of them, 2 x 16 rows)
    most = max(rows + groups * heads * 256, PIECES) + max(rows, PIECES) + 768 * 32
    if groups > 64:      # splits of one length: 256 workgroups over more than 64 row tiles
        most += 2 * rows
    got = _work(L, seqs, new, groups, prefix, heads, hq, hd, hints=hints, kind=kind)
    assert got <= most * (4 * hd + 8) + (1 << 16), (got, most * (4 * hd + 8))


def test_scratch_does_not_grow_with_padding():
    """Rows behind the last sequence take no splits' room."""
    L = _lib()
    one, padded = (_work(L, 2, 600, 1, 500, 1, 2, 64, rows=n, own=6600) for n in (1200, 12000))
    assert padded - one <= 2 * (12000 - 1200) * 2 * (4 * 64 + 8) + (256 * 256) * (4 * 64 + 8)
