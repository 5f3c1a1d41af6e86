"""The 4-bit cache and the rotary operators on the CPU: the arithmetic that
finds rows, pages and tiles (compiled for the host), what the entry points
refuse, the scaled frequencies, and the format's own properties."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

import kv4_ref as ref

ROOT = Path(__file__).resolve().parent.parent


def run_host(tmp_path, body):
    src = tmp_path / "t.cpp"
    src.write_text('#include <cstdio>\n#include <cstdlib>\n#include "bfp_rows.h"\n#include "bfp_kv4.h"\n'
                   "using namespace bfp;\nint main() {\n" + body + "\n}\n")
    exe = tmp_path / "t"
    subprocess.run(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only", "-O1", "-std=c++17",
                    f"-I{ROOT / 'include'}", f"-I{ROOT / 'tinyllm-fpga_amd' / 'csrc'}", str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout


def test_division_by_multiplication(tmp_path):
    out = run_host(tmp_path, """
  unsigned ds[] = {1, 2, 3, 4, 5, 6, 7, 9, 15, 16, 17, 63, 64, 65, 127, 1000, 4095, 4096, 4097, 65535, 65537,
                   1000003, 0x3fffffff, 0x40000000, 0x40000001, 0x7fffffff};
  long bad = 0, n = 0;
  for (unsigned d : ds) {
    FastDiv f(d);
    unsigned long long s = 88172645463325252ull + d;
    for (int i = 0; i < 20000; ++i) {
      s ^= s << 13; s ^= s >> 7; s ^= s << 17;
      unsigned v = (unsigned)(s >> 33);
      if (i < 64) v = (unsigned)i;
      else if (i < 128) v = 0x7fffffffu - (i - 64);
      else if (i % 2) v = v / d * d - (i % 4 == 1 ? 1 : 0);   // multiples and what lies before them
      v &= 0x7fffffffu;
      unsigned r, q = f.div(v, r);
      bad += q != v / d || r != v % d;
      ++n;
    }
  }
  printf("%ld %ld", bad, n);""")
    assert out.split()[0] == "0" and int(out.split()[1]) == 26 * 20000


def test_rows_and_pages_stay_inside(tmp_path):
    """Whatever the batch's arrays hold: rows within the row arrays, pages
    within the table and the cache."""
    out = run_host(tmp_path, """
  int vals[] = {-2147483647 - 1, -2147483647, -7, -1, 0, 1, 2, 3, 9, 10, 11, 100, 2147483646, 2147483647};
  long bad = 0;
  for (int a : vals) for (int b : vals) for (int len : vals) for (int mq : {0, 1, 3, 2147483647}) for (int nr : {0, 1, 10}) {
    Kv4Span s = kv4_span(a, b, len, nr, mq);
    if (s.n < 0 || s.row0 < 0 || s.row0 + (long)s.n > nr || s.n > mq) ++bad;
    // positions: at + i for i < n never leaves int
    long p = (long)s.at + s.n;
    if (p > 2147483647L || (long)s.at < -2147483648L) ++bad;
  }
  int table[4] = {3, -1, 7, 2147483647};
  for (int p : vals) {
    int id = kv4_page(table, 3, 5, p);
    int want = p == 0 ? 3 : -1;
    if (id != want) ++bad;
  }
  // the last tile of a cache of 2^31 - 1 pages: 64 bits
  long long t = kv4_tile(2147483646LL, 4096, 4095, 16, 15, 256, 255);
  if (t != 2147483647LL * 4096 * 16 * 256 - 1) ++bad;
  printf("%ld", bad);""")
    assert out == "0"


def test_page_zero_of_an_ordinary_span(tmp_path):
    out = run_host(tmp_path, """
  Kv4Span s = kv4_span(5, 8, 20, 100, 4);
  Kv4Span e = kv4_span(5, 8, 1, 100, 4);
  Kv4Span c = kv4_span(5, 8, 20, 100, 2);
  printf("%d %d %d / %d %d / %d %d", s.row0, s.n, s.at, e.n, e.at, c.n, c.at);""")
    assert out == "5 3 17 / 3 -2 / 2 17"


def test_rows_that_are_cut_off_still_count(tmp_path):
    """Row arrays that end inside a sequence: its rows keep their positions."""
    out = run_host(tmp_path, """
  Kv4Span s = kv4_span(5, 8, 20, 7, 4);
  Kv4Span e = kv4_span(5, 8, 20, 5, 4);
  Kv4Span n = kv4_span(-2, 3, 20, 9, 4);
  printf("%d %d %d / %d / %d %d %d", s.row0, s.n, s.at, e.n, n.row0, n.n, n.at);""")
    assert out == "5 2 17 / 0 / 0 3 17"


# ------------------------------------------------------------------ refusals
def _lib():
    from bfp import _lib
    return _lib


def _cache(L, **kw):
    d = dict(k=4096, k_e=4096, v=4096, v_e=4096, n_pages=4, page=16, heads=2, hd=64)
    d.update(kw)
    return L.Kv4C(**d)


def _batch(L, **kw):
    d = dict(pages=4096, start=4096, len=4096, n_seq=2, n_rows=4, width=3, max_q=1, max_len=0)
    d.update(kw)
    return L.Kv4BatchC(**d)


def _rows(L, heads=2, type=0, p=4096, e=None, rs=None, hs=64):
    return L.RowsC(p, e, type, heads, heads * 64 if rs is None else rs, hs)


def _refused(L, name, *args):
    rc = getattr(L.lib(), name)(*args)
    assert rc == -22, (name, rc)
    return L.lib().bfp_last_error().decode()


BAD_CACHE = [dict(k=None), dict(v_e=None), dict(page=8), dict(page=48), dict(page=512), dict(n_pages=0), dict(heads=0),
             dict(hd=0), dict(hd=40), dict(hd=272), dict(k=4104), dict(k_e=4097)]
BAD_BATCH = [dict(pages=None), dict(start=None), dict(len=None), dict(n_seq=-1), dict(n_seq=65536), dict(n_rows=-1),
             dict(width=0), dict(max_q=-1), dict(max_len=-1), dict(start=4098)]


@pytest.mark.parametrize("cache,batch", [(c, {}) for c in BAD_CACHE] + [({}, b) for b in BAD_BATCH])
def test_refuses_bad_caches_and_batches(cache, batch):
    L = _lib()
    c, b = _cache(L, **cache), _batch(L, **batch)
    r = _rows(L)
    k, v, q, o = (C.byref(r) for _ in range(4))
    # nothing may be launched here: every call has to stop at the check
    _refused(L, "bfp_kv4_append_d", C.byref(c), C.byref(b), k, v, None, None, None, None, 0, 0, 0, None)
    _refused(L, "bfp_kv4_read_d", C.byref(c), C.byref(b), k, v, None)
    _refused(L, "bfp_kv4_attn_d", C.byref(c), C.byref(b), q, o, 1.0, 0, None, 0, None)
    assert L.lib().bfp_kv4_attn_work(C.byref(c), C.byref(b), q, o, 0) == 0


BAD_ROWS = [dict(p=None), dict(type=4), dict(type=-1), dict(type=3), dict(p=4098), dict(p=4100), dict(rs=-128),
            dict(hs=32), dict(heads=3), dict(rs=132), dict(hs=66), dict(type=3, e=4096, rs=136)]


@pytest.mark.parametrize("bad", BAD_ROWS)
def test_refuses_bad_rows(bad):
    L = _lib()
    c, b, good, r = _cache(L), _batch(L), _rows(L), _rows(L, **bad)
    app = lambda k, v, q=None, o=None: (C.byref(c), C.byref(b), C.byref(k), C.byref(v), q, o, None, None, 0, 0, 0, None)  # noqa: E731
    _refused(L, "bfp_kv4_append_d", *app(r, good))
    _refused(L, "bfp_kv4_append_d", *app(good, r))
    _refused(L, "bfp_kv4_read_d", C.byref(c), C.byref(b), C.byref(r), None, None)
    _refused(L, "bfp_kv4_attn_d", C.byref(c), C.byref(b), C.byref(r), C.byref(good), 1.0, 0, None, 0, None)
    if not {"rs", "hs"} & set(bad) and bad.get("p") not in (4098, 4100) or bad.get("rs") == -128:
        # results may lie at any aligned element, with any strides that keep them apart
        _refused(L, "bfp_kv4_attn_d", C.byref(c), C.byref(b), C.byref(good), C.byref(r), 1.0, 0, None, 0, None)


def test_refuses_bad_calls():
    L = _lib()
    c, b, r = _cache(L), _batch(L), _rows(L)
    R = C.byref(r)
    app = lambda q, o, t, n, rot: _refused(L, "bfp_kv4_append_d", C.byref(c), C.byref(b), R, R, q, o, None, t, n, rot, 0, None)  # noqa: E731
    app(R, None, None, 0, 0)                    # q without q_out
    app(None, R, None, 0, 0)
    app(R, R, None, 0, 0)                       # over k
    app(None, None, 4096, 16, 3)                # odd rot
    app(None, None, 4096, 16, 66)               # wider than the head
    app(None, None, 4096, 16, 0)
    app(None, None, 4096, 0, 64)                # an empty table
    app(None, None, 4100, 16, 64)               # its alignment
    tiles = _rows(L, type=3, e=4096)
    app(R, C.byref(tiles), None, 0, 0)          # rotated queries as tiles
    _refused(L, "bfp_kv4_read_d", C.byref(c), C.byref(b), None, None, None)
    _refused(L, "bfp_kv4_read_d", C.byref(c), C.byref(b), C.byref(tiles), None, None)
    attn = lambda q, *a: _refused(L, "bfp_kv4_attn_d", C.byref(c), C.byref(b), C.byref(q), R, *a)  # noqa: E731
    attn(r, float("nan"), 0, None, 0, None)
    attn(r, 1.0, -1, None, 0, None)
    attn(_rows(L, heads=3), 1.0, 0, None, 0, None)
    attn(_rows(L, heads=1), 1.0, 0, None, 0, None)
    rope = lambda x, n, hd, pos, t, n_pos, rot, y: _refused(  # noqa: E731
        L, "bfp_rope_d", x, n, hd, pos, t, n_pos, rot, 0, y, None)
    rope(None, 4, 64, 4096, 4096, 16, 64, R)
    rope(R, -1, 64, 4096, 4096, 16, 64, R)
    rope(R, 4, 64, None, 4096, 16, 64, R)
    rope(R, 4, 64, 4096, None, 16, 64, R)
    rope(R, 4, 64, 4096, 4096, 0, 64, R)
    rope(R, 4, 64, 4096, 4096, 16, 65, R)
    rope(R, 4, 64, 4096, 4096, 16, 66, R)
    rope(R, 4, 64, 4096, 4096, 16, 64, C.byref(tiles))
    rope(R, 4, 64, 4096, 4096, 16, 64, C.byref(_rows(L, heads=3)))
    inv = np.zeros(256)
    table = lambda *a: _refused(L, "bfp_rope_table_d", inv.ctypes.data, *a, None)  # noqa: E731
    table(0, 1.0, 0, 4, 4096)
    table(257, 1.0, 0, 4, 4096)
    table(4, 1.0, -1, 4, 4096)
    table(4, 1.0, 0, -1, 4096)
    table(4, 1.0, 2 ** 31 - 3, 4, 4096)
    table(4, 1.0, 0, 4, None)


def test_scratch_too_small_is_refused():
    L = _lib()
    c, b = _cache(L, n_pages=4096), _batch(L, width=2000, max_q=1, n_seq=1, n_rows=1)
    r = _rows(L)
    n = L.lib().bfp_kv4_attn_work(C.byref(c), C.byref(b), C.byref(r), C.byref(r), 0)
    assert n > 0
    for work, size in ((None, n), (4096, n - 1), (4104, n)):
        msg = _refused(L, "bfp_kv4_attn_d", C.byref(c), C.byref(b), C.byref(r), C.byref(r), 1.0, 0, work, size, None)
        assert str(n) in msg


def test_nothing_to_do_is_no_error():
    """Empty batches return before any launch (there is no GPU here)."""
    L = _lib()
    c, r = _cache(L), _rows(L)
    R = C.byref(r)
    for kw in (dict(n_seq=0), dict(max_q=0), dict(n_rows=0)):
        b = _batch(L, **kw)
        assert L.lib().bfp_kv4_append_d(C.byref(c), C.byref(b), R, R, None, None, None, None, 0, 0, 0, None) == 0
        assert L.lib().bfp_kv4_read_d(C.byref(c), C.byref(b), R, R, None) == 0
        assert L.lib().bfp_kv4_attn_d(C.byref(c), C.byref(b), R, R, 1.0, 0, None, 0, None) == 0
    assert L.lib().bfp_rope_d(R, 0, 64, 4096, 4096, 16, 64, 0, R, None) == 0


# --------------------------------------------------------------- frequencies
@pytest.mark.parametrize("rot", [2, 16, 34, 64, 128])
@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "parts", "bands"])
def test_frequencies(rot, scaling):
    from bfp.rotary import rope_freqs
    if scaling == "ntk" and rot == 2:
        with pytest.raises(Exception):
            rope_freqs(rot, 10000.0, scaling, 4.0, 2048)
        return
    for base, factor, orig in ((10000.0, 4.0, 2048), (500000.0, 16.0, 8192), (10000.0, 1.0, 100)):
        got, ms = rope_freqs(rot, base, scaling, factor, orig)
        want, wms = ref.freqs(rot, base, scaling, factor, orig)
        # a power, a division and at most two products and a sum, a few 2^-53 each
        assert np.abs(got - want).max() <= 0 + 16 * 2.0 ** -53 * want.max() and (np.abs(got / want - 1) < 1e-12).all()
        assert abs(ms - wms) < 1e-15


def test_frequencies_refuse():
    from bfp._lib import BfpError
    from bfp.rotary import rope_freqs
    for args in ((0,), (3,), (514,), (64, 1.0), (64, float("inf")), (64, 1e4, "linear", 0.5), (64, 1e4, "parts", 2.0, 0),
                 (64, 1e4, "bands", float("nan"), 2048)):
        with pytest.raises(BfpError):
            rope_freqs(*args)
    with pytest.raises(ValueError):
        rope_freqs(64, scaling="other")


# -------------------------------------------------------------------- format
def test_plain_format_is_nearest():
    """The plain conversion the GPU tests compare with: every value goes to
    the nearest element of its tile's grid, and the grid holds the largest."""
    rng = np.random.default_rng(5)
    v = rng.standard_normal((400, 16)) * 2.0 ** rng.integers(-20, 20, (400, 1))
    codes, exps = ref.encode(v)
    got = ref.value(codes, exps)
    grid = np.concatenate([ref.GRID, -ref.GRID])
    scale = 2.0 ** (exps.reshape(-1, 1) - 127.0)
    best = np.abs(v[..., None] - grid * scale[..., None]).min(-1)
    assert (np.abs(got - v) == best).all()
    top = np.abs(v).max(-1)
    assert (top < 7 * scale[:, 0]).all() and (top >= 3.5 * scale[:, 0]).all()


@pytest.mark.parametrize("window", [0, 1, 5])
def test_plain_attention_both_ways(window):
    """The tests' two plain implementations agree."""
    rng = np.random.default_rng(5)
    lens, news = [9, 0, 3, 20], [4, 0, 5, 20]
    start = np.concatenate([[0], np.cumsum(news)])
    keys, vals = ([rng.standard_normal((n, 2, 16)) for n in lens] for _ in range(2))
    there = [rng.random(n) < 0.7 for n in lens]
    q = rng.standard_normal((start[-1], 6, 16))
    for t in (None, there):
        one, two = (f(q, keys, vals, start, lens, 3, 0.4, window, t) for f in (ref.attend, ref.attend_all))
        for x, y in zip(one, two):
            assert np.abs(x - y).max() < 1e-12


def test_what_a_struct_points_to_cannot_be_replaced():
    from bfp._rows import Fixed

    class Thing(Fixed):
        def __init__(self):
            self.k, self._n = 1, 2
    t = Thing()
    t._n = 3
    with pytest.raises(AttributeError):
        t.k = 2
    assert (t.k, t._n) == (1, 3)


def test_more_threads_than_a_launch_has_are_refused():
    """65535 prompts of a million rows each."""
    L = _lib()
    c = C.byref(_cache(L, heads=64))
    b = C.byref(_batch(L, n_seq=65535, n_rows=2 ** 31 - 1, width=70000, max_q=1 << 20))
    r = C.byref(_rows(L, heads=64, rs=4096))
    assert "too many" in _refused(L, "bfp_kv4_attn_d", c, b, r, r, 1.0, 0, 4096, 1 << 62, None)
