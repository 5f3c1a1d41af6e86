"""The 4-bit paged cache and the attention over it against plain 64-bit
numpy: types, layouts, ragged and empty sequences, windows, pages that do
not exist, NaN where nobody looks, splits, graphs, and a step from matvec to
matvec through the cache."""
import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _say(*a):
    print("[kv4]", *a, flush=True)


def _typed(val, kind):
    """float64 values -> (device rows, the values they hold)."""
    import torch
    if kind == "tile":
        from oracle import bfp_sim as sim
        m, e = sim.tile_quantize(val.reshape(-1))
        held = np.asarray(sim.tile_decode(m, e)).reshape(val.shape)
        m = torch.from_numpy(np.ascontiguousarray(np.asarray(m, np.int16).reshape(val.shape))).cuda()
        e = torch.from_numpy(np.ascontiguousarray(np.asarray(e, np.int8).reshape(*val.shape[:-1], -1))).cuda()
        return (m, e), held
    t = torch.from_numpy(val).to(_dt(kind))
    return t.cuda(), t.double().numpy()


def _int(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).cuda()


class Setup:
    """Sequences of lens tokens, the last news of them new; pages dealt out
    of order; every byte of the cache that no token has written is noise."""

    def __init__(self, seed, lens, news, page, heads, hd, spare=3):
        import torch
        from bfp.kv4 import Batch, Fp4Cache
        self.rng = rng = np.random.default_rng(seed)
        self.lens, self.news, self.page, self.heads, self.hd = list(lens), list(news), page, heads, hd
        need = [-(-max(n, 0) // page) for n in lens]
        self.width = max(max(need), 1) + 1
        n_pages = sum(need) + spare
        ids = rng.permutation(n_pages)
        self.table = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.rows = int(self.start[-1])
        self.bytes = {k: rng.integers(0, 256, (n_pages, heads, hd // 16, page) + ((8,) if k in "kv" else ()), dtype=np.uint8)
                      for k in ("k", "ke", "v", "ve")}
        self.keys = [rng.standard_normal((max(n, 0), heads, hd)) * 1.5 for n in lens]
        self.vals = [rng.standard_normal((max(n, 0), heads, hd)) for n in lens]
        for b in range(len(lens)):
            for name, x in (("k", self.keys), ("v", self.vals)):
                codes, exps = ref.encode(x[b]) if len(x[b]) else (np.zeros(x[b].shape, int), np.zeros(x[b].shape[:2] + (hd // 16,), int))
                x[b] = ref.value(codes, exps) if len(x[b]) else x[b]
                for p in range(len(x[b])):
                    self.put(name, b, p, codes[p], exps[p])
        self.cache = Fp4Cache.from_buffers(*(torch.from_numpy(self.bytes[k]).cuda() for k in ("k", "ke", "v", "ve")))
        self.batch = Batch(_int(self.table), _int(self.start), _int(self.lens), max_q=max(max(news), 0), max_len=max(max(lens), 0))

    def put(self, name, b, p, codes, exps):
        where = (self.table[b, p // self.page], slice(None), slice(None), p % self.page)
        self.bytes[name][where] = (codes[..., 0::2] | (codes[..., 1::2] << 4)).reshape(self.heads, self.hd // 16, 8)
        self.bytes[name + "e"][where] = exps

    def positions(self):
        """(sequence, position) of every row."""
        return [(b, max(self.lens[b], 0) - n + i) for b, n in enumerate(self.news) for i in range(n)]


# ------------------------------------------------------------- append, read
APPEND = [  # lens, news, page, heads, hd, query heads, rot, interleaved, type
    ([1], [1], 16, 1, 16, 1, 16, False, "f32"),
    ([5, 17, 16, 33], [1, 1, 1, 1], 16, 3, 64, 9, 64, False, "tile"),
    ([5, 17, 16, 33], [1, 1, 1, 1], 16, 3, 64, 9, 64, True, "bf16"),
    ([40, 0, 100], [40, 0, 17], 32, 2, 128, 4, 128, False, "bf16"),
    ([70, 19], [70, 3], 64, 1, 96, 5, 34, False, "f16"),      # half 17: partners value by value
    ([70, 19], [70, 3], 64, 1, 96, 5, 34, True, "f32"),
    ([20, 2], [20, 2], 16, 5, 80, 0, 40, False, "f32"),       # half 20
    ([300, 1, 2], [300, 1, 2], 256, 2, 256, 2, 64, True, "tile"),
    ([18, 18], [18, 18], 128, 2, 48, 2, 0, False, "bf16"),    # nothing turned
    ([3, 50], [5, 50], 16, 2, 32, 2, 32, False, "f32"),       # more rows than tokens
]


@pytest.mark.parametrize("case", APPEND, ids=str)
def test_append_and_read(gpu, case):
    import torch
    lens, news, page, heads, hd, hq, rot, inter, kind = case
    s = Setup(7, lens, news, page, heads, hd)
    n = s.rows
    (k, kv), (v, vv) = (_typed(s.rng.standard_normal((n, heads, hd)) * 3, kind) for _ in range(2))
    q, qv = _typed(s.rng.standard_normal((n, hq, hd)), kind) if hq else (None, None)
    table = ref.angles(400, rot).astype(np.float32) if rot else None
    where = s.positions()
    pos = np.array([p for _, p in where])
    turn = lambda x: ref.rotate(x, pos, table, inter) if rot else x  # noqa: E731
    wk, wv = turn(kv), vv
    for t, (b, p) in enumerate(where):
        if p >= 0:
            for name, x in (("k", wk), ("v", wv)):
                codes, exps = ref.encode(x[t])
                s.put(name, b, p, codes, exps)
    _say(case)
    qo = s.cache.append(s.batch, k, v, torch.from_numpy(table).cuda() if rot else None, interleaved=inter, q=q)
    # every byte of the cache: what was written, and what was not
    for name, t in (("k", s.cache.k), ("ke", s.cache.k_exp), ("v", s.cache.v), ("ve", s.cache.v_exp)):
        got = t.cpu().numpy()
        if name in "kv":   # a zero has no sign of its own
            got, want = (_unsign(x) for x in (got, s.bytes[name]))
        else:
            want = s.bytes[name]
        assert (got == want).all(), name
    if hq:
        name = "f32" if kind == "tile" else kind
        want = np.where((pos >= 0)[:, None, None], turn(qv), 0)
        tiny = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}[name] / 2
        assert (np.abs(qo.double().cpu().numpy() - want) <= HALF[name] * np.abs(want) + 2.0 ** -49 + tiny).all()
    for dt in ("f32", "bf16"):
        rk, rv = s.cache.read(s.batch, n, dtype=_dt(dt))
        ok = (pos >= 0)[:, None, None]
        assert (rk.double().cpu().numpy() == np.where(ok, ref.quant4(wk), 0)).all()
        assert (rv.double().cpu().numpy() == np.where(ok, ref.quant4(wv), 0)).all()


def _unsign(b):
    lo, hi = b & 15, b >> 4
    return np.where(lo == 8, 0, lo) | (np.where(hi == 8, 0, hi) << 4)


def test_append_borders(gpu):
    """Values on and beside every border between two elements, from each
    side and in float32's smallest steps; exponents at the format's ends;
    infinities and NaN."""
    import torch
    rows = []
    for e in (-130, -101, -100, -99, -20, 0, 3, 97, 100):
        edges = np.concatenate([ref.MIDS, ref.GRID, [7.0, 6.9999995, 7.5, 8.0]])
        for sign in (1, -1):
            v = np.float32(sign) * np.concatenate([edges, np.nextafter(np.float32(edges), np.float32(9)),
                                                   np.nextafter(np.float32(edges), np.float32(-1))]).astype(np.float32)
            v = np.resize(v, 64)
            v[0::16] = 6.0                     # pins the tile's exponent
            rows.append(np.ldexp(v, e).astype(np.float32))
            w = v.copy()
            w[0::16] = v[1::16]
            rows.append(np.ldexp(w, e).astype(np.float32))
    special = np.zeros((6, 64), np.float32)
    special[0, 3], special[1, 20], special[2, 40] = np.inf, -np.inf, np.nan
    special[3, :] = np.float32(3.4e38)
    special[4, :16] = np.float32(1e-45)
    special[5, :] = -0.0
    x = np.stack(rows + list(special)).reshape(-1, 1, 64)
    n = len(x)
    s = Setup(1, [n], [n], 64, 1, 64)
    t = torch.from_numpy(x).cuda()
    s.cache.append(s.batch, t, t)
    rk, rv = s.cache.read(s.batch, n)
    want = ref.quant4(x.astype(np.float64))
    for r in (rk, rv):
        got = r.double().cpu().numpy()
        assert (np.isnan(got) == np.isnan(want)).all()
        assert (got == want)[~np.isnan(want)].all()


def test_append_rotated_borders(gpu):
    """Rotated keys that lie within a few 2^-30 of a border: the products are
    exact and the sum is rounded in 64 bits, so every element is the
    definition's."""
    import torch
    rng = np.random.default_rng(12)
    table = np.stack([np.float32(rng.uniform(-1, 1, (200, 32))), np.float32(rng.uniform(-1, 1, (200, 32)))], -1)
    x = rng.standard_normal((200, 1, 64)).astype(np.float32)
    c, sn = table[..., 0].astype(np.float64), table[..., 1].astype(np.float64)
    # choose a so that a c - b s is near an edge
    edge = rng.choice(ref.MIDS, (200, 32)) * rng.choice([-1, 1], (200, 32))
    b = x[:, 0, 32:].astype(np.float64)
    a = np.where(np.abs(c) > 0.1, (edge + b * sn) / np.where(np.abs(c) > 0.1, c, 1), x[:, 0, :32])
    x[:, 0, :32] = a.astype(np.float32)
    s = Setup(2, [200], [200], 32, 1, 64)
    t = torch.from_numpy(x).cuda()
    s.cache.append(s.batch, t, t, torch.from_numpy(table).cuda())
    rk, _ = s.cache.read(s.batch, 200)
    want = ref.quant4(ref.rotate(x, np.arange(200), table))
    assert (rk.double().cpu().numpy() == want).all()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("hq,hd,rot,n", [(3, 64, 64, 5), (4, 96, 34, 40), (32, 128, 64, 1500), (5, 80, 40, 33)])
def test_append_turns_queries_in_place(gpu, inter, hq, hd, rot, n):
    import torch
    s = Setup(4, [n, 3], [n, 5], 16, 1, hd)       # two rows without a slot: zeros
    table = torch.from_numpy(ref.angles(n, rot).astype(np.float32)).cuda()
    for kind in ("f32", "bf16"):
        k = torch.randn(s.rows, 1, hd, device="cuda", dtype=_dt(kind))
        q = torch.randn(s.rows, hq, hd, device="cuda", dtype=_dt(kind))
        want = s.cache.append(s.batch, k, k, table, interleaved=inter, q=q)
        same = q.clone()
        assert s.cache.append(s.batch, k, k, table, interleaved=inter, q=same, q_out=same) is same
        assert torch.equal(same, want) and (same[n:n + 2] == 0).all()


def test_append_leaves_the_rest(gpu):
    """Rows past the last sequence, pages that do not exist, positions
    outside the table, own positions."""
    import torch
    from bfp.kv4 import Batch
    s = Setup(3, [20, 20, 20], [2, 2, 2], 16, 2, 64)
    bad = s.table.copy()
    bad[0, 1], bad[1, 1] = -5, len(s.bytes["k"])        # the new tokens' pages
    batch = Batch(_int(bad), _int(s.start), _int([20, 20, 200]), max_q=2)   # and a position past the table
    k = torch.randn(9, 2, 64, device="cuda")
    q = torch.randn(9, 4, 64, device="cuda")
    q_out = torch.full((9, 4, 64), 7.0, device="cuda")
    angles = torch.from_numpy(ref.angles(30, 64).astype(np.float32)).cuda()
    s.cache.append(batch, k, k, angles, q=q, q_out=q_out)
    for name, t in (("k", s.cache.k), ("ke", s.cache.k_exp), ("v", s.cache.v), ("ve", s.cache.v_exp)):
        assert (t.cpu().numpy() == s.bytes[name]).all(), name
    assert (q_out[:6] == 0).all() and (q_out[6:] == 7).all()
    out = torch.full((9, 2, 64), 5.0, device="cuda")
    s.cache.read(batch, k=out)
    assert (out[:6] == 0).all() and (out[6:] == 5).all()
    # a position the rotation does not know: NaN, in the query and the cached key; the value is as it is
    pos = _int([0, 30, -1, 29, 5, 5, 0, 0, 0])
    q_out = s.cache.append(s.batch, k, k, angles, pos=pos, q=q)
    rk, rv = s.cache.read(s.batch, 6)
    nan = torch.isnan(rk).flatten(1)
    assert nan[[1, 2]].all() and not nan[[0, 3, 4, 5]].any() and not torch.isnan(rv).any()
    assert torch.isnan(q_out[[1, 2]]).all()
    p = np.array([0, 0, 0, 29, 5, 5])
    want = ref.quant4(ref.rotate(k[:6].double().cpu().numpy(), p, angles.cpu().numpy()))
    assert (rk[[0, 3, 4, 5]].double().cpu().numpy() == want[[0, 3, 4, 5]]).all()


# ---------------------------------------------------------------- attention
def _terms_error(kind, out_kind, rows):
    """How far a probability's own rounding is off: three terms, two, one."""
    if kind == "f32" or out_kind in ("f32", "tile"):
        return 2.0 ** -24
    return 2.0 ** -16 if rows <= 8 or kind != "bf16" or out_kind != "bf16" else 2.0 ** -8


def check(s, q, qv, kind, out_kind, window=0, scale=None, there=None, got=None, max_p=None):
    hq = qv.shape[1]
    sc = s.hd ** -0.5 if scale is None else scale
    want, weight, big = ref.attend(qv, s.keys, s.vals, s.start, s.lens, hq // s.heads, sc, window, there)
    # what the results may be off by; probabilities are carried in one
    # bfloat16 where a tile of 16 columns is full anyway, so the coarser bound
    p_half = _terms_error(kind, out_kind, 1 << 20) if max_p is None else max_p
    bound = ref.attend_bound(want, weight, big, max(max(s.lens), 1), s.hd, HALF[out_kind], p_half)
    g = got.double().cpu().numpy()
    err = np.abs(g - want)
    assert np.isfinite(g).all()
    assert (err <= bound).all(), (err.max(), (err / bound).max())
    return g, want


ATTEND = [  # lens, news, page, heads, hd, group, type, out type, window
    ([1], [1], 16, 1, 16, 1, "f32", "f32", 0),
    ([1, 0, 2, 15, 16, 17], [1] * 6, 16, 3, 64, 3, "bf16", "bf16", 0),
    ([63, 64, 65, 127, 128, 129], [1] * 6, 16, 1, 64, 3, "tile", "f32", 0),
    ([200, 3, 0, 77], [1, 1, 0, 1], 32, 2, 128, 4, "f16", "f16", 0),
    ([300, 555], [1, 1], 64, 2, 128, 8, "bf16", "bf16", 0),
    ([300, 30], [1, 1], 64, 2, 128, 16, "bf16", "bf16", 0),
    ([300, 30], [1, 1], 16, 1, 64, 9, "bf16", "f32", 0),
    ([333, 12], [1, 1], 128, 1, 80, 5, "f32", "f32", 0),
    ([100, 90], [1, 1], 256, 2, 256, 2, "bf16", "bf16", 0),
    ([100, 90], [1, 1], 16, 1, 192, 3, "f16", "f32", 0),
    ([70, 33], [1, 1], 16, 2, 48, 1, "tile", "bf16", 0),
    ([70, 33], [1, 1], 16, 2, 32, 40, "bf16", "bf16", 0),
    ([2000], [1], 16, 3, 64, 3, "bf16", "bf16", 0),          # split
    ([2000, 700], [1, 1], 64, 1, 112, 4, "f32", "f32", 0),
    ([40, 7, 0, 130], [40, 5, 0, 3], 16, 2, 64, 3, "bf16", "bf16", 0),
    ([40, 7, 0, 130], [40, 5, 0, 3], 16, 2, 64, 3, "f32", "f32", 0),
    ([150, 20], [150, 20], 32, 1, 128, 4, "f16", "f16", 0),
    ([150, 20], [64, 20], 32, 1, 96, 1, "tile", "f32", 0),
    ([3, 9, 2], [5, 9, 7], 16, 1, 64, 2, "f32", "f32", 0),    # rows that see nothing
    ([300, 60, 5], [1, 1, 1], 16, 2, 64, 3, "f32", "f32", 1),
    ([300, 60, 5], [1, 1, 1], 16, 2, 64, 3, "bf16", "bf16", 37),
    ([300, 60, 5], [200, 60, 5], 32, 1, 64, 2, "f32", "f32", 50),
    ([300, 60, 5], [200, 60, 5], 32, 1, 128, 4, "bf16", "bf16", 64),
    ([400], [400], 64, 1, 256, 2, "bf16", "bf16", 0),
    ([260, 64], [260, 64], 64, 2, 16, 6, "f32", "bf16", 0),
]


@pytest.mark.parametrize("case", ATTEND, ids=str)
def test_attend(gpu, case):
    lens, news, page, heads, hd, group, kind, out_kind, window = case
    s = Setup(11, lens, news, page, heads, hd)
    q, qv = _typed(s.rng.standard_normal((s.rows, heads * group, hd)) * 2, kind)
    _say(case)
    out = s.cache.attend(s.batch, q, window=window, dtype=_dt(out_kind))
    assert out.dtype == _dt(out_kind)
    check(s, q, qv, kind, out_kind, window, got=out)


def test_attend_row_by_row_is_the_same(gpu):
    """A prompt in one call, in pieces and token by token: float32 results
    within the two calls' own bounds of each other."""
    from bfp.kv4 import Batch
    s = Setup(13, [200], [200], 32, 2, 64)
    q, qv = _typed(s.rng.standard_normal((200, 6, 64)), "f32")
    whole, _ = check(s, q, qv, "f32", "f32", got=s.cache.attend(s.batch, q))
    for a, b in ((0, 1), (0, 64), (64, 65), (65, 200), (199, 200)):
        part = Batch(s.batch.pages, _int([0, b - a]), _int([b]), max_q=b - a)
        got = s.cache.attend(part, q[a:b]).double().cpu().numpy()
        assert np.abs(got - whole[a:b]).max() < 2e-5, (a, b)


def test_attend_strides_and_tiles_out(gpu):
    """Queries inside joined rows, results between other columns, heads
    before rows, tiles out."""
    import torch
    from bfp import _dev
    from bfp._lib import call
    s = Setup(17, [90, 40], [3, 40], 16, 2, 64)
    full = torch.randn(s.rows, 6 + 4, 64, device="cuda")
    q = full[:, 2:8]
    want = s.cache.attend(s.batch, q.contiguous())
    check(s, q, q.double().cpu().numpy(), "f32", "f32", got=want)
    assert torch.equal(s.cache.attend(s.batch, q), want)
    wide = torch.full((s.rows, 9, 64), 3.0, device="cuda")
    s.cache.attend(s.batch, q, out=wide[:, 1:7])
    assert torch.equal(wide[:, 1:7], want) and (wide[:, 0] == 3).all() and (wide[:, 7:] == 3).all()
    turned = torch.empty(6, s.rows, 64, device="cuda").transpose(0, 1)
    assert torch.equal(s.cache.attend(s.batch, q, out=turned), want)
    odd = torch.empty(s.rows * 6 * 65 + 1, device="cuda")[1:].view(s.rows, 6, 65)[:, :, :64]   # any alignment
    assert torch.equal(s.cache.attend(s.batch, q, out=odd), want)
    m = torch.empty(s.rows, 6, 64, dtype=torch.int16, device="cuda")
    e = torch.empty(s.rows, 6, 4, dtype=torch.int8, device="cuda")
    s.cache.attend(s.batch, q, out=(m, e))
    wm, we = torch.empty_like(m), torch.empty_like(e)
    call("bfp_tile_quantize_f32_d", want.data_ptr(), want.numel(), wm.data_ptr(), we.data_ptr(), _dev.stream())
    assert torch.equal(m, wm) and torch.equal(e, we)


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("news", [[1, 1], [33, 70]])
def test_attend_pages_that_do_not_exist(gpu, window, news):
    """Tokens on such pages are not seen; a sequence with none gives zeros."""
    from bfp.kv4 import Batch
    s = Setup(19, [140, 70], news, 16, 2, 64)
    bad = s.table.copy()
    bad[0, 2], bad[0, 8], bad[1, :] = -1, 10 ** 6, -7
    there = [np.array([bad[0, p // 16] in s.table[0] and bad[0, p // 16] >= 0 for p in range(140)]), np.zeros(70, bool)]
    batch = Batch(_int(bad), s.batch.start, s.batch.lens, max_q=max(news), max_len=140)
    q, qv = _typed(s.rng.standard_normal((s.rows, 4, 64)), "f32")
    got, _ = check(s, q, qv, "f32", "f32", window, there=there, got=s.cache.attend(batch, q, window=window))
    assert (got[news[0]:] == 0).all()
    # a length past the table's last page: only what has pages is there
    batch = Batch(s.batch.pages[:, :3].contiguous(), s.batch.start, s.batch.lens, max_q=max(news))
    there = [np.arange(140) < 48, np.arange(70) < 48]
    check(s, q, qv, "f32", "f32", window, there=there, got=s.cache.attend(batch, q, window=window))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("news,window", [([1], 0), ([100], 0), ([60], 20)])
def test_attend_nan_stays_with_those_who_see_it(gpu, kind, news, window):
    """A cached token with NaN in some tiles of its value or key reaches the
    rows that see it and no other."""
    s = Setup(23, [130], news, 16, 1, 64)
    q, qv = _typed(s.rng.standard_normal((s.rows, 3, 64)), kind)
    clean, _ = check(s, q, qv, kind, kind, window, got=s.cache.attend(s.batch, q, window=window))
    pos = np.arange(130 - news[0], 130)
    for p, tile in ((129, 1), (100, 3), (77, 0), (3, 2)):
        where = (int(s.table[0, p // 16]), 0, tile, p % 16)
        sees = (pos >= p) & ((pos - window < p) if window else True)
        for exps, dims in ((s.cache.v_exp, slice(16 * tile, 16 * tile + 16)), (s.cache.k_exp, slice(0, 64))):
            old = int(exps[where])
            exps[where] = 255
            got = s.cache.attend(s.batch, q, window=window).double().cpu().numpy()
            exps[where] = old
            nan = np.zeros(got.shape, bool)
            nan[sees, :, dims] = True
            assert (np.isnan(got) == nan).all(), (p, tile)
            assert (got[~nan] == clean[~nan]).all()


def test_attend_extreme_scores(gpu):
    """Scores of thousands, a scale of zero, a negative one, one that drives
    all but one probability out of range; queries with NaN or infinities
    spoil their own row."""
    import torch
    s = Setup(29, [100, 50], [1, 9], 16, 1, 64)
    q, qv = _typed(s.rng.standard_normal((s.rows, 2, 64)) * 4, "f32")
    for scale in (0.0, -0.3, 20.0):
        check(s, q, qv, "f32", "f32", scale=scale, got=s.cache.attend(s.batch, q, scale=scale))
    good = s.cache.attend(s.batch, q)
    q2 = q.clone()
    q2[2, 1, 5], q2[4, 0, 60] = float("nan"), float("inf")
    got = s.cache.attend(s.batch, q2)
    bad = torch.isnan(got)
    assert bad[2, 1].all() and bad[4, 0].all() and int(bad.sum()) == 128
    assert torch.equal(got[~bad], good[~bad])


def test_attend_large_exponents(gpu):
    """Values and keys at the ends of the format's exponents."""
    s = Setup(31, [80], [2], 16, 1, 32)
    for name, e in (("v", 90), ("v", -100), ("k", -90)):
        s2 = Setup(31, [80], [2], 16, 1, 32)
        x = s2.vals if name == "v" else s2.keys
        x[0] = ref.quant4(x[0] * 2.0 ** e)
        exps = s2.cache.v_exp if name == "v" else s2.cache.k_exp
        for p in range(80):
            exps[int(s2.table[0, p // 16]), :, :, p % 16] = _u8(ref.encode(x[0][p])[1])
            data = s2.cache.v if name == "v" else s2.cache.k
            codes = ref.encode(x[0][p])[0]
            data[int(s2.table[0, p // 16]), :, :, p % 16] = _u8((codes[..., 0::2] | (codes[..., 1::2] << 4)).reshape(1, 2, 8))
        q, qv = _typed(s2.rng.standard_normal((2, 2, 32)) * (2.0 ** 80 if name == "k" else 1), "f32")
        check(s2, q, qv, "f32", "f32", got=s2.cache.attend(s2.batch, q))


def _u8(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.uint8))).cuda()


def test_rows_outside_every_sequence(gpu):
    """Rows before the first and past the last sequence keep what they held;
    sequences without rows are passed over."""
    import torch
    from bfp.kv4 import Batch
    s = Setup(37, [50, 20, 30], [2, 0, 3], 16, 1, 64)
    start = _int(s.start + 2)
    batch = Batch(s.batch.pages, start, s.batch.lens, max_q=3)
    q = torch.randn(10, 2, 64, device="cuda")
    out = torch.full((10, 2, 64), 9.0, device="cuda")
    s.cache.attend(batch, q, out=out)
    assert (out[:2] == 9).all() and (out[7:] == 9).all()
    assert torch.equal(out[2:7], s.cache.attend(s.batch, q[2:7].contiguous()))
    # fewer rows than the sequences claim: the rows that are there
    few = torch.full((4, 2, 64), 9.0, device="cuda")
    s.cache.attend(batch, q[:4].contiguous(), out=few)
    assert torch.equal(few[2:], out[2:4])


def test_long_offsets(gpu):
    """Pages whose bytes lie past 2^31 and 2^32 of the cache's arrays."""
    import torch
    from bfp.kv4 import Batch, Fp4Cache
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB of GPU memory")
    page, heads, hd = 256, 8, 256
    per = heads * page * hd // 2
    n_pages = (1 << 32) // per + 9
    cache = Fp4Cache(n_pages, page, heads, hd)
    ids = [n_pages - 1, 0, (1 << 31) // per + 1, (1 << 32) // per]
    lens, n = [4 * page], 4 * page
    rng = np.random.default_rng(41)
    k, v = (torch.from_numpy(rng.standard_normal((n, heads, hd)).astype(np.float32)).cuda() for _ in range(2))
    cache.append(Batch(_int([ids]), _int([0, n]), _int(lens), max_q=n), k, v)
    rk, rv = cache.read(Batch(_int([ids]), _int([0, n]), _int(lens), max_q=n), n)
    small = Fp4Cache(4, page, heads, hd)
    sb = Batch(_int([[2, 1, 0, 3]]), _int([0, n]), _int(lens), max_q=n)
    small.append(sb, k, v)
    wk, wv = small.read(sb, n)
    assert torch.equal(rk, wk) and torch.equal(rv, wv) and float(rk.abs().max()) > 0
    q = torch.randn(1, 16, hd, device="cuda", dtype=torch.bfloat16)
    one = Batch(_int([ids]), _int([0, 1]), _int(lens), max_q=1)
    assert torch.equal(cache.attend(one, q), small.attend(Batch(_int([[2, 1, 0, 3]]), _int([0, 1]), _int(lens), max_q=1), q))


def test_same_result_every_time(gpu):
    import torch
    s = Setup(43, [1900, 700, 64], [1, 1, 1], 16, 3, 64)
    q = torch.randn(3, 9, 64, device="cuda", dtype=torch.bfloat16)
    first = s.cache.attend(s.batch, q)
    for _ in range(20):
        assert torch.equal(s.cache.attend(s.batch, q), first)


def test_other_stream_and_captured_steps(gpu):
    """A decode step (append, attend) on another stream, and captured and
    replayed while the sequences grow; two graphs with a workspace each,
    replayed in turn."""
    import torch
    from bfp import rotary
    from bfp.kv4 import Batch, Fp4Cache
    heads, hq, hd, page, n = 2, 6, 64, 16, 3
    table = rotary.rope_table(rotary.rope_freqs(hd)[0], 2048)
    pages = torch.arange(n * 64, dtype=torch.int32, device="cuda").view(n, 64).contiguous()
    start = torch.arange(n + 1, dtype=torch.int32, device="cuda")

    def fresh():
        c = Fp4Cache(n * 64, page, heads, hd)
        g = torch.Generator(device="cuda").manual_seed(8)
        k, v = (torch.randn(900, heads, hd, generator=g, device="cuda") for _ in range(2))
        c.append(Batch(pages, _int([0, 800, 880, 900]), _int([800, 80, 20]), max_q=800), k, v, table)
        return c

    def step(cache, batch, x, q_out, out, work):
        cache.append(batch, x[:, hq:hq + heads], x[:, hq + heads:], table, q=x[:, :hq], q_out=q_out)
        cache.attend(batch, q_out, out=out, work=work)

    def state():
        lens = _int([800, 80, 20])
        b = Batch(pages, start, lens, max_q=1, max_len=1024)
        x = torch.zeros(n, hq + 2 * heads, hd, device="cuda")
        q_out, out = torch.zeros(n, hq, hd, device="cuda"), torch.zeros(n, hq, hd, device="cuda")
        cache = fresh()
        work = torch.empty(max(cache.attend_work(b, q_out, out), 1), dtype=torch.uint8, device="cuda")
        return cache, b, x, q_out, out, work, lens
    inputs = [torch.randn(n, hq + 2 * heads, hd, device="cuda") for _ in range(6)]
    cache, b, x, q_out, out, work, lens = state()
    eager = []
    for y in inputs:
        lens += 1
        x.copy_(y)
        step(cache, b, x, q_out, out, work)
        eager.append(out.clone())
    # another stream
    cache, b, x, q_out, out, work, lens = state()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for i, y in enumerate(inputs):
            lens += 1
            x.copy_(y)
            step(cache, b, x, q_out, out, work)
            assert torch.equal(out, eager[i]), i
    torch.cuda.current_stream().wait_stream(s)
    # two captured graphs, replayed in turn
    held = [state() for _ in range(2)]
    graphs = []
    for st in held:
        cache, b, x, q_out, out, work, lens = st
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out.zero_()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(cache, b, x, q_out, out, work)
        graphs.append(graph)
    for i, y in enumerate(inputs):
        for st, graph in zip(held, graphs):
            st[6].add_(1)
            st[2].copy_(y)
            graph.replay()
        torch.cuda.synchronize()
        for st in held:
            assert torch.equal(st[4], eager[i]), i


def test_step_from_matvec_to_matvec(gpu):
    """A layer's attention the way a program with the matvec engine runs it:
    Q, K and V as tiles from the packed weights, rotated and appended, the
    attention's result as tiles into the output projection.  Each stage
    against the plain one on the stage's own inputs."""
    import torch
    from bfp import _dev, api, rotary
    from bfp._lib import call
    from bfp.kv4 import Batch, Fp4Cache
    from oracle import bfp_sim as sim
    D, hq, heads, hd, page, n = 192, 3, 1, 64, 16, 4
    rng = np.random.default_rng(47)
    W = [api.PackedMatrix.from_float(rng.standard_normal((r, D)).astype(np.float32) * 0.05) for r in ((hq + 2 * heads) * hd, D)]
    table = rotary.rope_table(rotary.rope_freqs(hd)[0], 64)
    cache = Fp4Cache(8, page, heads, hd)
    pages = _int([[3, 1], [0, 7], [2, 4], [6, 5]])
    start = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    keys = [np.zeros((0, heads, hd)) for _ in range(n)]
    vals = [np.zeros((0, heads, hd)) for _ in range(n)]

    def matvec(P, xm, xe):
        ym = torch.empty(n, P.n_out, dtype=torch.int16, device="cuda")
        ye = torch.empty(n, P.n_out // 16, dtype=torch.int8, device="cuda")
        call("bfp_matvec_ring_d", _dev.ptr(P.P_m), _dev.ptr(P.P_e), P.n_out, P.n_in, n, 1, 0, 0, xm.data_ptr(),
             xe.data_ptr(), P.n_in, ym.data_ptr(), ye.data_ptr(), P.n_out, 0, _dev.stream())
        return ym, ye
    angles = table.cpu().numpy()
    for step in range(1, 20):
        h, hv = _typed(rng.standard_normal((n, 1, D)), "tile")
        ym, ye = matvec(W[0], h[0].view(n, D), h[1].view(n, D // 16))
        y = (ym.view(n, -1, hd), ye.view(n, -1, hd // 16))
        part = lambda a, b: (y[0][:, a:b], y[1][:, a:b])  # noqa: E731
        batch = Batch(pages, start, _int([step] * n), max_q=1, max_len=32)
        q = cache.append(batch, part(hq, hq + heads), part(hq + heads, hq + 2 * heads), table, q=part(0, hq))
        m = torch.empty(n, hq, hd, dtype=torch.int16, device="cuda")
        e = torch.empty(n, hq, hd // 16, dtype=torch.int8, device="cuda")
        cache.attend(batch, q, out=(m, e))
        om, oe = matvec(W[1], m.view(n, D), e.view(n, D // 16))
        # plain
        yv = np.asarray(sim.tile_decode(ym.cpu().numpy().reshape(-1, 16), ye.cpu().numpy().reshape(-1))).reshape(n, -1, hd)
        pos = np.full(n, step - 1)
        kq = ref.quant4(ref.rotate(yv[:, hq:hq + heads], pos, angles))
        vq = ref.quant4(yv[:, hq + heads:])
        for b in range(n):
            keys[b], vals[b] = np.concatenate([keys[b], kq[b:b + 1]]), np.concatenate([vals[b], vq[b:b + 1]])
        qv = q.double().cpu().numpy()
        wq = ref.rotate(yv[:, :hq], pos, angles)
        assert (np.abs(qv - wq) <= 2.0 ** -24 * np.abs(wq) + 2.0 ** -40).all()
        want, weight, big = ref.attend(qv, keys, vals, np.arange(n + 1), [step] * n, hq, hd ** -0.5)
        bound = ref.attend_bound(want, weight, big, step, hd, 2.0 ** -24, 2.0 ** -24)
        got = np.asarray(sim.tile_decode(m.cpu().numpy().reshape(-1, 16), e.cpu().numpy().reshape(-1))).reshape(want.shape)
        unit = 2.0 ** (e.double().cpu().numpy() - 15)     # a tile's step
        assert (np.abs(got - want) <= bound + np.repeat(unit, 16, -1) / 2).all()
        Wm, We = W[1].unpack()
        for b in range(n):
            xm, xe = m[b].cpu().numpy().reshape(-1, 16), e[b].cpu().numpy().reshape(-1)
            wm, we = sim.tile_quantize(sim.matvec_hw_golden(xm, xe, Wm, We))
            assert (om[b].cpu().numpy() == np.asarray(wm).reshape(-1)).all() and (oe[b].cpu().numpy() == we).all()


def test_refusals(gpu):
    import torch
    from bfp._lib import BfpError
    from bfp.kv4 import Batch, Fp4Cache
    s = Setup(53, [20, 5], [1, 1], 16, 2, 64)
    q = torch.zeros(2, 4, 64, device="cuda")
    k = torch.zeros(2, 2, 64, device="cuda")
    pages, start, lens = s.batch.pages, s.batch.start, s.batch.lens
    for bad in (
            lambda: Fp4Cache(0, 16, 1, 64), lambda: Fp4Cache(1, 24, 1, 64), lambda: Fp4Cache(1, 16, 1, 40),
            lambda: Fp4Cache(1, 16, 1, 272), lambda: Fp4Cache.from_buffers(s.cache.k, s.cache.v, s.cache.v, s.cache.v_exp),
            lambda: Batch(pages[0], start, lens, 1), lambda: Batch(pages.long(), start, lens, 1),
            lambda: Batch(pages, lens, lens, 1), lambda: Batch(pages, start.cpu(), lens, 1),
            lambda: Batch(pages, start, lens, -1),
            lambda: s.cache.append(s.batch, k[:, :1], k[:, :1]), lambda: s.cache.append(s.batch, k, k[:1]),
            lambda: s.cache.append(s.batch, k, k.int()), lambda: s.cache.append(s.batch, k, k, q_out=q),
            lambda: s.cache.append(s.batch, k, k, q=q[:1]), lambda: s.cache.append(s.batch, k, k, pos=start[:1]),
            lambda: s.cache.append(s.batch, k, k, torch.zeros(4, 64, device="cuda")),
            lambda: s.cache.read(s.batch), lambda: s.cache.read(s.batch, k=k[:, :1]),
            lambda: s.cache.attend(s.batch, q[:, :3]), lambda: s.cache.attend(s.batch, q[..., :32]),
            lambda: s.cache.attend(s.batch, q.cpu()), lambda: s.cache.attend(s.batch, q, out=q[:1]),
            lambda: s.cache.attend(s.batch, q.transpose(0, 1).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: s.cache.attend(s.batch, q, window=-1), lambda: s.cache.attend(s.batch, q, scale=float("inf")),
                lambda: s.cache.attend(s.batch, torch.zeros(2 * 4 * 64 + 1, device="cuda")[1:].view(2, 4, 64))):
        with pytest.raises(BfpError):
            bad()
    assert s.cache.attend(s.batch, q[:0]).shape == (0, 4, 64)
