"""The bounds of pages' keys, the pages that they let a row pick, and the
attention over those pages, against plain 64-bit arithmetic."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import HALF, Setup, _dt, _int, _say, _typed

pytestmark = pytest.mark.gpu


def bounds_of(s, b, p):
    """lo, hi (heads, hd) of sequence b's page p: all of its tokens."""
    k = s.keys[b][p * s.page:min((p + 1) * s.page, s.lens[b])]
    return k.min(0), k.max(0)


def all_bounds(s, n_pages, rng=None):
    """Bounds of every page that a sequence holds; anything elsewhere."""
    buf = np.full((n_pages, s.heads, 2, s.hd), 3.0e30)
    for b, n in enumerate(s.lens):
        for p in range(-(-max(n, 0) // s.page)):
            buf[s.table[b, p], :, 0], buf[s.table[b, p], :, 1] = bounds_of(s, b, p)
    return buf


def choose(s, buf, qv, group, n, first, last):
    """Picks by the definition, in 64 bits (math.fsum-like order does not
    matter here: products of few bits)."""
    out = np.full((s.rows, s.heads, n), -1)
    for t, (b, p) in enumerate(s.positions()):
        if p < 0:
            continue
        m = min(p // s.page, s.table.shape[1] - 1) + 1
        ids = s.table[b, :m]
        there = (ids >= 0) & (ids < len(buf))
        for h in range(s.heads):
            q = qv[t, h * group:(h + 1) * group]
            lo, hi = (np.where(there[:, None], buf[np.where(there, ids, 0), h, i], 0) for i in (0, 1))
            score = (np.maximum(q, 0).sum(0) * hi).sum(-1) + (np.minimum(q, 0).sum(0) * lo).sum(-1)
            score[np.isnan(score)] = np.inf
            at = np.arange(m)
            forced = (at < first) | (at >= m - last)
            order = sorted(at[there], key=lambda i: (not forced[i], -score[i], i))[:n]
            out[t, h, :len(order)] = sorted(order)
    return out


def attend_picks(s, qv, picks, group, scale):
    """attend() with a list for every row and KV head."""
    out, weight, big = np.zeros(qv.shape), np.zeros(qv.shape), np.zeros(qv.shape[:2])
    n_pages = s.bytes["k"].shape[0]
    for t, (b, p) in enumerate(s.positions()):
        for h in range(s.heads):
            see = [x for j in picks[t, h] if 0 <= j < s.table.shape[1] and 0 <= s.table[b, j] < n_pages
                   for x in range(j * s.page, (j + 1) * s.page) if x <= p]
            if not see:
                continue
            k, v = s.keys[b][see, h], s.vals[b][see, h]
            for j in range(h * group, (h + 1) * group):
                sc = (k * qv[t, j]).sum(-1) * scale
                big[t, j] = (np.abs(k * qv[t, j]).sum(-1) * abs(scale)).max()
                w = np.exp(sc - sc.max())
                out[t, j] = w @ v / w.sum()
                weight[t, j] = w @ np.abs(v) / w.sum()
    return out, weight, big


# -------------------------------------------------------------------- bounds
@pytest.mark.parametrize("case", [
    ([1], [1], 16, 1, 16), ([5, 17, 16, 33], [1, 1, 1, 1], 16, 3, 64), ([40, 0, 100], [40, 0, 17], 32, 2, 128),
    ([70, 19], [70, 3], 64, 1, 96), ([300, 1, 257], [300, 1, 2], 256, 2, 256), ([129, 130], [1, 130], 128, 5, 80),
    ([3, 50], [5, 50], 16, 2, 48)], ids=str)
def test_bounds(gpu, case):
    import torch
    from bfp.kv4 import PageBounds
    lens, news, page, heads, hd = case
    s = Setup(11, lens, news, page, heads, hd)
    n_pages = s.bytes["k"].shape[0]
    old = torch.randn(n_pages, heads, 2, hd, device="cuda").bfloat16()
    bounds = PageBounds.from_buffer(s.cache, old.clone())
    want = old.double().cpu().numpy()
    for b, (new, n) in enumerate(zip(news, lens)):
        first = max(n - new, 0)
        for p in range(first // page, -(-n // page)) if new and n > first else ():
            want[s.table[b, p], :, 0], want[s.table[b, p], :, 1] = bounds_of(s, b, p)
    _say(case)
    bounds.update(s.batch)
    assert (bounds.buf.double().cpu().numpy() == want).all()


def test_bounds_of_tiles_without_values(gpu):
    """A NaN tile of a token that is there makes its channels' bounds NaN; one
    behind the last token does not."""
    import torch
    from bfp.kv4 import PageBounds
    s = Setup(3, [20, 20], [20, 20], 16, 2, 32)
    s.cache.k_exp[int(s.table[0, 0]), 1, 0, 7] = 255
    s.cache.k_exp[int(s.table[1, 1]), 0, 1, 9] = 255       # position 25
    s.cache.k_exp[int(s.table[1, 0]), 0, 1, 9] = 253       # past bfloat16's range: no value either
    bounds = PageBounds(s.cache)
    bounds.update(s.batch)
    got = bounds.buf.double().cpu().numpy()
    for b in range(2):
        for p in range(2):
            want = np.stack(bounds_of(s, b, p), 1)
            if (b, p) == (0, 0):
                want[1, :, :16] = np.nan
            if (b, p) == (1, 0):
                want[0, :, 16:] = np.nan
            assert np.array_equal(got[s.table[b, p]], want, equal_nan=True), (b, p)
    assert torch.equal(bounds.buf[int(set(range(len(got))).difference(s.table.ravel()).pop())].float(), torch.zeros(2, 2, 32, device="cuda"))


# --------------------------------------------------------------------- picks
SELECT = [  # lens, news, page, heads, hd, query heads, n, first, last, type
    ([1], [1], 16, 1, 16, 1, 1, 0, 1, "f32"),
    ([500, 33, 0, 16], [1, 1, 1, 1], 16, 3, 64, 9, 8, 1, 2, "tile"),
    ([500, 333], [1, 1], 16, 2, 128, 16, 4, 1, 2, "bf16"),
    ([800, 64], [40, 64], 16, 2, 48, 2, 7, 0, 1, "f16"),       # rows by 16, odd widths
    ([300, 299], [3, 5], 16, 1, 80, 5, 3, 2, 1, "f32"),
    ([2000], [2], 32, 1, 256, 4, 20, 1, 4, "bf16"),
    ([40], [40], 16, 2, 112, 2, 30, 1, 1, "f32"),              # more than there are
    ([3, 50], [5, 50], 16, 2, 32, 2, 2, 1, 1, "bf16"),         # more rows than tokens
    ([9000], [1], 16, 1, 32, 1, 40, 1, 2, "f16"),              # several pieces of pages
    ([600], [17], 128, 1, 64, 3, 2, 0, 2, "bf16"),             # nothing but the last
]


@pytest.mark.parametrize("case", SELECT, ids=str)
def test_select(gpu, case):
    import torch
    from bfp.kv4 import PageBounds
    lens, news, page, heads, hd, hq, n, first, last, kind = case
    s = Setup(21, lens, news, page, heads, hd)
    buf = all_bounds(s, s.bytes["k"].shape[0])
    bounds = PageBounds.from_buffer(s.cache, torch.from_numpy(buf).cuda().bfloat16())
    q, qv = _typed(s.rng.standard_normal((s.rows, hq, hd)), kind)
    _say(case)
    got = bounds.select(s.batch, q, n, first=first, last=last).cpu().numpy()
    assert (got == choose(s, buf, qv, hq // heads, n, first, last)).all()


def _flat(lens, news, page, heads, hd, hq, fill, seed=5, kind="f32"):
    """A batch whose pages all have the bounds that fill(rng, page number) gives."""
    import torch
    from bfp.kv4 import PageBounds
    s = Setup(seed, lens, news, page, heads, hd)
    n_pages = s.bytes["k"].shape[0]
    buf = np.stack([fill(s.rng, i) for i in range(n_pages)])
    t = torch.from_numpy(buf).cuda().bfloat16()
    q, qv = _typed(s.rng.standard_normal((s.rows, hq, hd)), kind)
    return s, t.double().cpu().numpy(), PageBounds.from_buffer(s.cache, t), q, qv


def test_select_equal_scores(gpu):
    """All pages alike, or alike in groups: the lower ones."""
    one = np.random.default_rng(1).standard_normal((4, 2, 2, 32))
    for kinds in (1, 4):
        for lens, news in (([700, 64], [2, 2]), ([700], [30]), ([700], [300]), ([3000, 5], [4, 1]), ([3000], [300])):
            s, buf, bounds, q, qv = _flat(lens, news, 16, 2, 32, 4, lambda rng, i: one[i * 7 % kinds])
            got = bounds.select(s.batch, q, 9, first=1, last=2).cpu().numpy()
            assert (got == choose(s, buf, qv, 2, 9, 1, 2)).all()


def test_select_scores_closer_than_float32(gpu):
    """Scores that differ by less than float32 sums can tell: a large term
    that all pages share, and a small one that orders them."""
    def fill(rng, i):
        b = np.zeros((1, 2, 64))
        b[..., 0] = 2.0 ** 20
        b[..., 1:] = rng.integers(-8, 9, 63) * 2.0 ** -6
        return b
    import torch
    for news in ([1, 1], [20, 20]):
        s, buf, bounds, q, qv = _flat([900, 500], news, 16, 1, 64, 2, fill)
        q = torch.ones_like(q) + q.sign() * 2.0 ** -10
        qv = q.double().cpu().numpy()
        got = bounds.select(s.batch, q, 11, first=0, last=1).cpu().numpy()
        assert (got == choose(s, buf, qv, 2, 11, 0, 1)).all()


def test_select_extremes(gpu):
    """NaN bounds come first, infinite queries and scores past float32 choose
    by the 64-bit scores all the same, pages that the cache does not have are
    not picked."""
    import torch

    def fill(rng, i):
        b = rng.standard_normal((2, 2, 32)) * 2.0 ** 100
        if i % 13 == 5:
            b[1] = np.nan
        return b
    s, buf, bounds, q, qv = _flat([640, 320], [1, 3], 16, 2, 32, 4, fill)
    q = q * 2.0 ** 60
    q[1, 0, 3] = float("inf")
    s.batch.pages[0, 7] = -1
    s.batch.pages[0, 9] = 2 ** 30
    s.table[0, 7], s.table[0, 9] = -1, 2 ** 30
    got = bounds.select(s.batch, q, 12, first=1, last=2).cpu().numpy()
    want = choose(s, buf, q.double().cpu().numpy(), 2, 12, 1, 2)
    assert (got[0] == want[0]).all() and (got[2:] == want[2:]).all()
    assert (got[1, 1] == want[1, 1]).all()      # the other KV head of the row with the infinity
    assert torch.isfinite(q).sum() == q.numel() - 1


@pytest.mark.parametrize("news", [[1, 1], [7, 9]])
def test_select_scores_below_float32(gpu, news):
    """Scores that are minus infinity in float32 are pages all the same."""
    def fill(rng, i):
        return -2.0 ** 100 * rng.integers(1, 100, (2, 1, 32)).repeat(2, 1)
    s, buf, bounds, q, qv = _flat([640, 320], news, 16, 2, 32, 4, fill)
    q = (q.abs() + 0.5) * 2.0 ** 60
    got = bounds.select(s.batch, q, 12, first=1, last=2).cpu().numpy()
    assert (got == choose(s, buf, q.double().cpu().numpy(), 2, 12, 1, 2)).all()


@pytest.mark.parametrize("width", [3000, 6200, 7000, 7943, 7944, 16384])
def test_select_of_wide_tables(gpu, width):
    """Scores of more and more pages in the workgroup's memory."""
    import torch
    from bfp.kv4 import Batch, Fp4Cache, PageBounds
    cache = Fp4Cache(width, 16, 1, 16)
    g = torch.Generator().manual_seed(width)
    buf = torch.randint(-64, 65, (width, 1, 2, 16), generator=g).bfloat16()
    order = torch.randperm(width, generator=g)
    for rows in (1, 530):
        batch = Batch(_int(order.numpy()[None]), _int([0, rows]), _int([16 * width]), max_q=rows)
        q = torch.randint(-8, 9, (rows, 1, 16), generator=g).float().cuda()
        got = PageBounds.from_buffer(cache, buf.cuda()).select(batch, q, 33, first=1, last=2).cpu()
        b, x = buf[order].double(), q.double().cpu()
        for t in {0, rows // 2, rows - 1}:
            m = (16 * width - rows + t) // 16 + 1
            score = ((x[t, 0].clamp(min=0) * b[:m, 0, 1]).sum(-1) + (x[t, 0].clamp(max=0) * b[:m, 0, 0]).sum(-1)).numpy()   # whole numbers
            score[[0, m - 2, m - 1]] = np.inf
            want = sorted(np.lexsort((np.arange(m), -score))[:33])
            assert (got[t, 0].numpy() == want).all(), (rows, t)


def test_select_leaves_other_rows(gpu):
    import torch
    s, buf, bounds, q, qv = _flat([100, 90], [2, 3], 16, 1, 16, 1, lambda rng, i: rng.standard_normal((1, 2, 16)))
    out = torch.full((s.rows + 4, 1, 3), 77, dtype=torch.int32, device="cuda")
    more = torch.cat([q, q[:4]])
    got = bounds.select(s.batch, more, 3, out=out).cpu().numpy()
    assert (got[:s.rows] == choose(s, buf, qv, 1, 3, 1, 2)).all() and (got[s.rows:] == 77).all()


def test_select_in_pieces(gpu, monkeypatch):
    """More scores than the scratch is given at once."""
    lens, news = [60000], [1200]
    rng = np.random.default_rng(2)
    import torch
    from bfp.kv4 import Batch, Fp4Cache, PageBounds
    width = 60000 // 16
    cache = Fp4Cache(width, 16, 16, 16)
    bounds = PageBounds.from_buffer(cache, torch.from_numpy(rng.standard_normal((width, 16, 2, 16))).cuda().bfloat16())
    batch = Batch(_int(rng.permutation(width)[None]), _int([0, 1200]), _int([60000]), max_q=1200)
    q = torch.randn(1200, 16, 16, device="cuda")
    assert bounds.select_work(batch, q) <= 1 << 28
    got = bounds.select(batch, q, 6, first=0, last=1)
    b = bounds.buf[batch.pages[0].long()].double()               # width, heads, 2, hd
    x = q.double()
    for t in (0, 1, 500, 1023, 1024, 1199):
        score = (x[t].clamp(min=0) * b[:, :, 1]).sum(-1) + (x[t].clamp(max=0) * b[:, :, 0]).sum(-1)     # width, heads
        m = (60000 - 1200 + t) // 16 + 1
        score = score[:m]
        score[m - 1] = float("inf")
        want = score.topk(6, dim=0)[1].sort(dim=0)[0].t()
        assert (got[t].long() == want).all(), t


# ----------------------------------------------------------------- attention
PICKED = [  # lens, news, page, heads, hd, query heads, n, type, out type
    ([1], [1], 16, 1, 16, 1, 1, "f32", None),
    ([500, 33, 0, 16], [1, 1, 1, 1], 16, 3, 64, 9, 8, "tile", None),
    ([500, 333], [1, 1], 16, 2, 128, 32, 4, "bf16", None),        # 16 query heads a KV head
    ([300, 200], [3, 20], 16, 2, 48, 2, 5, "f16", None),
    ([300, 300], [2, 2], 32, 1, 80, 40, 6, "f32", None),          # several row tiles a token
    ([900], [1], 64, 1, 256, 8, 9, "bf16", "f32"),
    ([700], [2], 256, 2, 192, 2, 2, "bf16", None),
    ([3, 50], [5, 50], 16, 2, 32, 2, 2, "bf16", None),            # more rows than tokens
    ([6000, 5000], [1, 1], 16, 1, 64, 3, 200, "f32", None),       # shared by many workgroups
    ([5000], [1], 64, 2, 128, 8, 70, "bf16", None),
    ([1200], [700], 16, 2, 64, 4, 4, "f16", None),                # many rows
    ([1000], [900], 16, 2, 32, 2, 4, "bf16", None),               # and more
    ([900], [800], 32, 2, 256, 2, 3, "f32", None),
    ([9000], [1], 64, 2, 64, 4, 80, "bf16", None),                # long lists
    ([2600, 1500], [1, 1], 64, 1, 256, 4, 20, "f16", None),
    ([2600, 1500], [1, 2], 128, 1, 160, 20, 12, "tile", None),
]


@pytest.mark.parametrize("case", PICKED, ids=str)
def test_attend_picks(gpu, case):
    import torch
    lens, news, page, heads, hd, hq, n, kind, out = case
    s = Setup(31, lens, news, page, heads, hd)
    group, scale = hq // heads, 1 / np.sqrt(hd)
    q, qv = _typed(s.rng.standard_normal((s.rows, hq, hd)) * 1.5, kind)
    picks = np.full((s.rows, heads, n), -1)
    for t, (b, p) in enumerate(s.positions()):
        for h in range(heads):
            m = max(p // page, 0) + 1
            k = min(n, m)
            picks[t, h, :k] = s.rng.permutation(m)[:k]
            if t % 3 == 1:
                s.rng.shuffle(picks[t, h])                        # lists with gaps
    _say(case)
    got = s.cache.attend(s.batch, q, picks=_int(picks), dtype=_dt(out) if out else None)
    want, weight, big = attend_picks(s, qv, picks, group, scale)
    res = out or ("f32" if kind == "tile" else kind)
    one = res == "bf16" and kind == "bf16" and group > 8
    # probabilities: whole in float32, 2^-16 in two terms, rounded to bfloat16 in one
    p_half = 2.0 ** -24 if "f32" in (kind, res) or kind == "tile" else 2.0 ** -8 if one else 2.0 ** -16
    bound = ref.attend_bound(want, weight, big, n * page, hd, HALF[res], 2 * p_half)
    bad = np.abs(got.double().cpu().numpy() - want) - bound
    assert (bad <= 0).all(), (bad.max(), np.unravel_index(bad.argmax(), bad.shape))


def test_picks_of_all_pages_are_plain_attention(gpu):
    """A list of every page gives what attend without a list gives, to the
    order of the sums."""
    import torch
    s = Setup(8, [200, 77, 16], [4, 1, 3], 16, 2, 64)
    q, qv = _typed(s.rng.standard_normal((s.rows, 6, 64)), "f32")
    every = torch.arange(s.width, device="cuda", dtype=torch.int32).repeat(s.rows, 2, 1).contiguous()
    a, b = s.cache.attend(s.batch, q), s.cache.attend(s.batch, q, picks=every)
    want, weight, big = attend_picks(s, qv, every.cpu().numpy(), 3, 1 / 8)
    bound = ref.attend_bound(want, weight, big, 208, 64, HALF["f32"], 2.0 ** -24)
    assert (np.abs((a - b).double().cpu().numpy()) <= 2 * bound).all()


def test_lists_that_name_nothing(gpu):
    """Numbers outside the table and pages that the cache does not have are
    not seen; a row with nothing to see is zero; other rows stay."""
    import torch
    s = Setup(9, [100, 60], [1, 1], 16, 1, 32)
    s.batch.pages[0, 2] = 10 ** 6
    s.table[0, 2] = 10 ** 6
    q, qv = _typed(s.rng.standard_normal((3, 2, 32)), "f32")
    picks = np.array([[[-5, 2, 1, 2 ** 31 - 1]], [[-1, -1, s.width, -2 ** 31]], [[0, 1, 2, 3]]])
    out = torch.full((3, 2, 32), 7.0, device="cuda")
    s.cache.attend(s.batch, q, picks=_int(picks), out=out)
    got = out.double().cpu().numpy()
    want, weight, big = attend_picks(s, qv[:2], picks, 2, 1 / np.sqrt(32))
    assert (np.abs(got[:2] - want) <= ref.attend_bound(want, weight, big, 64, 32, HALF["f32"], 2.0 ** -23)).all()
    assert (got[1] == 0).all() and (got[2] == 7).all()


@pytest.mark.parametrize("many", [False, True])
def test_picked_rows_do_not_see_other_bytes(gpu, many):
    """NaN keys and values in pages that are not listed, or behind a row's
    position; a listed NaN value shows."""
    import torch
    news = [3, 3] if not many else [40, 40]
    s = Setup(10, [100, 90], news, 16, 2, 32)
    clean = s.cache.attend
    q, qv = _typed(s.rng.standard_normal((s.rows, 4, 32)), "f32")
    picks = np.zeros((s.rows, 2, 2), int)
    for t, (b, p) in enumerate(s.positions()):
        picks[t, :, 1] = p // 16
    want, weight, big = attend_picks(s, qv, picks, 2, 1 / np.sqrt(32))
    for b in range(2):                                   # a page that nobody lists; slots behind the end
        listed = set(picks[s.start[b]:s.start[b + 1]].ravel())
        for p in range(-(-s.lens[b] // 16)):
            if p not in listed:
                s.cache.k_exp[int(s.table[b, p])] = 255
                s.cache.v_exp[int(s.table[b, p])] = 255
        last = s.lens[b] // 16
        s.cache.k_exp[int(s.table[b, last]), :, :, s.lens[b] % 16:] = 255
        s.cache.v_exp[int(s.table[b, last]), :, :, s.lens[b] % 16:] = 254
    got = clean(s.batch, q, picks=_int(picks)).double().cpu().numpy()
    assert (np.abs(got - want) <= ref.attend_bound(want, weight, big, 32, 32, HALF["f32"], 2.0 ** -23)).all()
    # the newest value of sequence 0: its last row alone sees it
    s.cache.v_exp[int(s.table[0, 99 // 16]), 1, 0, 99 % 16] = 255
    got = clean(s.batch, q, picks=_int(picks)).double().cpu().numpy()
    t = s.start[1] - 1
    assert np.isnan(got[t, 2:, :16]).all() and np.isfinite(got[t, 2:, 16:]).all() and np.isfinite(got[t, :2]).all()
    assert np.isfinite(np.delete(got, t, 0)).all()


def test_steps_with_pool_bounds_and_picks(gpu):
    """A sequence grows token by token and is forked: pages from a pool that
    moves keys and bounds, picks, attention; every step against plain
    arithmetic."""
    import torch
    from bfp.kv4 import Batch, Fp4Cache, PageBounds
    from bfp.pages import PagePool
    rng = np.random.default_rng(4)
    cache = Fp4Cache(40, 16, 2, 32)
    bounds = PageBounds(cache)
    pool = PagePool([cache, bounds])
    table = torch.full((3, 12), -1, dtype=torch.int32, device="cuda")
    lens = _int([0, 0, 0])
    keys, vals = [np.zeros((0, 2, 32))] * 3, [np.zeros((0, 2, 32))] * 3

    def step(live, new):
        start = np.concatenate([[0], np.cumsum([new if b in live else 0 for b in range(3)])])
        batch = Batch(table, _int(start), lens, max_q=new)
        batch.lens += _int([new if b in live else 0 for b in range(3)])
        pool.reserve(batch)
        n = int(start[-1])
        k, v, q = (rng.standard_normal((n, h, 32)) for h in (2, 2, 4))
        f = lambda x: torch.from_numpy(x).float().cuda()  # noqa: E731
        cache.append(batch, f(k), f(v))
        bounds.update(batch)
        for b in live:
            rows = slice(start[b], start[b + 1])
            keys[b] = np.concatenate([keys[b], ref.quant4(k[rows].astype(np.float32))])
            vals[b] = np.concatenate([vals[b], ref.quant4(v[rows].astype(np.float32))])
        picks = bounds.select(batch, f(q), 3, first=1, last=1)
        out = cache.attend(batch, f(q), picks=picks).double().cpu().numpy()
        got = picks.cpu().numpy()
        qv = q.astype(np.float32).astype(np.float64)
        for b in live:
            for i in range(new):
                t, p = start[b] + i, len(keys[b]) - new + i
                for h in range(2):
                    # bounds are of all tokens up to the batch's last
                    pages = [keys[b][16 * j:16 * j + 16, h] for j in range(p // 16 + 1)]
                    x = qv[t, 2 * h:2 * h + 2]
                    sc = [sum(np.maximum(y * a.min(0), y * a.max(0)).sum() for y in x) for a in pages]
                    sc[0], sc[-1] = np.inf, np.inf
                    want = sorted(sorted(range(len(sc)), key=lambda j: (-sc[j], j))[:3])
                    assert list(got[t, h][:len(want)]) == want and (got[t, h][len(want):] == -1).all()
                    see = [j for w in want for j in range(16 * w, 16 * w + 16) if j <= p]
                    for e in range(2):
                        s = keys[b][see, h] @ x[e] / np.sqrt(32)
                        w = np.exp(s - s.max())
                        o = w @ vals[b][see, h] / w.sum()
                        big = (np.abs(keys[b][see, h]) @ np.abs(x[e])).max() / np.sqrt(32)
                        bound = ref.attend_bound(o, w @ np.abs(vals[b][see, h]) / w.sum(), np.array(big), len(see), 32, HALF["f32"], 2.0 ** -24)
                        assert (np.abs(out[t, 2 * h + e] - o) <= bound).all()
    step([0], 30)
    for _ in range(4):
        step([0], 7)
    print("[kv4] fork", flush=True)
    pool.fork(table[0:1], lens[0:1], _int([0, 0]), out=(table[1:3], lens[1:3]))
    keys[1:], vals[1:] = [keys[0]] * 2, [vals[0]] * 2
    step([0, 1, 2], 1)
    step([0, 1, 2], 9)
    pool.free(table[0:1])
    lens[0:1].zero_()
    keys[0] = vals[0] = np.zeros((0, 2, 32))
    live = int(pool.compact(table))
    print("[kv4] compact", live, flush=True)
    assert int(table.max()) == live - 1 and int((pool.refs > 0).sum()) == live
    step([1, 2], 20)
    assert int(pool.short) == 0


def test_captured_picks(gpu):
    """Bounds, picks and attention captured once and replayed while lengths
    and queries change; two graphs share the scratch in turn."""
    import torch
    from bfp.kv4 import PageBounds
    s = Setup(12, [400, 200], [1, 1], 16, 2, 64)
    bounds = PageBounds.from_buffer(s.cache, torch.from_numpy(all_bounds(s, s.bytes["k"].shape[0])).cuda().bfloat16())
    q = torch.randn(2, 4, 64, device="cuda")
    picks = torch.empty(2, 2, 6, dtype=torch.int32, device="cuda")
    work = torch.empty(max(bounds.select_work(s.batch, q), s.cache.attend_work(s.batch, q, picks=picks), 16), dtype=torch.uint8, device="cuda")
    outs, graphs = [torch.empty_like(q), torch.empty_like(q)], []

    def step(out):
        bounds.update(s.batch)
        bounds.select(s.batch, q, 6, out=picks, work=work)
        s.cache.attend(s.batch, q, picks=picks, out=out, work=work)
    side = torch.cuda.Stream()
    for out in outs:
        with torch.cuda.stream(side):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                step(out)
            graphs.append(g)
    torch.cuda.synchronize()
    for i in range(4):
        q.copy_(torch.randn(2, 4, 64, device="cuda"))
        s.batch.lens.copy_(_int([400 - 37 * i, 200 - 16 * i]))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = s.cache.attend(s.batch, q, picks=bounds.select(s.batch, q, 6))
        for out in outs:
            assert torch.equal(out, want)


def test_refusals_of_the_python_side(gpu):
    import torch
    from bfp.kv4 import Fp4Cache, PageBounds
    s = Setup(1, [40], [1], 16, 2, 32)
    bounds = PageBounds(s.cache)
    q = torch.randn(1, 4, 32, device="cuda")
    good = torch.zeros(1, 2, 2, dtype=torch.int32, device="cuda")
    for bad in (good.long(), good[:, :1], good.cpu(), good[0], torch.zeros(1, 2, 4, dtype=torch.int32, device="cuda")[:, :, ::2]):
        with pytest.raises(ValueError):
            s.cache.attend(s.batch, q, picks=bad)
    with pytest.raises(ValueError):
        s.cache.attend(s.batch, q, picks=good, window=3)
    with pytest.raises(ValueError):
        PageBounds.from_buffer(s.cache, bounds.buf.float())
    with pytest.raises(ValueError):
        bounds.select(s.batch, q[:, :3], 2)
    for kw in (dict(n=0), dict(n=2, first=-1), dict(n=2, last=0), dict(n=2 ** 31)):
        with pytest.raises(ValueError):
            bounds.select(s.batch, q, **kw)
    with pytest.raises(Exception, match="first=1 and last=2"):
        bounds.select(s.batch, q, 2)
    with pytest.raises(ValueError):
        bounds.select(s.batch, q, 3, out=good)
    with pytest.raises(ValueError):
        bounds.select(s.batch, q, 3, work=torch.empty(64, device="cuda")[::2])
    with pytest.raises(Exception, match="scratch"):
        bounds.select(s.batch, q, 3, work=torch.empty(1, device="cuda"))
    with pytest.raises(AttributeError):
        bounds.buf = good
    assert Fp4Cache(2, 16, 1, 16).attend is not None
