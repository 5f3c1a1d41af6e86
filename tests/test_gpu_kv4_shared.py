"""Attention over a prefix that sequences share, against plain 64-bit
arithmetic over each sequence's own tokens: what a group shares is read from
the group's pages and nowhere else."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import HALF, _dt, _int, _say, _typed

pytestmark = pytest.mark.gpu


class Cached:
    """Sequences of lens tokens with pages dealt out of order, random tiles,
    and noise in every byte that no token has."""

    def __init__(self, seed, lens, page, heads, hd, spare=3):
        import torch
        from bfp.kv4 import Fp4Cache
        self.rng = rng = np.random.default_rng(seed)
        need = [-(-max(n, 0) // page) for n in lens]
        n_pages = sum(need) + spare
        ids = rng.permutation(n_pages)
        self.width = max(max(need), 1) + 1
        self.table = np.full((len(lens), self.width), -1, np.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = ids[sum(need[:b]):sum(need[:b + 1])]
        held = {}
        for name in "kv":
            data = rng.integers(0, 256, (n_pages, heads, hd // 16, page, 8), dtype=np.uint8)
            exps = rng.integers(0, 256, (n_pages, heads, hd // 16, page), dtype=np.uint8)
            values = []
            for b, n in enumerate(lens):
                n = max(n, 0)
                codes, e = rng.integers(0, 16, (n, heads, hd)), rng.integers(124, 128, (n, heads, hd // 16))
                at, slot = self.table[b, np.arange(n) // page], np.arange(n) % page
                data[at, :, :, slot] = (codes[..., 0::2] | (codes[..., 1::2] << 4)).reshape(n, heads, hd // 16, 8)
                exps[at, :, :, slot] = e
                values.append(ref.value(codes, e))
            held[name], held[name + "e"] = data, exps
            setattr(self, {"k": "keys", "v": "vals"}[name], values)
        self.cache = Fp4Cache.from_buffers(*(torch.from_numpy(held[x]).cuda() for x in ("k", "ke", "v", "ve")))


class Groups:
    """share: tokens of each group; of: the group of each sequence (-1:
    none), neighbours alike; lens with the shared tokens.  A sequence's own
    table holds nonsense before the shared tokens end, and where they end
    inside a page, that page's slots before the end hold other tokens."""

    def __init__(self, seed, share, of, lens, news, page, heads, hd, max_rows=None, hints=True):
        from bfp.kv4 import Batch, Shared
        g = len(share)
        self.s = s = Cached(seed, list(share) + list(lens), page, heads, hd)
        self.g, self.lens, self.news, self.of = g, list(lens), list(news), of
        self.start = np.concatenate([[0], np.cumsum(news)])
        self.rows = int(self.start[-1])
        bounds = [0] * (g + 1)                          # groups of neighbours: where each begins
        for k in range(g):
            mine = [b for b, x in enumerate(of) if x == k]
            bounds[k] = mine[0] if mine else bounds[k - 1] if k else 0
            bounds[k + 1] = mine[-1] + 1 if mine else bounds[k]
        assert all(bounds[x] <= b < bounds[x + 1] for b, x in enumerate(of) if x >= 0)
        assert not any(bounds[0] <= b < bounds[g] for b, x in enumerate(of) if x < 0)      # (between groups: one that shares 0)
        self.table = s.table[g:].copy()
        self.keys, self.vals, self.there = [], [], []
        for b, n in enumerate(lens):
            p = share[of[b]] if of[b] >= 0 else 0
            a = min(max(n, 0), p)
            k, v = s.keys[g + b], s.vals[g + b]
            self.keys.append(np.concatenate([s.keys[max(of[b], 0)][:a], k[a:]]) if a else k)
            self.vals.append(np.concatenate([s.vals[max(of[b], 0)][:a], v[a:]]) if a else v)
            self.table[b, :p // page] = [-1, 2 ** 30, 0][b % 3]
        news_of = [sum(n for n, x in zip(news, of) if x == k) for k in range(g)]
        self.batch = Batch(_int(self.table), _int(self.start), _int(lens), max_q=max(max(news), 0), max_len=max(max(lens), 0) if hints else 0)
        self.shared = Shared(_int(s.table[:g]), _int(bounds), _int(share), max_rows=max(news_of) if max_rows is None else max_rows,
                             max_len=max(share) if hints else 0)

    def want(self, qv, group, scale, window):
        return ref.attend_all(qv, self.keys, self.vals, self.start, self.lens, group, scale, window)


def _bound(want, weight, big, n_keys, hd, kind, res, rows):
    """Probabilities: whole in float32 results, 2^-16 off in two terms, rounded to
    bfloat16 where a part has more than 8 rows a KV head in bfloat16."""
    p_half = 2.0 ** -24 if "f32" in (kind, res) or "tile" in (kind, res) else 2.0 ** -8 if (kind, res) == ("bf16", "bf16") and rows > 8 else 2.0 ** -16
    return ref.attend_bound(want, weight, big, n_keys, hd, HALF[res], 2 * p_half)


CASES = [  # share, of, lens, news, page, heads, hd, query heads, type, result, window
    ([1], [0], [2], [1], 16, 1, 16, 1, "f32", None, 0),
    ([304], [0] * 5, [500, 305, 444, 320, 330], [1] * 5, 16, 3, 64, 9, "tile", None, 0),
    ([40, 77], [0, 0, 1, 1, 1], [41, 60, 80, 78, 200], [1] * 5, 16, 2, 128, 8, "bf16", None, 0),
    ([40, 77], [-1, 0, 0, 1, -1], [30, 60, 41, 90, 10], [2, 1, 1, 3, 4], 16, 2, 48, 4, "f16", None, 0),     # some share nothing
    ([100], [0, 0, 0, 0], [100, 50, 0, 103], [3, 2, 1, 4], 16, 1, 32, 2, "f32", None, 0),                    # rows inside the prefix, none
    ([100], [0, 0], [120, 3], [5, 5], 32, 2, 80, 2, "bf16", "f32", 0),                                       # more rows than tokens
    ([64, 0, 32], [0, 0, 1, 2], [70, 65, 9, 40], [1, 1, 2, 1], 64, 1, 96, 3, "f16", None, 0),                # nothing shared
    ([200], [0, 0, 0], [260, 230, 201], [20, 9, 1], 16, 2, 64, 4, "bf16", None, 50),                         # a window into the prefix
    ([300], [0, 0, 0], [400, 330, 301], [60, 20, 1], 64, 1, 128, 4, "f16", None, 90),                        # and past it, for some
    ([5000], [0] * 3, [5040, 5001, 5300], [1, 1, 1], 64, 2, 128, 8, "bf16", None, 0),                        # keys shared out
    ([4000], [0] * 40, [4000 + 3 * i + 1 for i in range(40)], [1] * 40, 32, 1, 64, 8, "bf16", None, 0),      # prompts' kernel, split
    ([1000, 700], [0] * 6 + [1] * 5, [1100] * 6 + [790] * 5, [13] * 6 + [14] * 5, 64, 2, 96, 8, "f16", None, 0),  # rows of one and a quarter workgroups
    ([1000], [0] * 7, [1100] * 7, [11] * 7, 16, 1, 32, 4, "bf16", None, 400),
    ([6000, 900], [0] * 9 + [1] * 3, [6100] * 9 + [1000] * 3, [3] * 12, 64, 1, 128, 4, "bf16", None, 0),
    ([6000], [0] * 9, [6100] * 9, [3] * 9, 16, 2, 112, 6, "f16", None, 0),
    ([700], [0] * 9, [800] * 9, [10] * 9, 32, 1, 128, 3, "f16", None, 200),
    ([21000], [0] * 3, [21010, 21050, 21001], [1] * 3, 64, 8, 48, 8, "f16", None, 0),                        # few rows that share out their keys
    ([27000], [0] * 2, [27001, 27300], [1, 2], 128, 1, 128, 2, "bf16", None, 0),
    ([34000], [0] * 2, [34001, 34002], [1, 1], 256, 1, 256, 2, "f16", None, 0),
    ([500], [0, 0], [6600, 6200], [600, 560], 64, 1, 64, 2, "bf16", None, 0),                                # prompts behind it, split
    ([3000], [0] * 8, [3100] * 8, [40] * 8, 64, 1, 256, 4, "bf16", None, 700),
    ([3100], [0] * 8, [3200] * 8, [40] * 8, 64, 1, 192, 4, "f16", None, 0),
    ([2000], [0] * 8, [2100] * 8, [40] * 8, 32, 1, 240, 4, "f32", None, 0),
    ([500] * 66, list(range(66)), [540 + g for g in range(66)], [20] * 66, 32, 1, 64, 16, "bf16", None, 0),
    ([900, 700], [0] * 6 + [1] * 5, [950] * 6 + [790] * 5, [50] * 6 + [90] * 5, 64, 2, 64, 4, "f32", None, 0),
    ([900], [0] * 7, [960] * 7, [40] * 7, 16, 1, 192, 4, "f16", None, 0),
    ([600], [0] * 5, [700] * 5, [30] * 5, 128, 1, 256, 4, "bf16", None, 300),
    ([900] * 70, list(range(70)), [940 + g for g in range(70)], [40] * 70, 32, 1, 32, 4, "bf16", None, 0),   # more groups than lanes, split
    ([200, 100], [0] * 3 + [1] * 2, [441, 440, 450, 340, 350], [240] * 5, 16, 64, 16, 64, "bf16", None, 0),  # more row tiles than pieces
    ([304], [0, 0, -1], [9000, 310, 5000], [1, 1, 1], 16, 1, 64, 2, "tile", None, 0),                        # long after the prefix
    ([100], [0, 0], [3200, 2100], [60, 50], 32, 1, 64, 4, "bf16", None, 0),                                  # and split there
    ([3000, 0, 10], [0, 1, 2], [3300, 2900, 400], [70, 60, 50], 64, 2, 128, 4, "f16", None, 500),
    ([40], [0] * 130, [41 + b % 7 for b in range(130)], [1] * 130, 16, 1, 16, 1, "f32", None, 0),            # more sequences than lanes
    ([33], [0] * 70, [34 + b % 5 if b % 3 else 0 for b in range(70)], [1 if b % 2 else 0 for b in range(70)], 16, 1, 32, 2, "f32", None, 7),
]


@pytest.mark.parametrize("hints", [True, False])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{len(c[1])}-{c[4:]}")
def test_shared(gpu, case, hints):
    share, of, lens, news, page, heads, hd, hq, kind, out, window = case
    t = Groups(41, share, of, lens, news, page, heads, hd, hints=hints, max_rows=None if hints else 0)
    group, scale = hq // heads, 1 / np.sqrt(hd)
    q, qv = _typed(t.s.rng.standard_normal((t.rows, hq, hd)) * 1.5, kind)
    _say(case[0], case[4:], hints)
    got = t.s.cache.attend(t.batch, q, shared=t.shared, window=window, dtype=_dt(out) if out else None)
    want, weight, big = t.want(qv, group, scale, window)
    res = out or ("f32" if kind == "tile" else kind)
    bound = _bound(want, weight, big, max(lens), hd, kind, res, t.rows * group)
    bad = np.abs(got.double().cpu().numpy() - want) - bound
    assert (bad <= 0).all(), (bad.max(), np.unravel_index(bad.argmax(), bad.shape))


def test_shared_tiles_out_in_place_and_other_rows(gpu):
    """Results as 16-bit tiles, on the queries, and rows behind the last
    sequence left alone."""
    import torch
    t = Groups(5, [70], [0, 0], [90, 71], [2, 1], 16, 2, 32)
    q, qv = _typed(t.s.rng.standard_normal((5, 4, 32)), "f32")
    want, weight, big = t.want(qv[:3], 2, 1 / np.sqrt(32), 0)
    bound = _bound(want, weight, big, 90, 32, "f32", "f32", 6)
    m = torch.full((5, 4, 32), 7, dtype=torch.int16, device="cuda")
    e = torch.full((5, 4, 2), 7, dtype=torch.int8, device="cuda")
    t.s.cache.attend(t.batch, q, shared=t.shared, out=(m, e))
    step = np.repeat(2.0 ** (e[:3].cpu().numpy().astype(float) - 15), 16, -1)
    got = m[:3].cpu().numpy() * step
    assert (np.abs(got - want) <= bound + step).all()      # at most one step: a rounding, cut at the ends
    assert (m[3:] == 7).all() and (e[3:] == 7).all()
    keep = q.clone()
    t.s.cache.attend(t.batch, q, shared=t.shared, out=q)
    assert (np.abs(q[:3].double().cpu().numpy() - want) <= bound).all() and torch.equal(q[3:], keep[3:])


@pytest.mark.parametrize("rows", [1, 30])
def test_shared_rows_do_not_see_other_bytes(gpu, rows):
    """NaN behind what is shared, behind a row's own position, and in own
    pages before the shared tokens' end; a NaN value that is seen shows."""
    share, lens = [50], [60 + rows, 52 + rows]
    t = Groups(6, share, [0, 0], lens, [rows, rows], 16, 2, 32)
    q, qv = _typed(t.s.rng.standard_normal((2 * rows, 4, 32)), "f32")
    want, weight, big = t.want(qv, 2, 1 / np.sqrt(32), 0)
    bound = _bound(want, weight, big, max(lens), 32, "f32", "f32", 4 * rows)
    c, s = t.s.cache, t.s
    group_page = int(s.table[0, 3])
    for x in (c.k_exp, c.v_exp):
        x[group_page, :, :, 2:] = 255                              # positions 50..63 of the group's pages
        for b in range(2):
            x[int(t.table[b, 3]), :, :, :2] = 254                  # positions 48, 49 of the sequences' own
            n = lens[b]
            if n % 16:
                x[int(t.table[b, n // 16]), :, :, n % 16:] = 255   # behind the end
    got = c.attend(t.batch, q, shared=t.shared).double().cpu().numpy()
    assert (np.abs(got - want) <= bound).all()
    c.v_exp[int(s.table[0, 0]), 1, 0, 5] = 255                     # position 5, shared: every row
    got = c.attend(t.batch, q, shared=t.shared).double().cpu().numpy()
    assert np.isnan(got[:, 2:, :16]).all() and np.isfinite(got[:, 2:, 16:]).all() and np.isfinite(got[:, :2]).all()


def test_shared_groups_that_hold_nonsense(gpu):
    """Lengths below 0 and past the table, sequences past the batch, pages that
    the cache does not have."""
    import torch
    from bfp.kv4 import Shared
    t = Groups(7, [48], [0, 0, 0], [60, 55, 50], [1, 2, 1], 16, 1, 32)
    q, qv = _typed(t.s.rng.standard_normal((4, 2, 32)), "f32")
    plain = t.s.table[1:]                                          # the sequences' own pages hold all of their tokens
    t.batch.pages.copy_(_int(plain))
    own = [(t.s.keys[1 + b], t.s.vals[1 + b]) for b in range(3)]
    big_int = 2 ** 31 - 1

    def check(shared, keys, vals, there):
        got = t.s.cache.attend(t.batch, q, shared=shared).double().cpu().numpy()
        want, weight, big = ref.attend_all(qv, keys, vals, t.start, t.lens, 2, 1 / np.sqrt(32), 0, there)
        assert (np.abs(got - want) <= _bound(want, weight, big, 60, 32, "f32", "f32", 8)).all()
    k, v = [x[0] for x in own], [x[1] for x in own]
    every = [np.ones(n, bool) for n in t.lens]
    pages = _int(t.s.table[:1])
    # a length below 0, or groups that lie outside the batch: nothing is shared
    check(Shared(pages, _int([0, 3]), _int([-5])), k, v, every)
    check(Shared(pages, _int([3, 9]), _int([48])), k, v, every)
    check(Shared(pages, _int([-9, -2]), _int([48])), k, v, every)
    # longer than its table: what it has no page for is not seen
    both = [np.concatenate([t.s.keys[0], np.zeros((16, 1, 32))])[:n] for n in t.lens]
    vals = [np.concatenate([t.s.vals[0], np.zeros((16, 1, 32))])[:n] for n in t.lens]
    seen = [np.arange(n) < 48 for n in t.lens]
    check(Shared(pages, _int([0, 3]), _int([big_int])), both, vals, seen)
    # pages that are not there
    bad = t.s.table[:1].copy()
    bad[0, 1] = 10 ** 6
    keys = [np.concatenate([t.s.keys[0][:48], x[48:]]) for x in k]
    vals = [np.concatenate([t.s.vals[0][:48], x[48:]]) for x in v]
    check(Shared(_int(bad), _int([-3, big_int]), _int([48])), keys, vals, [np.arange(n) // 16 != 1 for n in t.lens])


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("hd", [32, 128])
def test_rows_past_all_positions(gpu, new, hd):
    """Lengths near 2^31 with a window, so that a row's first key lies past
    every table: nothing is seen, and nothing past the cache is read."""
    import torch
    from bfp.kv4 import Shared
    t = Groups(8, [48], [0, 0, 0], [60 + new, 55 + new, 50 + new], [new] * 3, 16, 1, hd)
    q, _ = _typed(t.s.rng.standard_normal((3 * new, 2, hd)), "f32")
    for n in (2 ** 31 - 1, 2 ** 31 - 64, 0x7fff0000, 0x7fff0001):
        t.batch.lens.fill_(n)
        for window in (1, 63, 64):
            for shared in (None, t.shared, Shared(t.shared.pages, t.shared.start, _int([n]))):
                got = t.s.cache.attend(t.batch, q, shared=shared, window=window)
                assert (got == 0).all()
    torch.cuda.synchronize()


def test_shared_is_attend_where_tables_agree(gpu):
    """Forked sequences of a pool: the group's table is the parent's."""
    import torch
    from bfp.kv4 import Batch, Fp4Cache, Shared
    from bfp.pages import PagePool
    cache = Fp4Cache(60, 16, 2, 64)
    pool = PagePool(cache)
    table, lens = torch.full((4, 20), -1, dtype=torch.int32, device="cuda"), _int([150, 0, 0, 0])
    prompt = Batch(table, _int([0, 150, 150, 150, 150]), lens, max_q=150)
    pool.reserve(prompt)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    rand = lambda n, h: torch.randn(n, h, 64, generator=g, device="cuda")  # noqa: E731
    cache.append(prompt, rand(150, 2), rand(150, 2))
    pool.fork(table[:1], lens[:1], _int([0, 0, 0]), out=(table[1:], lens[1:]))
    batch = Batch(table, _int([0, 1, 2, 3, 4]), lens, max_q=1)
    shared = Shared(table[:1], _int([0, 4]), _int([150]))
    for _ in range(3):
        batch.lens += 1
        pool.reserve(batch)
        cache.append(batch, rand(4, 2), rand(4, 2))
        q = rand(4, 6)
        a, b = cache.attend(batch, q), cache.attend(batch, q, shared=shared)
        keys, vals = cache.read(Batch(table, _int([0] + [int(x) for x in batch.lens.cumsum(0)]), batch.lens, max_q=200), int(batch.lens.sum()))
        ends = np.concatenate([[0], np.cumsum(batch.lens.cpu().numpy())])
        k, v = ([x[ends[b]:ends[b + 1]].double().cpu().numpy() for b in range(4)] for x in (keys, vals))
        want, weight, big = ref.attend_all(q.double().cpu().numpy(), k, v, np.arange(5), batch.lens.cpu().numpy(), 3, 1 / 8, 0)
        for got in (a, b):
            assert (np.abs(got.double().cpu().numpy() - want) <= _bound(want, weight, big, 153, 64, "f32", "f32", 12)).all()


@pytest.mark.parametrize("new", [1, 40])
def test_captured_shared(gpu, new):
    """Captured once, replayed while lengths, groups and queries change; the
    other stream's call has scratch of its own."""
    import torch
    t = Groups(9, [300, 200], [0, 0, 0, 1, 1], [340, 350, 344, 260, 244], [new] * 5, 16, 2, 64, max_rows=0)
    q = torch.randn(t.rows, 8, 64, device="cuda", dtype=torch.bfloat16)
    out = torch.empty_like(q)
    work = torch.empty(t.s.cache.attend_work(t.batch, q, shared=t.shared), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            t.s.cache.attend(t.batch, q, shared=t.shared, out=out, work=work)
    torch.cuda.synchronize()
    for i in range(5):
        q.copy_(torch.randn(t.rows, 8, 64, device="cuda"))
        t.shared.lens.copy_(_int([300 - 20 * i, 200 - 50 * i]))
        t.shared.start.copy_(_int([0, 3 - i % 2, 5]))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            want = t.s.cache.attend(t.batch, q, shared=t.shared)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_refusals_of_the_python_side(gpu):
    import torch
    from bfp.kv4 import Shared
    t = Groups(1, [20], [0], [30], [1], 16, 2, 32)
    pages, start, lens = t.shared.pages, t.shared.start, t.shared.lens
    for a in ((pages[0], start, lens), (pages.long(), start, lens), (pages, start[:1], lens), (pages, start, lens.cpu()),
              (pages[:, :0], start, lens), (pages[:0], start[:1], lens[:0])):
        with pytest.raises(ValueError):
            Shared(*a)
    with pytest.raises(ValueError):
        Shared(pages, start, lens, max_rows=-1)
    q = torch.randn(1, 4, 32, device="cuda")
    with pytest.raises(ValueError):
        t.s.cache.attend(t.batch, q, shared=t.shared, picks=torch.zeros(1, 2, 1, dtype=torch.int32, device="cuda"))
    with pytest.raises(Exception, match="scratch"):
        t.s.cache.attend(t.batch, q, shared=t.shared, work=torch.empty(1, device="cuda"))
    with pytest.raises(AttributeError):
        t.shared.lens = lens.clone()
