"""The page pool against a plain one, call after call: numbers, counts and
every byte of every page."""
import numpy as np
import pytest

import pages_ref

pytestmark = pytest.mark.gpu


def _int(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).cuda()


class Both:
    """A pool on the device and the plain one.  Page p's bytes are all
    derived from a number, so a copied page can be told."""

    def __init__(self, n_pages, page, heads=2, hd=32, layers=2, refs=None):
        import torch
        from bfp.kv4 import Fp4Cache
        from bfp.pages import PagePool
        self.caches = [Fp4Cache(n_pages, page, heads, hd) for _ in range(layers)]
        self.tensors = [t for c in self.caches for t in (c.k, c.k_exp, c.v, c.v_exp)]
        ids = torch.arange(n_pages, device="cuda")
        for i, t in enumerate(self.tensors):
            each = torch.arange(t[0].numel(), device="cuda")
            t.copy_(((ids[:, None] * 37 + each * 11 + i * 101 + (ids[:, None] >> 8)) % 251).to(torch.uint8).view(t.shape))
        self.first = [t.clone() for t in self.tensors]
        self.pool, self.ref = PagePool(self.caches, refs=refs), pages_ref.Pool(n_pages, page)

    def check(self):
        assert (self.pool.refs.cpu().numpy() == self.ref.refs).all()
        assert int(self.pool.short) == self.ref.short
        idx = _int(self.ref.content).long()
        for t, f in zip(self.tensors, self.first):
            assert (t == f[idx]).all()


def _batch(table, news, lens):
    from bfp.kv4 import Batch
    start = np.concatenate([[0], np.cumsum(news)])
    return Batch(_int(table), _int(start), _int(lens), max_q=max(max(news), 0)), start


def test_life_of_sequences(gpu):
    """Prompts, steps, branches at whole pages and inside them, ends, a
    compaction, and more steps."""
    b = Both(40, 16)
    table = np.full((3, 8), -1)
    lens = np.array([37, 16, 0])
    batch, start = _batch(table, [37, 16, 0], lens)
    print("[pages] prompts", flush=True)
    b.pool.reserve(batch)
    b.ref.reserve(table, start, lens)
    assert (batch.pages.cpu().numpy() == table).all()
    b.check()
    for step in range(20):
        lens = lens + 1
        one, start = _batch(table, [1, 1, 1], lens)
        b.pool.reserve(one)
        b.ref.reserve(table, start, lens)
        assert (one.pages.cpu().numpy() == table).all()
    b.check()
    print("[pages] branches", flush=True)
    parents = [0, 0, 2, 1, 0, 5, -1]
    got, got_lens = b.pool.fork(_int(table), _int(lens), _int(parents))
    want, want_lens = b.ref.fork(table, lens, parents)
    assert (got.cpu().numpy() == want).all() and (got_lens.cpu().numpy() == want_lens).all()
    b.check()
    print("[pages] ends", flush=True)
    dev = _int(table)
    b.pool.free(dev[0:2])
    b.ref.free(table[0:2])
    assert (dev.cpu().numpy() == table).all()
    b.check()
    live = b.pool.compact(dev, got)
    assert int(live) == b.ref.compact(table, want)
    assert (dev.cpu().numpy() == table).all() and (got.cpu().numpy() == want).all()
    b.check()
    assert (b.ref.refs[:int(live)] > 0).all() and (b.ref.refs[int(live):] == 0).all()
    print("[pages] after", flush=True)
    lens = want_lens + 3
    batch, start = _batch(want, [3] * 7, lens)
    b.pool.reserve(batch)
    b.ref.reserve(want, start, lens)
    assert (batch.pages.cpu().numpy() == want).all()
    b.check()


def test_too_few_pages(gpu):
    """What is not there is counted; who asked first has it."""
    b = Both(5, 32, layers=1)
    table, lens = np.full((3, 4), -1), np.array([64, 40, 128])
    batch, start = _batch(table, [64, 40, 128], lens)
    b.pool.reserve(batch)
    b.ref.reserve(table, start, lens)
    assert (batch.pages.cpu().numpy() == table).all() and b.ref.short == 3
    b.check()
    got, _ = b.pool.fork(_int(table), _int(lens), _int([1, 0, 1]))
    want, _ = b.ref.fork(table, lens, [1, 0, 1])
    assert (got.cpu().numpy() == want).all() and b.ref.short == 5
    b.check()


def test_tables_that_hold_nonsense(gpu):
    """Pages outside the pool, lengths below 0 and past the table, rows that
    end inside: bounded, and nothing else is touched."""
    b = Both(12, 16, layers=1)
    big = 2 ** 31 - 1
    table = np.array([[big, -7, 3, 12], [4, 5, 6, -1], [7, 8, 9, 10]])
    b.ref.refs[[3, 4, 5, 6, 7, 8, 9, 10]] = 1
    b.pool.refs.copy_(_int(b.ref.refs))
    lens = np.array([60, -5, big])
    got, got_lens = b.pool.fork(_int(table), _int(lens), _int([0, 1, 2, big, -big]))
    want, want_lens = b.ref.fork(table, lens, [0, 1, 2, big, -big])
    assert (got.cpu().numpy() == want).all() and (got_lens.cpu().numpy() == want_lens).all()
    b.check()
    dev = _int(table)
    b.pool.free(dev)
    b.ref.free(table)
    assert (dev.cpu().numpy() == table).all()
    b.check()
    b.pool.free(_int([[0, 1, 2, 2]]))     # nobody holds them any more: never below 0
    b.check()
    # a batch whose rows are more than its tokens, or past its table
    table = np.full((3, 2), -1)
    batch, start = _batch(table, [9, 3, 40], [5, 50, 32])
    b.pool.reserve(batch)
    b.ref.reserve(table, start, [5, 50, 32])
    assert (batch.pages.cpu().numpy() == table).all()
    b.check()


@pytest.mark.parametrize("n_pages,share", [(1, 1.0), (1, 0.0), (3, 0.5), (4095, 0.3), (4096, 0.99), (4097, 0.01), (70001, 0.6), (70001, 0.0)])
def test_compact_sizes(gpu, n_pages, share):
    b = Both(n_pages, 16, heads=1, hd=16, layers=1)
    rng = np.random.default_rng(n_pages)
    live = rng.permutation(n_pages)[:int(n_pages * share)]
    table = np.full((2, max(len(live), 1)), -1)
    table[0, :len(live)] = live
    table[1, :len(live) // 2] = live[:len(live) // 2]
    np.add.at(b.ref.refs, table[table >= 0], 1)
    b.pool.refs.copy_(_int(b.ref.refs))
    dev = _int(table)
    print("[pages] compact", n_pages, share, flush=True)
    got = b.pool.compact(dev)
    assert int(got) == b.ref.compact(table) == len(live)
    assert (dev.cpu().numpy() == table).all()
    b.check()


@pytest.mark.parametrize("n_pages,free,want", [(70001, 3, 3), (70001, 40000, 5000), (16384, 1, 4), (4097, 4097, 4000)])
def test_lowest_pages_of_a_large_pool(gpu, n_pages, free, want):
    """Free pages far apart, in any round of the search."""
    b = Both(n_pages, 16, heads=1, hd=16, layers=1)
    rng = np.random.default_rng(free)
    b.ref.refs[:] = 1
    gaps = np.sort(rng.permutation(n_pages)[:free])
    b.ref.refs[gaps] = 0
    b.pool.refs.copy_(_int(b.ref.refs))
    lens = [16 * (want - want // 2) - 3, 16 * (want // 2)]
    table = np.full((2, want), -1)
    batch, _ = _batch(table, lens, lens)
    b.pool.reserve(batch)
    flat = batch.pages.cpu().numpy()
    given = np.concatenate([flat[0, :want - want // 2], flat[1, :want // 2]])
    most = min(free, want)
    assert (given[:most] == gaps[:most]).all() and (given[most:] == -1).all()
    assert int(b.pool.short) == want - most


def test_many_sequences_and_children(gpu):
    """More entries and children than the workgroup has threads."""
    b = Both(9000, 16, heads=1, hd=16, layers=1)
    rng = np.random.default_rng(3)
    lens = rng.integers(1, 60, 2500)
    news = np.minimum(lens, rng.integers(1, 40, 2500))
    table = np.full((2500, 4), -1)
    batch, start = _batch(table, list(news), lens)
    b.pool.reserve(batch)
    # the plain one, by counting up: all pages are free
    at = 0
    for i in range(2500):
        for p in range((lens[i] - news[i]) // 16, (lens[i] - 1) // 16 + 1):
            table[i, p] = at
            at += 1
    b.ref.refs[:at] = 1
    assert (batch.pages.cpu().numpy() == table).all()
    b.check()
    parents = rng.integers(0, 2500, 1700)
    got, got_lens = b.pool.fork(batch.pages, batch.lens, _int(parents))
    whole = (lens[parents] // 16)[:, None] > np.arange(4)
    want = np.where(whole, table[parents], -1)
    np.add.at(b.ref.refs, want[want >= 0], 1)
    for i, j in enumerate(parents):
        p = lens[j] // 16
        if lens[j] % 16 and table[j, p] >= 0:
            want[i, p] = at
            b.ref.refs[at], b.ref.content[at] = 1, table[j, p]
            at += 1
    assert (got.cpu().numpy() == want).all() and (got_lens.cpu().numpy() == lens[parents]).all()
    b.check()


def test_more_arrays_than_one_launch_takes(gpu):
    b = Both(6, 16, heads=1, hd=16, layers=70)          # 280 arrays
    b.pool.copy(_int([0, 5, 9, 2, -1]), _int([1, 3, 4, 6, 2]))
    b.ref.content[[1, 3]] = [0, 5]
    b.check()
    table = np.array([[2, 5, -1]])
    b.ref.refs[[2, 5]] = 1
    b.pool.refs.copy_(_int(b.ref.refs))
    got, _ = b.pool.fork(_int(table), _int([20]), _int([0]))
    want, _ = b.ref.fork(table, [20], [0])
    assert (got.cpu().numpy() == want).all()
    b.check()
    dev = _int(np.concatenate([table, want]))
    tables = np.concatenate([table, want])
    assert int(b.pool.compact(dev)) == b.ref.compact(tables)
    assert (dev.cpu().numpy() == tables).all()
    b.check()


def test_narrower_tables_and_given_results(gpu):
    import torch
    b = Both(20, 16, layers=1)
    table = np.array([[4, 5, 6, 7], [1, 2, -1, -1]])
    b.ref.refs[[4, 5, 6, 7, 1, 2]] = 1
    b.pool.refs.copy_(_int(b.ref.refs))
    for width in (2, 3, 6):
        out = (torch.full((2, width), 77, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))
        got, got_lens = b.pool.fork(_int(table), _int([41, 17]), _int([0, 1]), out=out)
        want, want_lens = b.ref.fork(table, [41, 17], [0, 1], width)
        assert got is out[0] and (got.cpu().numpy() == want).all() and (got_lens.cpu().numpy() == want_lens).all()
        b.check()


def test_captured_steps(gpu):
    """A decode step's reserve and a fork, captured once and replayed while the
    program writes lengths and parents."""
    import torch
    b = Both(64, 16, layers=2)
    table = np.full((4, 6), -1)
    lens = np.array([5, 20, 0, 31])
    batch, start = _batch(table, [1, 1, 1, 1], lens)
    kids, kid_lens, parents = _int(np.full((3, 6), -1)), _int([0] * 3), _int([0, 0, 0])
    work = torch.empty(b.pool.work(3), dtype=torch.uint8, device="cuda")

    def step():
        b.pool.reserve(batch, work=work)
        b.pool.free(kids)
        b.pool.fork(batch.pages, batch.lens, parents, out=(kids, kid_lens), work=work)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    rkids = np.full((3, 6), -1)
    for i in range(6):
        lens = lens + 1
        par = [i % 4, 3, (i * 3) % 5]
        batch.lens.copy_(_int(lens))
        parents.copy_(_int(par))
        graph.replay()
        b.ref.reserve(table, start, lens)
        b.ref.free(rkids)
        rkids, rlens = b.ref.fork(table, lens, par)
        assert (batch.pages.cpu().numpy() == table).all()
        assert (kids.cpu().numpy() == rkids).all() and (kid_lens.cpu().numpy() == rlens).all()
        b.check()


def test_refusals_of_the_python_side(gpu):
    import torch
    from bfp.kv4 import Fp4Cache
    from bfp.pages import PagePool
    c = Fp4Cache(8, 16, 1, 16)
    pool = PagePool(c)
    t = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for bad in (t.cpu(), t.long(), t.t(), t[:, :2], t[0]):
        for call in (pool.free, pool.compact, lambda x: pool.fork(x, t[0, :2], t[1])):
            with pytest.raises(ValueError):
                call(bad)
    with pytest.raises(ValueError):
        PagePool([c, Fp4Cache(9, 16, 1, 16)])
    with pytest.raises(ValueError):
        PagePool([])
    with pytest.raises(ValueError):
        PagePool(c, refs=torch.zeros(7, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        pool.copy(t[0], t[1, :2])
    with pytest.raises(ValueError):
        pool.fork(t, _int([1, 1]), _int([0, 1]), out=(_int([[0, 0, 0]]), _int([0])))
    with pytest.raises(AttributeError):
        pool.refs = t
