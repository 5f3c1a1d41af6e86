"""The page pool where pages run out, and tables that a compaction finds out
of date."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_pages import Both, _batch, _int

pytestmark = pytest.mark.gpu


def test_branches_without_a_page_end_before_it(gpu):
    """A branch whose last page could not be copied goes on from its whole
    pages: a page that it is given later holds its own tokens alone."""
    import torch
    from bfp.kv4 import Batch, Fp4Cache
    from bfp.pages import PagePool
    cache = Fp4Cache(6, 16, 1, 32)
    pool = PagePool(cache)
    table, lens = torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), _int([40, 20])
    prompt = Batch(table, _int([0, 40, 60]), lens, max_q=40)
    pool.reserve(prompt)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    rand = lambda n, h: torch.randn(n, h, 32, generator=g, device="cuda")  # noqa: E731
    k, v = rand(60, 1), rand(60, 1)
    cache.append(prompt, k, v)
    got, got_lens = pool.fork(table, lens, _int([0, 0, 1, 0]))        # one page is left: the first branch's
    assert got.cpu().tolist() == [[0, 1, 5, -1], [0, 1, -1, -1], [3, -1, -1, -1], [0, 1, -1, -1]]
    assert got_lens.cpu().tolist() == [40, 32, 16, 32] and int(pool.short) == 3
    print("[pages] goes on", flush=True)
    pool.free(got[0:1])
    pool.free(got[2:])
    pool.free(table[1:2])                                             # pages 3, 4 and 5, full of other tokens
    one = Batch(got[1:2], _int([0, 1]), got_lens[1:2], max_q=1)
    one.lens += 1
    pool.reserve(one)
    assert got[1].cpu().tolist() == [0, 1, 3, -1] and pool.refs.cpu().tolist() == [2, 2, 1, 1, 0, 0]
    new_k, new_v, q = rand(1, 1), rand(1, 1), rand(1, 2)
    cache.append(one, new_k, new_v)
    out = cache.attend(one, q)
    keys = torch.cat([k[:32], new_k]).cpu().numpy()
    vals = torch.cat([v[:32], new_v]).cpu().numpy()
    want, weight, big = ref.attend_all(q.double().cpu().numpy(), [ref.quant4(keys)], [ref.quant4(vals)], [0, 1], [33], 2, 1 / np.sqrt(32))
    assert (np.abs(out.double().cpu().numpy() - want) <= ref.attend_bound(want, weight, big, 33, 32, 2.0 ** -24, 2.0 ** -24)).all()


def test_lengths_of_branches_that_lose_nothing(gpu):
    """Whole pages, a parent that has no page where it ends, and a table too
    narrow for the page: the length is the parent's."""
    b = Both(4, 16, layers=1)
    table = np.array([[0, 1, -1], [2, -1, -1], [3, 9, -1]])
    b.ref.refs[:] = 1
    b.pool.refs.copy_(_int(b.ref.refs))
    lens = [32, 16, 25]
    for width in (1, 3):
        out = (_int(np.full((3, width), 7)), _int([0] * 3))
        _, got = b.pool.fork(_int(table), _int(lens), _int([0, 1, 2]), out=out)
        b.ref.fork(table, lens, [0, 1, 2], width)
        assert got.cpu().tolist() == lens
    b.check()


@pytest.mark.parametrize("n_pages", [40, 5000])
def test_compaction_clears_entries_of_free_pages(gpu, n_pages):
    """A table whose pages were given up through another one names pages that
    a compaction fills with others' tokens: its entries become -1, below the
    held pages' number and above it."""
    import torch
    b = Both(n_pages, 16, heads=1, hd=16, layers=1)
    rng = np.random.default_rng(n_pages)
    held = rng.permutation(n_pages)[:n_pages // 2]
    b.ref.refs[held] = 1
    b.pool.refs.copy_(_int(b.ref.refs))
    stale = np.array([[p for p in range(n_pages) if b.ref.refs[p] == 0]])
    table = held[None].copy()
    odd = np.array([[-1, -7, n_pages, 2 ** 31 - 1, -2 ** 31]])
    dev = [_int(table), _int(stale), _int(odd)]
    live = b.pool.compact(*dev)
    assert int(live) == b.ref.compact(table)
    assert (dev[0].cpu().numpy() == table).all()
    assert (dev[1] == -1).all() and (dev[2].cpu().numpy() == odd).all()
    b.check()
