"""The attention over the 4-bit cache where contexts are long or rows are
many: keys shared between workgroups and joined, prompts whole and in
pieces, in every width and precision, against plain 64-bit numpy."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import HALF, _dt, _int, _say, _terms_error, _typed

pytestmark = pytest.mark.gpu


class Long:
    """Sequences whose cached values are random bytes: elements of every
    kind, exponents within a few powers of two; pages dealt out of order,
    noise where no token is."""

    def __init__(self, seed, lens, news, page, heads, hd, max_len=None, more_width=1):
        import torch
        from bfp.kv4 import Batch, Fp4Cache
        self.rng = rng = np.random.default_rng(seed)
        self.lens, self.news, self.page, self.heads, self.hd = list(lens), list(news), page, heads, hd
        need = [-(-max(n, 0) // page) for n in lens]
        n_pages = sum(need) + 3
        ids = rng.permutation(n_pages).astype(np.int32)
        self.table = np.full((len(lens), max(max(need), 1) + more_width), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.rows = int(self.start[-1])
        shape = (n_pages, heads, hd // 16, page)
        self.bytes = {k: rng.integers(0, 256, shape + ((8,) if k in "kv" else ()), dtype=np.uint8) for k in ("k", "ke", "v", "ve")}
        for b, n in enumerate(lens):
            for name, lo in (("ke", 123), ("ve", 122)):
                pages, at = self.where(b)
                self.bytes[name][pages, :, :, at] = rng.integers(lo, lo + 4, (max(n, 0), heads, hd // 16))
        self.read_back()
        self.cache = Fp4Cache.from_buffers(*(torch.from_numpy(self.bytes[k]).cuda() for k in ("k", "ke", "v", "ve")))
        self.batch = Batch(_int(self.table), _int(self.start), _int(self.lens), max_q=max(max(news), 0),
                           max_len=max(max(lens), 0) if max_len is None else max_len)

    def where(self, b):
        p = np.arange(max(self.lens[b], 0))
        return self.table[b, p // self.page], p % self.page

    def read_back(self):
        self.keys, self.vals = [], []
        for b in range(len(self.lens)):
            pages, at = self.where(b)
            for name, to in (("k", self.keys), ("v", self.vals)):
                x = self.bytes[name][pages, :, :, at]            # token, head, tile, 8
                codes = np.stack([x & 15, x >> 4], -1).reshape(len(at), self.heads, self.hd)
                to.append(ref.value(codes, self.bytes[name + "e"][pages, :, :, at]))

    def query(self, heads, kind, size=1.0):
        return _typed(self.rng.standard_normal((self.rows, heads, self.hd)) * size, kind)


def check(s, qv, kind, out_kind, got, window=0, there=None):
    hq = qv.shape[1]
    want, weight, big = ref.attend_all(qv, s.keys, s.vals, s.start, s.lens, hq // s.heads, s.hd ** -0.5, window, there)
    bound = ref.attend_bound(want, weight, big, max(max(s.lens), 1), s.hd, HALF[out_kind], _terms_error(kind, out_kind, 1 << 20))
    g = got.double().cpu().numpy()
    assert np.isfinite(g).all()
    err = np.abs(g - want)
    assert (err <= bound).all(), (err.max(), (err / bound).max())
    return g


LONG = [  # lens, news, page, heads, hd, group, type, out type, window
    ([9000, 1, 0, 4500], [1, 1, 0, 1], 16, 3, 64, 3, "bf16", "bf16", 0),
    ([9000, 100], [1, 1], 64, 1, 64, 16, "bf16", "bf16", 0),
    ([5000, 6001], [2, 1], 256, 2, 48, 5, "f32", "f32", 0),
    ([5000, 0, 6001, 64], [1, 0, 3, 1], 32, 1, 32, 2, "tile", "bf16", 0),
    ([4097], [1], 16, 1, 16, 1, "f32", "f32", 0),
    ([20000], [1], 16, 1, 16, 1, "f32", "f32", 0),                 # many parts of one row
    ([60000, 5], [1, 1], 256, 1, 16, 1, "f16", "f16", 0),          # and pieces as long as it takes
    ([30000, 29999], [1, 1], 64, 1, 64, 2, "f16", "f32", 5000),    # window
    ([9000, 700, 5000], [3, 700, 2], 64, 1, 64, 1, "bf16", "bf16", 4500),
    ([3000, 7, 2500], [1, 1, 1], 16, 2, 128, 16, "bf16", "bf16", 0),
    ([3000, 7, 2500], [1, 1, 1], 32, 2, 128, 4, "f16", "f16", 0),
    ([2113, 4000], [1, 2], 128, 1, 112, 4, "f32", "f32", 0),
    ([2600, 2600, 2600], [1, 5, 1], 16, 2, 80, 3, "tile", "f16", 2200),
    ([1100, 3000], [1, 1], 16, 1, 192, 12, "bf16", "bf16", 0),
    ([300, 100], [1, 1], 16, 2, 192, 9, "bf16", "bf16", 0),
    ([1100, 3000], [1, 1], 16, 1, 144, 3, "f16", "f32", 0),
    ([1100, 2000], [1, 1], 16, 3, 160, 2, "bf16", "bf16", 0),
    ([1900, 64], [1, 1], 64, 2, 256, 9, "bf16", "bf16", 0),
    ([1900, 1500], [1, 1], 64, 1, 256, 3, "f32", "f32", 0),
    ([1900, 1500], [1, 1], 64, 1, 208, 4, "f16", "f16", 1200),
]


@pytest.mark.parametrize("case", LONG, ids=str)
def test_long_contexts(gpu, case):
    lens, news, page, heads, hd, group, kind, out_kind, window = case
    s = Long(61, lens, news, page, heads, hd)
    q, qv = s.query(heads * group, kind)
    _say(case)
    check(s, qv, kind, out_kind, s.cache.attend(s.batch, q, window=window, dtype=_dt(out_kind)), window)


PROMPTS = [  # lens, news, page, heads, hd, group, type, out type, window
    ([2000], [1500], 16, 2, 32, 4, "bf16", "bf16", 0),
    ([700, 41], [700, 41], 16, 2, 32, 3, "f16", "f16", 0),
    ([1500], [1200], 16, 2, 32, 4, "f16", "f16", 0),
    ([600, 0, 333], [600, 0, 200], 32, 2, 16, 4, "f32", "f32", 0),
    ([2000, 900], [1500, 900], 64, 2, 64, 4, "bf16", "bf16", 0),
    ([1000, 3], [700, 3], 16, 3, 48, 2, "tile", "bf16", 0),
    ([900, 901], [900, 5], 16, 3, 64, 3, "f32", "f32", 0),
    ([900, 901], [900, 600], 16, 2, 64, 3, "f32", "f32", 100),
    ([1500, 800], [1500, 800], 256, 3, 96, 4, "bf16", "bf16", 0),
    ([700], [700], 16, 2, 96, 4, "f16", "f16", 0),
    ([1500, 40], [1200, 40], 16, 2, 96, 4, "tile", "f16", 0),
    ([700, 64], [500, 64], 128, 2, 80, 3, "f32", "bf16", 0),
    ([2000, 1200], [1500, 1200], 64, 3, 128, 4, "bf16", "bf16", 0),
    ([1000, 1200], [1000, 1000], 64, 1, 128, 8, "f16", "f16", 333),
    ([900], [800], 16, 2, 112, 3, "f32", "f32", 0),
    ([1500, 1300], [1500, 1300], 64, 3, 192, 4, "bf16", "bf16", 0),
    ([900], [800], 64, 2, 160, 4, "f16", "f16", 0),
    ([700], [700], 16, 2, 176, 2, "f32", "f32", 0),
    ([1500, 1300], [1500, 1300], 64, 3, 256, 4, "bf16", "bf16", 0),
    ([900], [800], 64, 2, 208, 4, "f16", "f16", 0),
    ([700], [700], 16, 2, 256, 2, "f32", "f32", 0),
    ([4000], [64], 64, 4, 128, 4, "bf16", "bf16", 0),               # keys in pieces
    ([6000, 500], [64, 30], 64, 1, 64, 4, "f32", "f32", 0),
]


@pytest.mark.parametrize("case", PROMPTS, ids=str)
def test_prompts(gpu, case):
    lens, news, page, heads, hd, group, kind, out_kind, window = case
    s = Long(67, lens, news, page, heads, hd)
    q, qv = s.query(heads * group, kind)
    _say(case)
    check(s, qv, kind, out_kind, s.cache.attend(s.batch, q, window=window, dtype=_dt(out_kind)), window)


@pytest.mark.parametrize("hd,news,kind", [(64, [1, 1], "bf16"), (128, [1, 1], "f32"), (64, [700, 3], "f32"), (64, [4, 2], "f16")])
def test_lengths_past_what_the_batch_says(gpu, hd, news, kind):
    """max_len is a hint: longer sequences are attended to all the same."""
    from bfp.kv4 import Batch
    s = Long(71, [9000, 4300], news, 64, 1, hd)
    q, qv = s.query(3, kind)
    for said in (1, 100, 5000, 0, 1 << 20):
        b = Batch(s.batch.pages, s.batch.start, s.batch.lens, max_q=max(news), max_len=said)
        check(s, qv, kind, "f32", s.cache.attend(b, q, dtype=_dt("f32")))


@pytest.mark.parametrize("hd,window", [(64, 0), (64, 100), (128, 0), (256, 0)])
def test_more_sequences_than_share_their_keys(gpu, hd, window):
    """Batches of hundreds, their table wide enough for long contexts."""
    rng = np.random.default_rng(73)
    lens = [int(n) for n in rng.integers(0, 70, 300)]
    lens[7], lens[299] = 5000, 1111
    s = Long(73, lens, [min(n, 1) for n in lens], 256, 1, hd, max_len=0)
    q, qv = s.query(2, "bf16")
    check(s, qv, "bf16", "bf16", s.cache.attend(s.batch, q, window=window), window)


@pytest.mark.parametrize("news,hd", [([1, 1], 64), ([600, 2], 64), ([300, 200], 128), ([1, 1], 256)])
@pytest.mark.parametrize("window", [0, 2500])
def test_pages_that_do_not_exist(gpu, news, hd, window):
    from bfp.kv4 import Batch
    s = Long(79, [6000, 3000], news, 64, 1, hd)
    bad = s.table.copy()
    bad[0, 2], bad[0, 40:80], bad[1, :] = -1, 10 ** 6, -7
    ok = bad[0] != s.table[0]
    there = [~ok[np.arange(6000) // 64], np.zeros(3000, bool)]
    batch = Batch(_int(bad), s.batch.start, s.batch.lens, max_q=max(news), max_len=6000)
    q, qv = s.query(4, "f32")
    got = check(s, qv, "f32", "f32", s.cache.attend(batch, q, window=window), window, there)
    assert (got[news[0]:] == 0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("news,window,hd", [([1], 0, 64), ([3], 4200, 64), ([800], 0, 64), ([800], 300, 64), ([500], 0, 128), ([1], 0, 256)])
def test_nan_stays_with_those_who_see_it(gpu, kind, news, window, hd):
    s = Long(83, [5001], news, 16, 1, hd)
    q, qv = s.query(8 if news[0] > 3 else 3, kind)
    clean = check(s, qv, kind, kind, s.cache.attend(s.batch, q, window=window), window)
    pos = np.arange(5001 - news[0], 5001)
    for p, tile in ((5000, 1), (4999, 0), (4607, 3), (803, 3), (3, 2)):
        where = (int(s.table[0, p // 16]), 0, tile, p % 16)
        sees = (pos >= p) & ((pos - window < p) if window else True)
        for exps, dims in ((s.cache.v_exp, slice(16 * tile, 16 * tile + 16)), (s.cache.k_exp, slice(0, hd))):
            old = int(exps[where])
            exps[where] = 255
            got = s.cache.attend(s.batch, q, window=window).double().cpu().numpy()
            exps[where] = old
            nan = np.zeros(got.shape, bool)
            nan[sees, :, dims] = True
            assert (np.isnan(got) == nan).all(), (p, tile)
            assert (got[~nan] == clean[~nan]).all()


@pytest.mark.parametrize("lens,news,hd", [([40, 7], [1, 1], 64), ([5000, 7], [2, 1], 64), ([300, 7], [1, 1], 256), ([900, 7], [600, 7], 64)])
@pytest.mark.parametrize("kind,group", [("f32", 2), ("f16", 2), ("bf16", 2), ("bf16", 12)])
def test_queries_that_are_not_finite(gpu, lens, news, hd, kind, group):
    """An infinite or NaN query makes its own row NaN, also where all of its
    products have one sign, and no other row."""
    import torch
    s = Long(89, lens, news, 16, 1, hd)
    # keys whose value 3 of the head is never zero and always positive
    for b in range(len(lens)):
        pages, at = s.where(b)
        x = s.bytes["k"][pages, :, 0, at]
        x[..., 1] = (x[..., 1] & 0x0f) | 0x20
        s.bytes["k"][pages, :, 0, at] = x
    s.read_back()
    s.cache.k.copy_(torch.from_numpy(s.bytes["k"]))
    q, qv = s.query(group, kind)
    clean = check(s, qv, kind, kind, s.cache.attend(s.batch, q))
    n = s.rows
    for value, row in ((float("inf"), 0), (float("-inf"), n - 1), (float("nan"), n // 2)):
        q2 = q.clone()
        q2[row, 1, 3] = value
        got = s.cache.attend(s.batch, q2).double().cpu().numpy()
        nan = np.zeros(got.shape, bool)
        nan[row, 1] = True
        assert (np.isnan(got) == nan).all(), (value, row)
        assert (got[~nan] == clean[~nan]).all()


@pytest.mark.parametrize("lens,news,hd,kind", [([9000, 4100], [1, 1], 64, "f32"), ([3000], [2], 128, "bf16"),
                                               ([900], [700], 64, "f32"), ([5000], [64], 128, "f16")])
def test_where_results_go(gpu, lens, news, hd, kind):
    """Strided, unaligned and in-place results, tiles out, rows outside."""
    import torch
    from bfp import _dev
    from bfp._lib import call
    from bfp.kv4 import Batch
    s = Long(97, lens, news, 64, 2, hd)
    q, qv = s.query(6, kind)
    n = s.rows
    want = s.cache.attend(s.batch, q)
    check(s, qv, kind, kind, want)
    odd = torch.empty(n * 6 * (hd + 1) + 1, device="cuda", dtype=q.dtype)[1:].view(n, 6, hd + 1)[:, :, :hd]
    assert torch.equal(s.cache.attend(s.batch, q, out=odd), want)
    joined = torch.full((n, 9, hd), 3.0, device="cuda", dtype=q.dtype)
    joined[:, 1:7] = q
    s.cache.attend(s.batch, joined[:, 1:7], out=joined[:, 1:7])      # in place
    assert torch.equal(joined[:, 1:7], want) and (joined[:, 0] == 3).all() and (joined[:, 7:] == 3).all()
    full = s.cache.attend(s.batch, q, dtype=torch.float32)
    m = torch.empty(n, 6, hd, dtype=torch.int16, device="cuda")
    e = torch.empty(n, 6, hd // 16, dtype=torch.int8, device="cuda")
    s.cache.attend(s.batch, q, out=(m, e))
    wm, we = torch.empty_like(m), torch.empty_like(e)
    call("bfp_tile_quantize_f32_d", full.data_ptr(), full.numel(), wm.data_ptr(), we.data_ptr(), _dev.stream())
    assert torch.equal(m, wm) and torch.equal(e, we)
    # rows before, between and after the sequences keep what they hold
    start = _int(s.start + 2)
    shifted = Batch(s.batch.pages, start, s.batch.lens, max_q=max(news), max_len=max(lens))
    q2 = torch.zeros(n + 5, 6, hd, device="cuda", dtype=q.dtype)
    q2[2:n + 2] = q
    out = torch.full_like(q2, 9.0)
    s.cache.attend(shifted, q2, out=out)
    assert torch.equal(out[2:n + 2], want) and (out[:2] == 9).all() and (out[n + 2:] == 9).all()


def test_as_many_sequences_as_a_batch_has(gpu):
    """65535 sequences of one token, more heads than workgroups of many waves
    could take in one launch: each gets its own value back."""
    import torch
    from bfp.kv4 import Batch, Fp4Cache
    n, heads = 65535, 65
    cache = Fp4Cache(n, 16, heads, 16)
    v = torch.randn(n, heads, 16, device="cuda", dtype=torch.bfloat16)
    one = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    batch = Batch(one[:n].view(n, 1).flip(0).contiguous(), one, torch.ones(n, dtype=torch.int32, device="cuda"), max_q=1, max_len=1)
    cache.append(batch, v, v)
    _, want = cache.read(batch, n, dtype=torch.bfloat16)
    assert torch.equal(cache.attend(batch, v), want)


def test_rows_cut_off_keep_their_positions(gpu):
    """Row arrays that end inside a sequence, whatever kernel takes them."""
    for lens, news in (([700, 500], [3, 4]), ([900, 800], [300, 700]), ([9000, 6000], [1, 3])):
        s = Long(113, lens, news, 64, 1, 64)
        q, _ = s.query(4, "f32")
        want = s.cache.attend(s.batch, q)
        n = s.rows - 2
        got = s.cache.attend(s.batch, q[:n].contiguous())
        # perhaps summed in another order; a position off by one changes a row by some 1e-3
        assert (got - want[:n]).abs().max() < 2e-5


def test_sequences_that_share_pages(gpu):
    """A common beginning cached once."""
    import torch
    from bfp.kv4 import Batch
    s = Long(101, [9000], [1], 64, 2, 64)
    q = torch.randn(3, 6, 64, device="cuda")
    lens = [9000, 4700, 100]
    pages = s.batch.pages.expand(3, -1).contiguous()
    got = s.cache.attend(Batch(pages, _int([0, 1, 2, 3]), _int(lens), max_q=1, max_len=9000), q)
    for b in range(3):
        want = s.cache.attend(Batch(s.batch.pages, _int([0, 1]), _int(lens[b:b + 1]), max_q=1, max_len=9000), q[b:b + 1])
        # cut elsewhere: the same sums in another order
        assert (got[b] - want[0]).abs().max() < 1e-4


def _steps(s, kind="bf16"):
    """Calls that share keys between workgroups, of growing lengths."""
    lens = [[4500, 1, 300], [4501, 64, 9000], [17, 6000, 8999], [1, 1, 1], [0, 0, 5000], [9000, 9000, 9000]]
    q, _ = s.query(6, kind)
    return q, [_int(n) for n in lens]


def test_same_result_every_time_whatever_the_scratch_held(gpu):
    import torch
    from bfp.kv4 import Batch
    s = Long(103, [9000] * 3, [1, 1, 1], 64, 2, 64)
    q, lens = _steps(s)
    b = [Batch(s.batch.pages, s.batch.start, n, max_q=1, max_len=9000) for n in lens]
    first = [s.cache.attend(x, q) for x in b]
    work = torch.empty(s.cache.attend_work(b[0], q), dtype=torch.uint8, device="cuda")
    assert work.numel() > 0
    for fill in (0, 255, 127):
        work.fill_(fill)
        for _ in range(5):
            for x, want in zip(b, first):       # the same scratch, call after call
                assert torch.equal(s.cache.attend(x, q, work=work), want)


def test_two_streams_at_once(gpu):
    """Calls under way at the same time, each with its own scratch."""
    import torch
    from bfp.kv4 import Batch
    s = Long(107, [9000] * 3, [1, 1, 1], 64, 2, 64)
    q, lens = _steps(s)
    b = [Batch(s.batch.pages, s.batch.start, n, max_q=1, max_len=9000) for n in lens]
    want = [s.cache.attend(x, q) for x in b]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] += [s.cache.attend(x, q) for x in b]
    torch.cuda.synchronize()
    for g in got:
        for i, x in enumerate(g):
            assert torch.equal(x, want[i % len(want)])


@pytest.mark.parametrize("news,kind", [([1, 1, 1], "bf16"), ([200, 1, 100], "f32")])
def test_captured_and_replayed(gpu, news, kind):
    """One captured call, replayed over lengths that change in its batch, with
    eager calls of the same scratch in between."""
    import torch
    from bfp.kv4 import Batch
    s = Long(109, [9000] * 3, news, 64, 2, 64)
    q, lens = _steps(s, kind)
    held = lens[0].clone()
    b = Batch(s.batch.pages, s.batch.start, held, max_q=max(news), max_len=9000)
    work = torch.empty(max(s.cache.attend_work(b, q), 1), dtype=torch.uint8, device="cuda")
    want = []
    for n in lens:
        held.copy_(n)
        want.append(s.cache.attend(b, q))
    out, again = torch.zeros_like(q), torch.zeros_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.cache.attend(b, q, out=out, work=work)
        s.cache.attend(b, q, out=again, work=work)
    for turn in range(3):
        for n, w in zip(lens, want):
            held.copy_(n)
            out.fill_(7)
            graph.replay()
            if turn:
                assert torch.equal(s.cache.attend(b, q, work=work), w)
            torch.cuda.synchronize()
            rows = sum(news)
            assert torch.equal(out[:rows], w[:rows]) and torch.equal(again[:rows], w[:rows])


def test_rows_far_apart(gpu):
    """Row strides whose offsets pass 2^31 values and 2^32 bytes: queries,
    new keys and values, and results."""
    import torch
    from bfp import rotary
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of GPU memory")
    n, far = 40, 1 << 26
    s = Long(127, [700], [n], 64, 2, 64)
    q, _ = s.query(6, "bf16")
    wide_q = torch.empty(n * far, dtype=torch.bfloat16, device="cuda").as_strided((n, 6, 64), (far, 64, 1))
    wide_o = torch.empty(n * far, dtype=torch.bfloat16, device="cuda").as_strided((n, 6, 64), (far, 64, 1))
    wide_q.copy_(q)
    s.cache.attend(s.batch, wide_q, out=wide_o)
    assert torch.equal(wide_o, s.cache.attend(s.batch, q))
    table = rotary.rope_table(rotary.rope_freqs(64)[0], 700)
    pos = torch.arange(660, 700, dtype=torch.int32, device="cuda")
    rotary.rope(wide_q, pos, table, out=wide_o)
    assert torch.equal(wide_o, rotary.rope(q, pos, table))
    k = wide_q[:, :2]
    turned = s.cache.append(s.batch, k, wide_q[:, 2:4], table, q=wide_q, q_out=wide_o)
    far_k, far_v = s.cache.read(s.batch, n)
    assert turned is wide_o and torch.equal(turned, rotary.rope(q, pos, table))
    s.cache.append(s.batch, q[:, :2], q[:, 2:4], table)
    near_k, near_v = s.cache.read(s.batch, n)
    assert torch.equal(far_k, near_k) and torch.equal(far_v, near_v)
    s.cache.read(s.batch, k=wide_o[:, :2], v=wide_o[:, 2:4])
    assert torch.equal(wide_o[:, :2].float(), near_k) and torch.equal(wide_o[:, 2:4].float(), near_v)
