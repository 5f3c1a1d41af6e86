"""The ends of what the rotary and 4-bit-cache operators allow: scales,
magnitudes and exponents at the limits, results that cannot be held, strides
that nothing uses, and the kernels that only large calls reach, against
plain 64-bit numpy."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import HALF, _dt, _int, _say
from test_gpu_kv4_long import Long

pytestmark = pytest.mark.gpu


class Few:
    """One sequence whose keys differ in value 0 of the head only and whose
    values are alike in every place: k0 and v (tokens) are elements of the
    format times 2^(exponent byte - 127)."""

    def __init__(self, k0, v, k_exp=127, v_exp=127, news=1, page=16, hd=16):
        import torch
        from bfp.kv4 import Batch, Fp4Cache
        self.heads, self.hd, self.n, self.rows = 1, hd, len(k0), news
        code = {x * s: i + (8 if s < 0 else 0) for i, x in enumerate(ref.GRID.tolist()) for s in (1, -1) if x or s > 0}
        n_pages = -(-self.n // page)
        raw = {name: np.zeros((n_pages, 1, hd // 16, page, 8), np.uint8) for name in "kv"}
        for t in range(self.n):
            raw["k"][t // page, 0, 0, t % page, 0] = code[float(k0[t])]
            raw["v"][t // page, 0, :, t % page] = code[float(v[t])] * 17
        exps = {name: np.full((n_pages, 1, hd // 16, page), e, np.uint8) for name, e in (("k", k_exp), ("v", v_exp))}
        self.cache = Fp4Cache.from_buffers(*(torch.from_numpy(x).cuda() for x in (raw["k"], exps["k"], raw["v"], exps["v"])))
        self.batch = Batch(_int(np.arange(n_pages)[None]), _int([0, news]), _int([self.n]), max_q=news, max_len=self.n)
        self.k0 = np.asarray(k0, float) * 2.0 ** (k_exp - 127)
        self.v = np.asarray(v, float) * 2.0 ** (v_exp - 127)

    def query(self, q0, kind):
        """Queries (rows, query heads) of value 0, zeros elsewhere."""
        import torch
        q = torch.zeros(self.rows, q0.shape[1], self.hd, dtype=_dt(kind))
        q[:, :, 0] = torch.from_numpy(q0).to(_dt(kind))
        return q.cuda(), q[:, :, 0].double().numpy()

    def want(self, q0, scale):
        """(result, weighted magnitudes, largest score) of each row and query head."""
        out = np.zeros(q0.shape + (3,))
        for i in range(self.rows):
            seen = self.n - self.rows + i + 1
            s = q0[i][:, None] * self.k0[:seen] * scale
            w = np.exp(s - s.max(-1, keepdims=True))
            out[i, :, 0], out[i, :, 1] = (w @ self.v[:seen] / w.sum(-1), w @ np.abs(self.v[:seen]) / w.sum(-1))
            out[i, :, 2] = np.abs(s).max(-1)
        return out[..., 0], out[..., 1], out[..., 2]


def test_lengths_counted_in_place(gpu):
    """batch.lens += 1, as a decode loop has it."""
    import torch
    from bfp.kv4 import Batch
    s = Long(157, [60, 9], [1, 1], 16, 1, 64)
    lens = torch.tensor([40, 8], dtype=torch.int32, device="cuda")
    b = Batch(s.batch.pages, s.batch.start, lens, max_q=1, max_len=60)
    q = torch.randn(2, 3, 64, device="cuda")
    for n in range(4):
        b.lens += 1
        assert b.lens is lens and lens.tolist() == [41 + n, 9 + n]
    want = Batch(s.batch.pages, s.batch.start, _int([44, 12]), max_q=1, max_len=60)
    got, want = s.cache.attend(b, q), s.cache.attend(want, q)
    # the second sequence now counts slots that no token has written: noise, which may be NaN
    assert torch.equal(got[0], want[0]) and torch.allclose(got, want, rtol=0, atol=0, equal_nan=True)


def test_one_row_of_any_stride(gpu):
    """The stride between rows where there is one, and between heads where
    there is one, is nobody's."""
    import torch
    from bfp.kv4 import Batch
    s = Long(139, [60], [1], 16, 1, 64)
    b = Batch(s.batch.pages, s.batch.start, s.batch.lens, max_q=1, max_len=60)
    for kind in (torch.float32, torch.bfloat16):
        k = torch.randn(1, 1, 64, device="cuda", dtype=kind)
        q = torch.randn(1, 3, 64, device="cuda", dtype=kind)
        odd_k, odd_q = (torch.zeros(4096, device="cuda", dtype=kind).as_strided(x.shape, st) for x, st in ((k, (67, 3, 1)), (q, (193, 64, 1))))
        odd_k.copy_(k)
        odd_q.copy_(q)
        s.cache.append(b, k, k)
        want, wk = s.cache.attend(b, q), s.cache.read(b, 1)[0]
        out = torch.zeros(4096, device="cuda", dtype=kind).as_strided((1, 3, 64), (193, 64, 1))
        turned = torch.zeros_like(out)
        assert s.cache.append(b, odd_k, odd_k, q=odd_q, q_out=turned) is turned and torch.equal(turned, q)
        back = torch.zeros(4096, device="cuda").as_strided((1, 1, 64), (5, 7, 1))
        s.cache.read(b, k=back)
        assert torch.equal(back, wk)
        assert torch.equal(s.cache.attend(b, odd_q, out=out), want) and torch.equal(out, want)


def test_a_type_that_the_result_does_not_have(gpu):
    import torch
    s = Long(149, [60], [2], 16, 1, 64)
    q = torch.randn(2, 3, 64, device="cuda")
    pair = (torch.empty(2, 3, 64, dtype=torch.int16, device="cuda"), torch.empty(2, 3, 4, dtype=torch.int8, device="cuda"))
    out, kv = torch.empty_like(q), torch.empty(2, 1, 64, device="cuda")
    for bad in (lambda: s.cache.attend(s.batch, q, out=out, dtype=torch.bfloat16), lambda: s.cache.attend(s.batch, q, out=pair, dtype=torch.float32),
                lambda: s.cache.attend_work(s.batch, q, out=out, dtype=torch.float16), lambda: s.cache.read(s.batch, k=kv, dtype=torch.bfloat16),
                lambda: s.cache.read(s.batch, n_rows=3, v=kv)):
        with pytest.raises(ValueError):
            bad()
    assert s.cache.attend(s.batch, q, out=out, dtype=torch.float32) is out
    assert s.cache.read(s.batch, n_rows=2, k=kv, dtype=torch.float32)[0] is kv


def test_numbers_that_an_int_does_not_hold(gpu):
    """They do not come back from the other end."""
    import torch
    from bfp.kv4 import Batch
    s = Long(151, [60], [2], 16, 1, 64)
    q = torch.randn(2, 3, 64, device="cuda")
    for bad in (2 ** 32 + 16, 2 ** 31, 2 ** 64 + 1):
        for call in (lambda: s.cache.attend(s.batch, q, window=bad), lambda: s.cache.attend_work(s.batch, q, window=bad),
                     lambda: Batch(s.batch.pages, s.batch.start, s.batch.lens, max_q=bad),
                     lambda: Batch(s.batch.pages, s.batch.start, s.batch.lens, max_q=1, max_len=bad)):
            with pytest.raises(ValueError):
                call()
    assert torch.equal(s.cache.attend(s.batch, q, window=2 ** 31 - 1), s.cache.attend(s.batch, q))


SCALES = [  # scale, exponent byte of the keys, size of the queries
    (2.0 ** -110, 227, 2.0 ** 8), (2.0 ** -120, 227, 2.0 ** 18), (2.0 ** -125, 227, 2.0 ** 22),
    (0.0, 227, 2.0 ** 20), (-0.0, 227, 2.0 ** 20), (1e-40, 227, 2.0 ** 20), (-1e-46, 227, 2.0 ** 20), (1e-320, 227, 1.0),
    (2.0 ** -20, 127, 2.0 ** 20), (2.0 ** 110, 27, 2.0 ** -10), (-2.0 ** 100, 27, 1.0), (2.0 ** 100, 67, 2.0 ** -40)]


@pytest.mark.parametrize("news", [1, 6, 700])
@pytest.mark.parametrize("scale,k_exp,size", SCALES)
def test_scales_at_the_ends(gpu, scale, k_exp, size, news):
    """Any scale that float32 holds, whatever the products' size, and those
    too small for it, which leave all scores alike."""
    rng = np.random.default_rng(3)
    n = 700
    s = Few(rng.choice(np.concatenate([ref.GRID, -ref.GRID[1:]]), n), rng.choice(ref.GRID, n), k_exp, news=news)
    for kind in ("f32", "bf16"):
        q, q0 = s.query(rng.uniform(-1, 1, (news, 4)) * size, kind)
        want, weight, big = s.want(q0, scale)
        got = s.cache.attend(s.batch, q, scale=scale).double().cpu().numpy()
        # a scale below float32's normal numbers is off by half of 2^-149, its score by that times q.k < 2^126
        lost = 2.0 ** -23 if abs(scale) < 2.0 ** -126 else 0.0
        bound = ref.attend_bound(want[..., None], weight[..., None], big, n, s.hd, HALF[kind],
                                 (2.0 ** -24 if kind == "f32" else 2.0 ** -8) + 2 * lost)
        assert np.isfinite(got).all()
        assert (np.abs(got - want[..., None]) <= bound).all(), (kind, np.abs(got - want[..., None]).max())


def test_sums_of_the_largest_values(gpu):
    """The largest value the cache holds in 200192 tokens whose scores all
    lie just under the point where the running maximum would follow: the
    result is that value."""
    import torch
    from bfp.kv4 import Batch
    n, news, page = 200192, 33024, 256
    s = Few(np.concatenate([np.full(page, -6.0), np.zeros(page)]), np.full(2 * page, 6.0), v_exp=227, page=page)
    batch = Batch(_int([[0] + [1] * (n // page - 1)]), _int([0, news]), _int([n]), max_q=news, max_len=n)
    q = torch.zeros(news, 1, 16, dtype=torch.bfloat16, device="cuda")
    q[:, :, 0] = 1
    out = s.cache.attend(batch, q, scale=7.9 / 6 * np.log(2)).double()
    top = 6 * 2.0 ** 100
    assert torch.isfinite(out).all()
    # two sums of n terms, 2^-23 each at most, and the result's own rounding
    assert float((out / top - 1).abs().max()) <= (2 * n + 16) * 2.0 ** -23 + 2.0 ** -8


@pytest.mark.parametrize("lens,news,window,hd,group", [(130, 100, 0, 64, 3), (130, 3, 0, 64, 3), (5001, 3, 0, 64, 3), (5001, 2, 4500, 128, 2),
                                                       (1200, 1000, 0, 128, 4), (900, 600, 300, 64, 4), (700, 400, 0, 256, 2)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_any_byte_stays_with_those_who_see_it(gpu, lens, news, window, hd, group, kind):
    """Exponent bytes that no append writes, the largest elements beside
    them: rows that do not see the token are as they were."""
    s = Long(131, [lens], [news], 16, 1, hd)
    q, _ = s.query(group, kind)
    clean = s.cache.attend(s.batch, q, window=window).double().cpu().numpy()
    pos = np.arange(lens - news, lens)
    for p, tile in ((lens - 1, 1), (lens - news // 2 - 1, 0), (lens - news, 3), (2, 2)):
        page, slot = int(s.table[0, p // 16]), p % 16
        sees = (pos >= p) & ((pos - window < p) if window else True)
        for exps, data, dims in ((s.cache.v_exp, s.cache.v, slice(16 * tile, 16 * tile + 16)), (s.cache.k_exp, s.cache.k, slice(0, hd))):
            old = int(exps[page, 0, tile, slot]), data[page, 0, tile, slot].clone()
            data[page, 0, tile, slot] = 0x7f
            for byte in (252, 253, 254, 255, 0):
                exps[page, 0, tile, slot] = byte
                got = s.cache.attend(s.batch, q, window=window).double().cpu().numpy()
                apart = np.ones(got.shape, bool)
                apart[sees, :, dims] = False
                assert (got[apart] == clean[apart]).all(), (p, tile, byte)
                if byte >= 253 and exps is s.cache.v_exp:
                    assert np.isnan(got[~apart]).all(), (p, tile, byte)
            exps[page, 0, tile, slot], data[page, 0, tile, slot] = old[0], old[1]


@pytest.mark.parametrize("lens,news,hd,group", [([40, 7], [1, 1], 64, 2), ([5000, 7], [2, 1], 64, 2), ([300, 7], [1, 1], 256, 2),
                                                ([900, 7], [600, 7], 64, 2), ([6000], [64], 64, 4), ([900], [800], 112, 3)])
def test_what_tiles_cannot_hold(gpu, lens, news, hd, group):
    """16-bit tiles have no NaN: such values are the most negative number
    that they have, whoever joins the rows."""
    import torch
    s = Long(137, lens, news, 16, 1, hd)
    n = s.rows

    def tiles(q):
        m = torch.empty(n, group, hd, dtype=torch.int16, device="cuda")
        e = torch.empty(n, group, hd // 16, dtype=torch.int8, device="cuda")
        s.cache.attend(s.batch, q, out=(m, e))
        return m, e
    for kind in ("f32", "bf16"):
        q, _ = s.query(group, kind)
        m, e = tiles(q)
        for value, row in ((float("nan"), 0), (float("inf"), n - 1), (float("-inf"), n // 2)):
            q2 = q.clone()
            q2[row, 1, 3] = value
            m2, e2 = tiles(q2)
            wm, we = m.clone(), e.clone()
            wm[row, 1], we[row, 1] = -32768, 127
            assert torch.equal(m2, wm) and torch.equal(e2, we), (kind, value, row)
    # a tile of a value that all rows of the last sequence see
    b, tile = len(lens) - 1, hd // 16 - 1
    s.cache.v_exp[int(s.table[b, 0]), 0, tile, 0] = 255
    m2, e2 = tiles(q)
    first = int(s.start[b])
    wm, we = m.clone(), e.clone()
    wm[first:, :, 16 * tile:], we[first:, :, tile] = -32768, 127
    assert torch.equal(m2, wm) and torch.equal(e2, we)


def test_one_term_probabilities_and_their_sum(gpu):
    """Where probabilities go into the product rounded to bfloat16, their
    sum takes them rounded too.  In every 64 keys one has the largest score,
    the others a probability that rounds up by nearly half a step: a sum of
    unrounded ones would leave the results 2^-8 too large."""
    k0 = np.where(np.arange(512) % 64 == 5, 0.0, -1.0)
    v = np.full(512, 2.0)
    v[[1, 90, 200, 300, 400, 511]] = 1.5
    s = Few(k0, v)
    scale = -np.log(0.5 + 2.0 ** -9 + 2.0 ** -13)
    q, q0 = s.query(np.ones((1, 16)), "bf16")
    want, _, _ = s.want(q0, scale)
    got = s.cache.attend(s.batch, q, scale=scale).double().cpu().numpy()
    assert 1.993 < want.min() and want.max() < 1.996
    # half a bfloat16 step of a result in [1, 2); one key in 64 (3% of the weight) is not rounded up as the
    # others are, by 2^-8, which moves the mean by 0.03 * 2^-8 of the values' spread of 0.5 at most
    assert (np.abs(got - want[..., None]) <= 2.0 ** -8 + 2.0 ** -14).all(), np.abs(got - want[..., None]).max()


def test_scratch_size_allocates_nothing(gpu):
    import torch
    s = Long(163, [9000], [1], 64, 2, 64)
    q = torch.zeros(1, 6, 64, device="cuda").expand(1 << 15, 6, 64)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    assert s.cache.attend_work(s.batch, q) > 0
    assert torch.cuda.max_memory_allocated() == before


LARGE = [  # rows, heads, hd, rot, type in, type out, heads beside them
    (2000, 33, 64, 64, "bf16", "bf16", 0), (2000, 33, 64, 64, "f32", "f32", 3), (1500, 33, 128, 64, "f16", "f16", 2),
    (1500, 33, 128, 64, "f32", "bf16", 1), (2100, 33, 64, 32, "bf16", "f32", 5), (4200, 17, 64, 64, "tile", "f32", 0),
    (4200, 17, 64, 32, "tile", "f16", 2), (8200, 8, 64, 64, "f16", "bf16", 0)]


def _large(seed, rows, heads, hd, kind, extra):
    """Rows inside wider ones and the values they hold."""
    import torch
    from bfp import api
    v = np.random.default_rng(seed).standard_normal((rows, heads + extra, hd)).astype(np.float32)
    if kind == "tile":
        m, e = api.tile_quantize(v.astype(np.float64).reshape(-1))
        m, e = np.asarray(m, np.int16).reshape(v.shape), np.asarray(e, np.int8).reshape(*v.shape[:2], hd // 16)
        held = m * np.repeat(2.0 ** (e.astype(float) - 15), 16, -1)
        return tuple(torch.from_numpy(np.ascontiguousarray(x)).cuda()[:, :heads] for x in (m, e)), held[:, :heads]
    t = torch.from_numpy(v).to(_dt(kind))
    return t.cuda()[:, :heads], t.double().numpy()[:, :heads]


def _rotated(got, want, name):
    # a float32 result is rounded once; a 16-bit one comes from a float32 value at most two steps off
    tiny = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}[name] / 2
    slack = 0 if name == "f32" else 2.0 ** -22
    return (np.abs(got.double().cpu().numpy() - want) <= (HALF[name] + slack) * np.abs(want) + 2.0 ** -49 + tiny).all()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("case", LARGE, ids=str)
def test_rotations_of_many_rows(gpu, case, inter):
    """Calls of 262144 units and more, where a thread turns two heads: odd
    head counts leave the last one alone; into new rows, into joined ones
    and, with the new keys' append, beside the cache."""
    import torch
    from bfp import rotary
    rows, heads, hd, rot, kind, out_kind, extra = case
    x, val = _large(rows + rot, rows, heads, hd, kind, extra)
    n_pos = 3000
    table = ref.angles(n_pos, rot).astype(np.float32)
    dev = torch.from_numpy(table).cuda()
    pos = np.random.default_rng(9).integers(0, n_pos, rows)
    want = ref.rotate(val, pos, table, inter)
    per_head = rot // (8 if inter else 16) + (hd - rot) // 8
    assert rows * heads * per_head >= 2 * 256 * 8 * 64      # the line above which two heads go together
    _say(case, inter)
    assert _rotated(rotary.rope(x, _int(pos), dev, interleaved=inter, dtype=_dt(out_kind)), want, out_kind)
    joined = torch.full((rows, heads + 3, hd), 7.0, device="cuda", dtype=_dt(out_kind))
    rotary.rope(x, _int(pos), dev, interleaved=inter, out=joined[:, 1:1 + heads])
    assert _rotated(joined[:, 1:1 + heads], want, out_kind)
    assert (joined[:, 0] == 7).all() and (joined[:, 1 + heads:] == 7).all()
    # queries with the append: sequences of ragged lengths, at the given positions
    cut = rows // 3
    s = Long(167, [cut, rows - cut - 2], [cut, rows - cut], 64, 1, hd)      # two rows without a slot: zeros
    k = torch.randn(rows, 1, hd, device="cuda")
    joined.fill_(7.0)
    s.cache.append(s.batch, k, k, dev, interleaved=inter, pos=_int(pos), q=x, q_out=joined[:, 2:2 + heads])
    want[cut:cut + 2] = 0
    assert _rotated(joined[:, 2:2 + heads], want, out_kind)
    assert (joined[:, :2] == 7).all() and (joined[:, 2 + heads:] == 7).all()


def test_few_rows_carry_probabilities_in_two_terms(gpu):
    """bfloat16 calls of up to 8 rows a KV head: two kinds of keys whose
    probabilities differ by 2^-10, which one bfloat16 does not hold, and
    whose values cancel."""
    n = 128
    s = Few(np.where(np.arange(n) % 2, -1.0, 0.0), np.where(np.arange(n) % 2, -1.0, 1.0))
    for group in (1, 3, 8):
        q, q0 = s.query(np.ones((1, group)), "bf16")
        want, weight, big = s.want(q0, 2.0 ** -10)
        got = s.cache.attend(s.batch, q, scale=2.0 ** -10).double().cpu().numpy()
        bound = ref.attend_bound(want[..., None], weight[..., None], big, n, 1, HALF["bf16"], 2.0 ** -16)
        assert (bound < np.abs(want[..., None]) / 2).all()
        assert (np.abs(got - want[..., None]) <= bound).all(), (group, np.abs(got - want[..., None]).max())


@pytest.mark.parametrize("lens,news,page,heads,hd,group", [([1, 0, 2, 15, 16, 17], [1, 0, 1, 1, 1, 1], 16, 3, 64, 3), ([300, 555], [1, 1], 64, 2, 128, 8),
                                                           ([2000], [1], 16, 3, 64, 3), ([40, 7, 130], [4, 2, 3], 16, 2, 64, 2)])
def test_few_rows_within_two_terms(gpu, lens, news, page, heads, hd, group):
    """The bound of two terms on ordinary calls of few rows."""
    from test_gpu_kv4 import Setup, _typed, check
    s = Setup(59, lens, news, page, heads, hd)
    q, qv = _typed(s.rng.standard_normal((s.rows, heads * group, hd)) * 2, "bf16")
    assert max(news) * group <= 8
    check(s, q, qv, "bf16", "bf16", got=s.cache.attend(s.batch, q), max_p=2.0 ** -16)
