"""Attention over a shared prefix where the two parts of the work differ:
sequences outside every group with more rows than the groups have, scratch
that holds NaN before the call."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import HALF, _dt, _int, _say, _typed
from test_gpu_kv4_shared import CASES, Groups, _bound

pytestmark = pytest.mark.gpu


def _attend(t, q, dtype=None, window=0):
    """attend() with scratch in which a part that nobody writes is NaN."""
    import torch
    size = t.s.cache.attend_work(t.batch, q, shared=t.shared, dtype=dtype, window=window)
    work = torch.full(((size + 3) // 4,), float("nan"), device="cuda")
    return t.s.cache.attend(t.batch, q, shared=t.shared, dtype=dtype, window=window, work=work)


@pytest.mark.parametrize("hints", [True, False])
@pytest.mark.parametrize("hd,hq,heads", [(64, 2, 2), (128, 2, 1), (256, 1, 1), (64, 9, 3), (128, 32, 8)])
@pytest.mark.parametrize("most,mine", [(9, 1), (16, 8), (17, 2), (20, 2)])
def test_more_rows_outside_the_groups(gpu, most, mine, hd, hq, heads, hints):
    """Groups of `mine` rows a KV head at most, a draft of `most` or more outside."""
    group = hq // heads
    one, draft = max(1, mine // group // 2), -(-most // group)
    t = Groups(3, [40], [0, 0, -1], [41 + one, 60, 70 + draft], [one, 1, draft], 16, heads, hd, hints=hints, max_rows=one + 1)
    q, qv = _typed(t.s.rng.standard_normal((t.rows, hq, hd)), "bf16")
    _say(most, mine, hd, hq, heads, hints)
    got = _attend(t, q).double().cpu().numpy()
    want, weight, big = t.want(qv, group, 1 / np.sqrt(hd), 0)
    assert (np.abs(got - want) <= _bound(want, weight, big, max(t.lens), hd, "bf16", "bf16", 9)).all()


@pytest.mark.parametrize("seqs,new,share,hd,hq,heads", [(5, 1, 304, 64, 9, 3), (9, 2, 400, 128, 4, 1), (40, 1, 500, 64, 8, 1), (24, 1, 500, 128, 16, 4),
                                                        (70, 8, 100, 32, 1, 1), (6, 4, 300, 192, 2, 1), (40, 1, 4000, 64, 8, 1)])
def test_bits_are_those_of_calls_without_groups(gpu, seqs, new, share, hd, hq, heads):
    """bfloat16 with up to 8 rows a KV head of a sequence: probabilities in two
    terms (2^-16 off), however many rows the group has.  Results that lie
    further from a rounding border than that and float32 may move them are the
    exact ones rounded; probabilities in bfloat16 move them to either side."""
    import torch
    t = Groups(21, [share], [0] * seqs, [share + new + b % 5 for b in range(seqs)], [new] * seqs, 16, heads, hd)
    q, qv = _typed(t.s.rng.standard_normal((t.rows, hq, hd)) * 0.01, "bf16")
    _say(seqs, new, share, hd, hq, heads)
    got = _attend(t, q).double().cpu().numpy()
    want, weight, big = t.want(qv, hq // heads, 1 / np.sqrt(hd), 0)
    off = ref.attend_bound(want, weight, big, max(t.lens), hd, 0, 2 * 2.0 ** -16)
    assert (np.abs(got - want) <= off + HALF["bf16"] * np.abs(want)).all()
    low, mid, high = (torch.from_numpy(x).bfloat16().double().numpy() for x in (want - off, want, want + off))
    sure = low == high
    assert share > 500 or sure.mean() > 0.02
    assert (got[sure] == mid[sure]).all()


def test_float32_is_as_exact_as_without_groups(gpu):
    """Probabilities one by one: key j and value j are 1 in channel j and 0
    elsewhere, so result j is 2^(q_j / 4) over the sum.  Scores are exact here, up
    to 8 powers of two below the largest, and exponents at most 16 below 0
    where the maximum goes 2^8 above it: each is rounded to 2^-21 and the
    exponential to 2^-23 (uniformly: over the root of 3), the result twice to 2^-24:
    2.1e-7 in all; a third more is allowed."""
    import torch
    rows, heads = 24, 3
    t = Groups(4, [16], [0] * rows, [17] * rows, [1] * rows, 16, 1, 32)
    c, s = t.s.cache, t.s
    one_hot = np.zeros((2, 16, 8), np.uint8)                 # tile, slot, byte
    one_hot[0, np.arange(16), np.arange(16) // 2] = 2 << (4 * (np.arange(16) % 2))
    own = np.zeros((2, 16, 8), np.uint8)
    own[1, 0, 0] = 2                                         # a row's own token: key 0, value 1 in channel 16
    for x, mine in ((c.k, 0 * own), (c.v, own)):
        x[int(s.table[0, 0]), 0] = torch.from_numpy(one_hot).cuda()
        for b in range(rows):
            x[int(t.table[b, 1]), 0] = torch.from_numpy(mine).cuda()
    c.k_exp.fill_(127), c.v_exp.fill_(127)
    q = np.zeros((rows, heads, 32))
    q[:, :, :16] = s.rng.random((rows, heads, 16)) * 31
    q, qv = _typed(q, "f32")
    p = np.concatenate([2.0 ** (qv[:, :, :16] / 4), np.ones((rows, heads, 1))], -1)
    want = p / p.sum(-1, keepdims=True)
    plain = t.batch.pages.clone()
    plain[:, 0] = int(s.table[0, 0])
    for shared in (t.shared, None):
        if shared is None:
            t.batch.pages.copy_(plain)
        got = c.attend(t.batch, q, scale=0.25 / 1.44269504088896340736, shared=shared).double().cpu().numpy()
        assert (got[:, :, 17:] == 0).all()
        off = got[:, :, :17] / want - 1
        _say("float32", shared is not None, np.sqrt((off ** 2).mean()), np.abs(off).max())
        assert np.sqrt((off ** 2).mean()) < 2.8e-7


@pytest.mark.parametrize("hints", [True, False])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{len(c[1])}-{c[4:]}")
def test_every_part_that_is_joined_was_written(gpu, case, hints):
    """Rows behind the last sequence, of more bytes than the scratch of the
    others, are left alone and change no result."""
    import torch
    share, of, lens, news, page, heads, hd, hq, kind, out, window = case
    t = Groups(43, share, of, lens, news, page, heads, hd, hints=hints, max_rows=None if hints else 0)
    _say(case[0], case[4:], hints)
    more = 70
    q, qv = _typed(t.s.rng.standard_normal((t.rows + more, hq, hd)) * 1.5, kind)
    res = out or ("f32" if kind == "tile" else kind)
    to = torch.full((t.rows + more, hq, hd), 7.0, dtype=_dt(res), device="cuda")
    size = t.s.cache.attend_work(t.batch, q, out=to, shared=t.shared, window=window)
    work = torch.full(((size + 3) // 4,), float("nan"), device="cuda")
    t.s.cache.attend(t.batch, q, out=to, shared=t.shared, window=window, work=work)
    got = to.double().cpu().numpy()
    want, weight, big = t.want(qv[:t.rows], hq // heads, 1 / np.sqrt(hd), window)
    bound = _bound(want, weight, big, max(lens), hd, kind, res, t.rows * (hq // heads))
    assert (np.abs(got[:t.rows] - want) <= bound).all() and (got[t.rows:] == 7).all()


def test_parts_of_two_kinds_of_groups(gpu):
    """Captured once; group ranges and lengths move from many row tiles, whose
    keys stay whole, to few, whose keys are split, and back."""
    import torch
    t = Groups(44, [2000, 1500], [0] * 6 + [1] * 6, [2000 + 70 + b for b in range(6)] + [1600 + b for b in range(6)], [60] * 12, 16, 8, 64, max_rows=0)
    q, qv = _typed(t.s.rng.standard_normal((t.rows, 32, 64)), "bf16")
    out = torch.empty_like(q)
    size = t.s.cache.attend_work(t.batch, q, shared=t.shared)
    work = torch.full(((size + 3) // 4,), float("nan"), device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            t.s.cache.attend(t.batch, q, shared=t.shared, out=out, work=work)
    torch.cuda.synchronize()
    table = t.table.copy()
    for b in range(12):       # own pages that hold the shared tokens, for the sequences that are taken out of their group
        whole = [2000, 1500][t.of[b]] // 16
        table[b, :whole] = t.s.table[t.of[b], :whole]
        if [2000, 1500][t.of[b]] % 16:
            end, own = int(t.s.table[t.of[b], whole]), int(t.table[b, whole])
            for x in (t.s.cache.k, t.s.cache.k_exp, t.s.cache.v, t.s.cache.v_exp):
                x[own, :, :, :[2000, 1500][t.of[b]] % 16] = x[end, :, :, :[2000, 1500][t.of[b]] % 16]
    t.batch.pages.copy_(_int(table))
    want, weight, big = t.want(qv, 4, 1 / 8, 0)
    bound = _bound(want, weight, big, max(t.lens), 64, "bf16", "bf16", 720 * 4)
    for start in ([0, 6, 12], [5, 6, 7], [6, 6, 12], [0, 6, 6], [0, 6, 12]):
        t.shared.start.copy_(_int(start))
        out.fill_(float("nan"))
        work.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert (np.abs(out.double().cpu().numpy() - want) <= bound).all(), start
