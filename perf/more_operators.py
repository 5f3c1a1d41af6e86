"""Measured cases of the 4-bit cache's pages (branches forked, a pool made
compact, the bounds of each page's keys) and of the two attentions that use
them: over a prefix that sequences share, and over the pages that a score
picks for each query.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges,
``prepare`` makes a case's inputs, ``run`` makes one pass: in plain torch
where ``own`` is false, through ``bfp.pages`` and ``bfp.kv4`` where it is
true.  ``exact`` is the result in 64 bits and ``work`` what a pass cannot do
without.

The cache holds tiles of 16 values: 16 four-bit E2M1 elements (0, 0.5, 1,
1.5, 2, 3, 4, 6 and their negatives) and one exponent byte E, value =
element * 2^(E-127).  A page holds ``page`` tokens of every KV head, tile by
tile: k, v (pages, heads, hd/16, page, 8) bytes, the lower half of a byte
first, and ke, ve (pages, heads, hd/16, page).  The bounds of a page are the
least and the largest key of each channel, (pages, heads, 2, hd) bfloat16.
"""
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "tinyllm-fpga_amd"))

own = False

TILE = 16
E_MIN, E_MAX, E_NAN = -100, 100, 255     # the cache's exponents, and the byte of a tile without values
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NEG, POS = float("-inf"), float("inf")


# ------------------------------------------------------------------- cases
def listed():
    return [
        # four answers to one chat of the framework's own model, 30 layers: latency
        {"name": "fork_chat", "kind": "fork", "parents": 1, "children": 4, "ctx": 700, "new": 1, "layers": 30, "hkv": 3,
         "hd": 64, "page": 16},
        # 256 beams of which each goes on from one of 64, with the few tokens of a draft
        {"name": "fork_beams", "kind": "fork", "parents": 64, "children": 256, "ctx": 2048, "new": 5, "layers": 8,
         "hkv": 8, "hd": 128, "page": 64},
        # a small pool after some chats have ended
        {"name": "compact_small", "kind": "compact", "pages": 509, "share": 0.55, "seqs": 6, "layers": 30, "hkv": 3,
         "hd": 64, "page": 16},
        # a large pool made compact before it gives memory back
        {"name": "compact_large", "kind": "compact", "pages": 8192, "share": 0.5, "seqs": 48, "layers": 2, "hkv": 8,
         "hd": 128, "page": 64},
        # the bounds that a decode step of 64 sequences changes
        {"name": "bounds_step", "kind": "bounds", "seqs": 64, "new": 1, "ctx": 2048, "hkv": 3, "hd": 64, "page": 16},
        # the bounds of three ragged prompts
        {"name": "bounds_prompt", "kind": "bounds", "seqs": 3, "new": 8192, "ctx": 9000, "hkv": 8, "hd": 128, "page": 64},
        # the next token of five chats behind one system prompt: latency
        {"name": "shared_chat", "kind": "shared", "groups": 1, "seqs": 5, "new": 1, "prefix": 304, "ctx": 200, "hq": 9,
         "hkv": 3, "hd": 64, "page": 16, "dtype": "tile", "window": 0},
        # the next token of 64 samples of one long problem
        {"name": "shared_batch", "kind": "shared", "groups": 1, "seqs": 64, "new": 1, "prefix": 16384, "ctx": 2048,
         "hq": 32, "hkv": 8, "hd": 128, "page": 64, "dtype": "bf16", "window": 0},
        # drafts and short questions on three long documents
        {"name": "shared_long", "kind": "shared", "groups": 3, "seqs": 21, "new": 17, "prefix": 65536, "ctx": 509,
         "hq": 16, "hkv": 4, "hd": 96, "page": 64, "dtype": "f16", "window": 0},
        # the next token of one chat at 16 times the framework's context, 64 pages of it: latency
        {"name": "sparse_single", "kind": "sparse", "seqs": 1, "new": 1, "ctx": 32767, "picks": 64, "first": 1, "last": 2,
         "hq": 9, "hkv": 3, "hd": 64, "page": 16, "dtype": "tile"},
        # the next token of eight very long documents, 32 pages of each
        {"name": "sparse_long", "kind": "sparse", "seqs": 8, "new": 1, "ctx": 131072, "picks": 32, "first": 1, "last": 2,
         "hq": 32, "hkv": 8, "hd": 128, "page": 64, "dtype": "bf16"},
        # a piece of a long prompt, every row with pages of its own
        {"name": "sparse_piece", "kind": "sparse", "seqs": 1, "new": 1021, "ctx": 32768, "picks": 24, "first": 1,
         "last": 4, "hq": 32, "hkv": 4, "hd": 128, "page": 32, "dtype": "f16"},
    ]


def _log_int(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    return min(max(v, lo), hi)


def draw(rng):
    kind = rng.choice(["fork", "compact", "bounds", "shared", "shared", "sparse", "sparse"])
    hd = rng.choice([32, 48, 64, 64, 80, 96, 112, 128, 128, 192, 256])
    page = rng.choice([16, 32, 64, 128])
    hkv = rng.randint(1, 8)
    shape = {"hkv": hkv, "hd": hd, "page": page}
    if kind == "fork":
        parents, new = _log_int(rng, 1, 64), rng.choice([1, 1, rng.randint(2, 80)])
        ctx = _log_int(rng, 1, 4096)
        layers = max(1, min(rng.randint(1, 30), (1 << 29) // (parents * (ctx + page) * hkv * hd)))
        children = min(_log_int(rng, 1, 256), max(1, (1 << 29) // (layers * (page + new) * hkv * hd)))
        return {"kind": kind, "parents": parents, "children": children, "ctx": ctx, "new": new, "layers": layers, **shape}
    if kind == "compact":
        layers = rng.randint(1, 30)
        pages = _log_int(rng, 64, max(64, min(20000, (1 << 30) // (layers * page * hkv * hd))))
        return {"kind": kind, "pages": pages, "share": rng.uniform(0.05, 0.95), "seqs": _log_int(rng, 1, 64),
                "layers": layers, **shape}
    seqs = _log_int(rng, 1, 64)
    if kind == "bounds":
        new = rng.choice([1, 1, _log_int(rng, 2, max(2, 16000 // seqs))])
        new = min(new, max(1, (24 << 20) // (seqs * hkv * hd)))
        return {"kind": kind, "seqs": seqs, "new": new, "ctx": new + _log_int(rng, 1, 4096), **shape}
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32", "tile"])
    if kind == "shared":
        groups = rng.choice([1, 1, 2, 3])
        seqs = max(seqs, groups)
        new = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 300)])
        new = max(1, min(new, 4096 // seqs))
        most = max(256, (1 << 28) // (seqs * new * hq * groups))
        prefix = min(_log_int(rng, 64, 65536), most, (1 << 28) // (groups * hkv * hd))
        ctx = new + min(_log_int(rng, 1, 2048), most, (1 << 28) // (seqs * hkv * hd))
        return {"kind": kind, "groups": groups, "seqs": seqs, "new": new, "prefix": prefix, "ctx": ctx, "hq": hq, **shape,
                "dtype": dtype, "window": rng.choice([0, 0, 0, _log_int(rng, 1, 8192)])}
    new = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 1000)])
    seqs = max(1, min(seqs, 1024 // new))
    picks = _log_int(rng, 4, max(4, min(128, 2048 // page, (1 << 28) // (seqs * new * hkv * hd * page))))
    ctx = new + min(_log_int(rng, 1, 131072), (1 << 29) // (seqs * hkv * hd), (1 << 26) * page // (seqs * new * hkv))
    return {"kind": kind, "seqs": seqs, "new": new, "ctx": ctx, "picks": picks, "first": rng.choice([0, 1, 1]),
            "last": rng.randint(1, 3), "hq": hq, **shape, "dtype": dtype}


def _part(b):
    """Sequence b's share of the longest one's length."""
    return 1.0 - 0.61 * ((b * 0.6180339887) % 1.0) if b else 1.0


def _lengths(case):
    """How many new tokens each sequence has and how long it is with them:
    ragged, the first the longest; past two sequences one that is empty (its
    row a padded batch's).  From the case alone, so that work() knows them."""
    n, new, ctx = case["seqs"], case["new"], case["ctx"]
    news = [max(1, int(new * _part(b))) for b in range(n)]
    lens = [max(q, int(ctx * _part(b))) for b, q in enumerate(news)]
    if n > 2:
        news[-1], lens[-1] = (1 if new == 1 else 0), 0
    return news, lens


def _groups(case):
    """Where the groups of sequences begin, and what each shares: as many
    tokens as the longest, then fewer, whole pages or not."""
    g, n = case["groups"], case["seqs"]
    first = [i * n // g for i in range(g)] + [n]
    return first, [max(1, int(case["prefix"] * _part(i))) for i in range(g)]


def _shared_lengths(case):
    """_lengths() of the tokens behind what the groups share."""
    news, own_lens = _lengths(case)
    first, share = _groups(case)
    of = [max(i for i in range(len(share)) if first[i] <= b) for b in range(case["seqs"])]
    return news, [n and n + share[of[b]] for b, n in enumerate(own_lens)], of


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _bytes(g, *shape):
    return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _tile16(v):
    """16-bit tiles of float32 values: (m int16, e int8), v ~ m 2^(e-15)."""
    t = v.double().unflatten(-1, (-1, TILE))
    e = torch.frexp(t.abs().amax(-1))[1].clamp(-127, 127)
    m = torch.round(torch.ldexp(t, (15 - e).unsqueeze(-1))).clamp(-32768, 32767)
    return m.flatten(-2).to(torch.int16), e.to(torch.int8)


def _typed(v, dtype):
    return _tile16(v) if dtype == "tile" else v.to(DTYPES[dtype])


def _quant4(v):
    """Values (..., hd) to the cache's tiles: bytes (..., hd/16, 8) and
    exponent bytes (..., hd/16)."""
    t = v.unflatten(-1, (-1, TILE))
    f, x = torch.frexp(t.abs().amax(-1))                       # f 2^x, f in [0.5, 1)
    e = (x - 3 + (f >= 0.875).int()).clamp(E_MIN, E_MAX)
    t = torch.ldexp(t, -e.unsqueeze(-1))
    a = t.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(a.dtype)
    a = (torch.round(a / step) * step).clamp(max=6)
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | ((t < 0).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _pool(case, pages, g, layers=0):
    """Pages as they are found: whatever bytes were there; of several layers
    one after the other."""
    shape = ((layers,) if layers else ()) + (pages, case["hkv"], case["hd"] // TILE, case["page"])
    return {"k": _bytes(g, *shape, TILE // 2), "ke": _bytes(g, *shape), "v": _bytes(g, *shape, TILE // 2), "ve": _bytes(g, *shape)}


def _tables(lens, page, g, extra=3, wide=0):
    """Pages for sequences of lens tokens, dealt out in no order -> table,
    how many there are, and one that nobody has."""
    need = [-(-n // page) for n in lens]
    width = max(max(need), 1) + wide
    pages = sum(need) + extra
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([sum(need[:b]) for b in range(len(need))], device="cuda")
    at = torch.arange(width, device="cuda")
    held = at[None] < torch.tensor(need, device="cuda")[:, None]
    return torch.where(held, ids[(first[:, None] + at).clamp(max=pages - 1)], -1).to(torch.int32), pages, ids


def _filled(case, pages, g):
    """Keys with a few strong channels that lean the way of their page's
    subject, and plainer values."""
    c = _pool(case, pages, g)
    hd, hkv, page = case["hd"], case["hkv"], case["page"]
    strong = 1.0 + 3.0 * (torch.rand(hkv, 1, hd, generator=g, device="cuda") > 0.95)
    step = max(1, (1 << 27) // (hkv * page * hd))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        keys = (0.8 * _randn(g, n, hkv, 1, hd) + _randn(g, n, hkv, page, hd)) * strong
        for data, exp, x in (("k", "ke", keys), ("v", "ve", _randn(g, n, hkv, page, hd))):
            d, e = _quant4(x)
            c[data][p:p + n], c[exp][p:p + n] = d.transpose(2, 3), e.transpose(2, 3)
    return c


def _batch(table, news, lens):
    return {"table": table, "start": _int([0] + news).cumsum(0).to(torch.int32), "lens": _int(lens), "max_q": max(news),
            "max_len": max(lens), "rows": sum(news)}


def prepare(case, seed):
    g = _gen(seed)
    return {"fork": _prepare_fork, "compact": _prepare_compact, "bounds": _prepare_bounds, "shared": _prepare_shared,
            "sparse": _prepare_sparse}[case["kind"]](case, g)


def _fork_lengths(case):
    lens = [max(1, int(case["ctx"] * _part(b))) for b in range(case["parents"])]
    return lens, [lens[i % case["parents"]] for i in range(case["children"])]


def _prepare_fork(case, g):
    """Parents with their pages, the children's tables as yet empty."""
    page, n = case["page"], case["children"]
    lens, child = _fork_lengths(case)
    room = sum(1 + -(-case["new"] // page) for _ in child)
    table, pages, ids = _tables(lens, page, g, extra=room + 3, wide=-(-case["new"] // page) + 1)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[table[table >= 0].long()] = 1
    parents = _int([i % case["parents"] for i in range(n)])
    return {"case": case, "pool": _pool(case, pages, g, case["layers"]), "table": table, "lens": _int(lens), "refs": refs,
            "short": _int([0]), "parents": parents, "children": torch.full((n, table.shape[1]), -1, dtype=torch.int32, device="cuda"),
            "child_lens": _int([0] * n), "start": torch.arange(n + 1, device="cuda", dtype=torch.int32) * case["new"],
            "rows": n * case["new"]}


def _prepare_compact(case, g):
    """Sequences that hold some of the pool's pages, each second of them the
    first half of its neighbour's, too."""
    pages, n = case["pages"], case["seqs"]
    live = max(1, int(pages * case["share"]))
    each = -(-live // n)
    ids = torch.randperm(pages, generator=g, device="cuda")[:live].to(torch.int32)
    table = torch.full((n * each,), -1, dtype=torch.int32, device="cuda")
    table[:live] = ids
    table = table.view(n, each)
    half = each // 2
    forks = torch.where(torch.arange(each, device="cuda") < half, table, -1)[::2]
    table = torch.cat([table, forks]).contiguous()
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs.index_add_(0, table[table >= 0].long(), torch.ones_like(table[table >= 0]))
    return {"case": case, "pool": _pool(case, pages, g, case["layers"]), "table0": table, "refs0": refs,
            "table": table.clone(), "refs": refs.clone(), "live": _int([0])}


def _prepare_bounds(case, g):
    news, lens = _lengths(case)
    table, pages, _ = _tables(lens, case["page"], g)
    c = _filled(case, pages, g)
    shape = (pages, case["hkv"], 2, case["hd"])
    return {"case": case, "cache": c, "batch": _batch(table, news, lens), "bounds": _randn(g, *shape).bfloat16()}


def _prepare_shared(case, g):
    """Tables of each group's prefix and of the sequences, whose first pages
    are the prefix's: the page in which the prefix ends is a sequence's own."""
    news, lens, of = _shared_lengths(case)
    first, share = _groups(case)
    page, n = case["page"], case["seqs"]
    prefix, count, _ = _tables(share, page, g)
    whole = [share[of[b]] // page for b in range(n)]
    own_lens = [max(0, x - page * w) for x, w in zip(lens, whole)]
    mine, more, _ = _tables(own_lens, page, g)
    width = max(-(-x // page) for x in lens)
    at = torch.arange(width, device="cuda")[None]
    w = torch.tensor(whole, device="cuda")[:, None]
    behind = torch.gather(mine, 1, (at - w).clamp(0, mine.shape[1] - 1))
    table = torch.where((at >= w) & (at - w < mine.shape[1]) & (behind >= 0), behind + count, -1)
    before = prefix[_int(of).long()][:, :width]
    before = torch.nn.functional.pad(before, (0, width - before.shape[1]), value=-1)
    table = torch.where((at < w) & (_int(lens)[:, None] > 0), before, table).to(torch.int32)
    c = _filled(case, count + more, g)
    # what the prefix holds in the page in which it ends, the sequences' own page holds, too
    for b in range(n):
        if lens[b] and share[of[b]] % page:
            src, dst, k = prefix[of[b], whole[b]].long(), table[b, whole[b]].long(), share[of[b]] % page
            for name in c:
                c[name][dst, :, :, :k] = c[name][src, :, :, :k]
    batch = _batch(table.contiguous(), news, lens)
    q = _typed(_randn(g, batch["rows"], case["hq"], case["hd"]), case["dtype"])
    max_rows = max(sum(news[first[i]:first[i + 1]]) for i in range(len(share)))
    return {"case": case, "cache": c, "batch": batch, "prefix": prefix, "first": _int(first), "share": _int(share),
            "max_rows": max_rows, "max_share": max(share), "of": _int(of), "own": max(x - share[of[b]] for b, x in enumerate(lens)), "q": q}


def _prepare_sparse(case, g):
    news, lens = _lengths(case)
    table, pages, _ = _tables(lens, case["page"], g)
    c = _filled(case, pages, g)
    bounds = torch.empty(pages, case["hkv"], 2, case["hd"], dtype=torch.bfloat16, device="cuda")
    step = max(1, (1 << 27) // (case["hkv"] * case["page"] * case["hd"]))
    for p in range(0, pages, step):                              # every page as if it were full
        k = _values4(c["k"][p:p + step].transpose(2, 3), c["ke"][p:p + step].transpose(2, 3))
        bounds[p:p + step, :, 0], bounds[p:p + step, :, 1] = k.amin(2).bfloat16(), k.amax(2).bfloat16()
    batch = _batch(table, news, lens)
    q = _typed(_randn(g, batch["rows"], case["hq"], case["hd"]), case["dtype"])
    return {"case": case, "cache": c, "batch": batch, "bounds": bounds, "q": q}


# --------------------------------------------------------------------- run
def run(state):
    if own:
        return _run_own(state, state["case"])
    return {"fork": _fork, "compact": _compact, "bounds": _bounds, "shared": _shared, "sparse": _sparse}[state["case"]["kind"]](state, state["case"])


def _run_own(state, case):
    if "handle" not in state:      # what a serving loop keeps from call to call
        state["handle"] = _handles(state, case)
    if case["kind"] == "fork":
        pool, batch = state["handle"]
        pool.free(batch.pages)                                   # the branches of the pass before
        pool.fork(state["table"], state["lens"], state["parents"], out=(batch.pages, batch.lens))
        batch.lens += case["new"]
        pool.reserve(batch)
        return _fork_outputs(state)
    if case["kind"] == "compact":
        pool = state["handle"]
        _restore(state)
        live = pool.compact(state["table"])
        return _compact_outputs(state, live)
    cache, batch, more = state["handle"]
    if case["kind"] == "bounds":
        more.update(batch)
        return state["bounds"]
    if case["kind"] == "shared":
        return cache.attend(batch, state["q"], window=case["window"], shared=more)
    picks = more.select(batch, state["q"], case["picks"], first=case["first"], last=case["last"])
    return cache.attend(batch, state["q"], picks=picks), picks


def _handles(state, case):
    from bfp import kv4, pages
    if case["kind"] in ("fork", "compact"):
        p = state["pool"]
        caches = [kv4.Fp4Cache.from_buffers(p["k"][i], p["ke"][i], p["v"][i], p["ve"][i]) for i in range(case["layers"])]
        pool = pages.PagePool(caches, refs=state["refs"])
        if case["kind"] == "compact":
            return pool
        state["short"] = pool.short
        return pool, kv4.Batch(state["children"], state["start"], state["child_lens"], max_q=case["new"])
    c, b = state["cache"], state["batch"]
    cache = kv4.Fp4Cache.from_buffers(c["k"], c["ke"], c["v"], c["ve"])
    batch = kv4.Batch(b["table"], b["start"], b["lens"], max_q=b["max_q"], max_len=b["max_len"])
    if case["kind"] == "shared":
        return cache, batch, kv4.Shared(state["prefix"], state["first"], state["share"], max_rows=state["max_rows"], max_len=state["max_share"])
    return cache, batch, kv4.PageBounds.from_buffer(cache, state["bounds"])


def _words(t):
    """Bytes that are only moved, as whole numbers."""
    return t.view(torch.int64) if t.dim() == 6 else t.flatten(1).view(torch.int64)


def _fork_outputs(state):
    return (state["children"], state["child_lens"], state["refs"], state["short"], *(_words(state["pool"][n]) for n in ("k", "ke", "v", "ve")))


def _restore(state):
    """The tables and counts as the program found them, so that every pass has the same pages to move."""
    state["table"].copy_(state["table0"])
    state["refs"].copy_(state["refs0"])


def _compact_outputs(state, live):
    return (state["table"], state["refs"], live, *(_words(state["pool"][n]) for n in ("k", "ke", "v", "ve")))


def _drop(refs, table):
    held = table >= 0
    refs.index_add_(0, table.clamp(min=0).flatten().long(), -held.flatten().to(torch.int32))
    table.fill_(-1)


def _give(refs, short, want):
    """The lowest free pages for the entries `want` of a table, in its order: their numbers, -1 past the last."""
    rank = (want.flatten().cumsum(0) - 1).view(want.shape)
    free = (refs == 0).nonzero().flatten()
    n = free.numel()
    short += (want.sum() - n).clamp(min=0).to(torch.int32)
    got = want & (rank < n)
    free = torch.nn.functional.pad(free, (0, 1))
    ids = torch.where(got, free[rank.clamp(0, max(n - 1, 0))], -1)
    refs[ids[got]] = 1
    return ids


def _fork(state, case):
    page, refs, children, lens = case["page"], state["refs"], state["children"], state["child_lens"]
    _drop(refs, children)
    table = state["table"][state["parents"].long()]
    lens.copy_(state["lens"][state["parents"].long()])
    at = torch.arange(table.shape[1], device="cuda")[None]
    whole, part = lens[:, None] // page, lens[:, None] % page
    kept = (at < whole) & (table >= 0)
    refs.index_add_(0, table.clamp(min=0).flatten().long(), kept.flatten().to(torch.int32))
    split = (at == whole) & (part > 0) & (table >= 0)
    fresh = _give(refs, state["short"], split)
    new = torch.where(kept, table.long(), torch.where(split, fresh, -1))
    src, dst = table[split & (fresh >= 0)].long(), fresh[split & (fresh >= 0)]
    for p in state["pool"].values():
        p[:, dst] = p[:, src]
    lens += case["new"]
    touched = (at >= (lens[:, None] - case["new"]) // page) & (at <= (lens[:, None] - 1) // page) & (new < 0)
    new = torch.where(touched, _give(refs, state["short"], touched), new)
    children.copy_(new)
    return _fork_outputs(state)


def _compact(state, case):
    _restore(state)
    refs, table = state["refs"], state["table"]
    used = refs > 0
    n = used.sum()
    ids = torch.arange(refs.numel(), device="cuda")
    src, dst = ids[used & (ids >= n)], ids[~used & (ids < n)]
    for p in state["pool"].values():
        p[:, dst] = p[:, src]
    to = ids.clone()
    to[src] = dst
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    refs[dst] = refs[src]
    refs[src] = 0
    return _compact_outputs(state, n.to(torch.int32).view(1))


def _wide(x, dtype):
    """Values of a tensor, or of 16-bit tiles, in a wider type (exact)."""
    if isinstance(x, tuple):
        m, e = x
        return torch.ldexp(m.to(dtype).unflatten(-1, (-1, TILE)), (e.to(torch.int32) - 15).unsqueeze(-1)).flatten(-2)
    return x.to(dtype)


def _values4(data, exp):
    """Tiles (..., hd/16, 8) and their exponents as float32 (..., hd)."""
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=data.device)
    v = lut[torch.stack([data & 15, data >> 4], -1).flatten(-2).int()]
    scale = torch.where(exp == E_NAN, torch.nan, torch.ldexp(torch.ones_like(exp, dtype=torch.float32), exp.int() - 127))
    return (v * scale.unsqueeze(-1)).flatten(-2)


def _bounds(state, case):
    batch, c, page = state["batch"], state["cache"], case["page"]
    lens, start = batch["lens"].long(), batch["start"].long()
    new = start[1:] - start[:-1]
    begin, end = (lens - new).clamp(min=0) // page, (lens + page - 1) // page
    p = begin[:, None] + torch.arange((batch["max_q"] + page - 2) // page + 1, device="cuda")
    seq, k = ((p < end[:, None]) & (new > 0)[:, None]).nonzero(as_tuple=True)
    p = p[seq, k]
    ids = batch["table"][seq, p].long()
    keys = _values4(c["k"][ids].transpose(2, 3), c["ke"][ids].transpose(2, 3))             # pages, hkv, slots, hd
    held = (torch.arange(page, device="cuda") < (lens[seq] - p * page)[:, None])[:, None, :, None]
    state["bounds"][ids, :, 0] = keys.masked_fill(~held, POS).amin(2).bfloat16()
    state["bounds"][ids, :, 1] = keys.masked_fill(~held, NEG).amax(2).bfloat16()
    return state["bounds"]


def _rows(batch):
    """Of every row of the batch: its sequence and its position."""
    row = torch.arange(batch["rows"], device="cuda")
    seq = torch.searchsorted(batch["start"].long(), row, right=True) - 1
    return seq, batch["lens"].long()[seq] - batch["start"].long()[seq + 1] + row


def _softmax_parts(q, k, v, seen):
    """Unfinished attention of rows (..., rows, hd) over keys (..., keys, hd): maxima, sums, and sums of values."""
    s = torch.matmul(q, k.transpose(-1, -2)).masked_fill_(~seen, NEG)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == NEG, torch.zeros_like(m), m)).exp_()
    return m, p.sum(-1, keepdim=True), torch.matmul(p, v)


def _tokens(c, ids):
    """The tokens of pages (..., width): keys and values (..., hkv, width * page, hd), zeros where there is no page."""
    d = ids.dim()
    held = lambda n: _values4(c[n][ids.clamp(min=0)].transpose(d + 1, d + 2), c[n + "e"][ids.clamp(min=0)].transpose(d + 1, d + 2))  # noqa: E731
    there = (ids >= 0)[..., None, None, None]
    flat = lambda x: torch.where(there, x, torch.zeros((), device="cuda")).transpose(d - 1, d).flatten(d, d + 1)  # noqa: E731
    return flat(held("k")), flat(held("v"))


def _shared(state, case):
    """The groups' prefixes with all rows of a group, then every sequence's own tokens; both joined."""
    batch, c, page, hq, hkv, hd = state["batch"], state["cache"], case["page"], case["hq"], case["hkv"], case["hd"]
    seq, pos = _rows(batch)
    start, first, share = batch["start"].long(), state["first"].long(), state["share"].long()
    of, window, group = state["of"].long(), case["window"] or 1 << 40, hq // hkv
    q = _wide(state["q"], torch.float32) / math.sqrt(hd)

    def part(begin, count, most, keys, vals, key_pos, limit):
        # rows begin .. begin + count - 1 of each owner, padded to most, against the owner's keys at key_pos below limit
        i = torch.arange(most, device="cuda")[None]
        row = (begin[:, None] + i).clamp(max=batch["rows"] - 1)
        mine = i < count[:, None]
        p = torch.where(mine, pos[row], -1)[:, :, None]
        seen = (key_pos[:, None] <= p) & (key_pos[:, None] > p - window) & (key_pos < limit[:, None])[:, None]
        x = q[row].unflatten(2, (hkv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)          # owners, hkv, group * n, hd
        got = _softmax_parts(x, keys, vals, seen.repeat(1, group, 1)[:, None])
        return [t.unflatten(2, (group, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)[mine] for t in got]    # rows, hq, .
    end = start[first]
    k, v = _tokens(c, state["prefix"].long())
    at = torch.arange(k.shape[2], device="cuda")[None].expand(len(share), -1)
    m1, l1, o1 = part(end[:-1], end[1:] - end[:-1], state["max_rows"], k, v, at, share)
    width = -(-state["own"] // page) + 1
    w = share[of] // page
    span = w[:, None] + torch.arange(width, device="cuda")
    ids = torch.where(span < batch["table"].shape[1], torch.gather(batch["table"].long(), 1, span.clamp(max=batch["table"].shape[1] - 1)), -1)
    k, v = _tokens(c, ids)
    at = (w * page)[:, None] + torch.arange(width * page, device="cuda")
    at = torch.where(at < share[of][:, None], 1 << 50, at)       # the prefix's own end is not seen twice
    m2, l2, o2 = part(start[:-1], start[1:] - start[:-1], batch["max_q"], k, v, at, torch.full_like(of, 1 << 49))
    m = torch.maximum(m1, m2)
    zero = torch.zeros((), device="cuda")
    f1, f2 = ((t - torch.where(m == NEG, zero, m)).exp() for t in (m1, m2))
    total = f1 * l1 + f2 * l2
    out = (f1 * o1 + f2 * o2) / torch.where(total == 0, torch.ones_like(total), total)
    return out.to(DTYPES.get(case["dtype"], torch.float32))


def _sparse(state, case):
    batch, c, page, hq, hkv, hd = state["batch"], state["cache"], case["page"], case["hq"], case["hkv"], case["hd"]
    seq, pos = _rows(batch)
    table = batch["table"].long()
    # scores in 64 bits: a page next to the border would go to either side otherwise
    i = torch.arange(batch["max_q"], device="cuda")[None]
    row = (batch["start"].long()[:-1, None] + i).clamp(max=batch["rows"] - 1)
    mine = i < (batch["start"][1:] - batch["start"][:-1]).long()[:, None]
    x = _wide(state["q"], torch.float64).unflatten(1, (hkv, hq // hkv))
    up, down = x.clamp(min=0).sum(2)[row].transpose(1, 2), x.clamp(max=0).sum(2)[row].transpose(1, 2)    # seqs, hkv, n, hd
    b = state["bounds"][table.clamp(min=0)].double().transpose(1, 2)                                      # seqs, hkv, width, 2, hd
    score = torch.matmul(up, b[..., 1, :].transpose(-1, -2)) + torch.matmul(down, b[..., 0, :].transpose(-1, -2))
    score = score.transpose(1, 2)[mine]                                                                   # rows, hkv, width
    at, mypage = torch.arange(table.shape[1], device="cuda"), pos[:, None, None] // page
    there = ((at <= mypage) & (pos >= 0)[:, None, None] & (table[seq] >= 0)[:, None]).expand(score.shape)
    score = torch.where((at < case["first"]) | (at > mypage - case["last"]), POS, score).masked_fill(~there, NEG)
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :case["picks"]]
    ok = torch.gather(there, -1, best)
    picks = torch.where(ok, best, 1 << 40).sort(-1)[0]
    picks = torch.nn.functional.pad(picks, (0, case["picks"] - picks.shape[-1]), value=1 << 40)
    ok = picks < 1 << 40
    # every row and KV head its own pages
    ids = torch.where(ok, table[seq][:, None].expand(-1, hkv, -1).gather(2, picks.clamp(max=table.shape[1] - 1)), 0)
    head = torch.arange(hkv, device="cuda")[None, :, None]
    held = lambda n: _values4(c[n][ids, head].transpose(3, 4), c[n + "e"][ids, head].transpose(3, 4)).flatten(2, 3)  # noqa: E731
    key_pos = (picks[..., None] * page + torch.arange(page, device="cuda")).flatten(2)                    # rows, hkv, keys
    seen = key_pos <= pos[:, None, None]
    zero = torch.zeros((), device="cuda")
    keys, vals = (torch.where(seen[..., None], held(n), zero) for n in "kv")
    q = (_wide(state["q"], torch.float32) / math.sqrt(hd)).unflatten(1, (hkv, hq // hkv))
    m, total, o = _softmax_parts(q, keys, vals, seen[:, :, None])
    out = (o / torch.where(total == 0, torch.ones_like(total), total)).flatten(1, 2)
    return out.to(DTYPES.get(case["dtype"], torch.float32)), torch.where(ok, picks, -1).to(torch.int32)


# -------------------------------------------------------------------- work
def _held(n_values):
    return n_values // 2 + n_values // TILE


def _given(n_values, dtype):
    return {"f32": 4 * n_values, "bf16": 2 * n_values, "f16": 2 * n_values, "tile": 2 * n_values + n_values // TILE}[dtype]


def work(case):
    kind, page, hkv, hd = case["kind"], case["page"], case["hkv"], case["hd"]
    page_bytes = 2 * _held(page * hkv * hd)
    if kind == "fork":
        lens, child = _fork_lengths(case)
        split = sum(1 for n in child if n % page)
        entries = sum(-(-(n + case["new"]) // page) for n in child)
        # a page in and out for every branch that ends inside one; tables in, out and given up; the pages' counts in and out
        return {"bytes": 2 * split * page_bytes * case["layers"] + 4 * entries * 3 + 8 * entries, "flops": 0}
    if kind == "compact":
        live = max(1, int(case["pages"] * case["share"]))
        moved = live * (case["pages"] - live) // case["pages"]
        return {"bytes": 2 * moved * page_bytes * case["layers"] + 8 * case["pages"] + 8 * live * 3 // 2, "flops": 0}
    if kind == "bounds":
        news, lens = _lengths(case)
        pages = sum(-(-n // page) - max(n - q, 0) // page for q, n in zip(news, lens) if n)
        tokens = sum(n - max(n - q, 0) // page * page for q, n in zip(news, lens) if n)
        return {"bytes": _held(tokens * hkv * hd) + 4 * pages * hkv * hd, "flops": 2 * tokens * hkv * hd}
    out = "f32" if case["dtype"] == "tile" else case["dtype"]
    hq = case["hq"]
    if kind == "shared":
        news, lens, of = _shared_lengths(case)
        _, share = _groups(case)
        window = case["window"] or 1 << 40
        keys = read = 0
        low = list(share)
        for b, (q, n) in enumerate(zip(news, lens)):
            keys += sum(min(p + 1, window) for p in range(max(n - q, 0), n))
            if n:
                low[of[b]] = min(low[of[b]], max(0, n - q + 1 - window))
                read += n - max(share[of[b]], n - q + 1 - window)
        read += sum(s - x for s, x in zip(share, low))
        nq = sum(news) * hq * hd
        return {"bytes": 2 * _held(read * hkv * hd) + _given(nq, case["dtype"]) + _given(nq, out), "flops": 4 * keys * hq * hd}
    news, lens = _lengths(case)
    keys = read = scored = bounds = 0
    for q, n in zip(news, lens):
        every = [min(p // page + 1, case["picks"]) * page for p in range(max(n - q, 0), n)]
        keys += sum(every)
        read += min(sum(every), n)
        scored += sum(p // page + 1 for p in range(max(n - q, 0), n))
        bounds += -(-n // page)
    nq = sum(news) * hq * hd
    return {"bytes": 2 * _held(read * hkv * hd) + 4 * bounds * hkv * hd + _given(nq, case["dtype"]) + _given(nq, out)
            + 4 * sum(news) * hkv * case["picks"], "flops": 4 * keys * hq * hd + 4 * scored * hkv * hd}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None                                             # whole numbers, and bytes that are moved
    state = prepare(case, seed)
    return {"bounds": _exact_bounds, "shared": _exact_shared, "sparse": _exact_sparse}[case["kind"]](state, case)


def _exact_values(x):
    if not isinstance(x, tuple):
        return x.double()
    m, e = x
    return m.double() * torch.exp2(e.double() - 15).repeat_interleave(TILE, -1)


def _exact_held(c, name, ids, h, page):
    """The tokens of pages ids of KV head h, one after the other, in 64 bits."""
    d = c[name][ids, h].transpose(1, 2).reshape(len(ids) * page, -1)
    e = c[name + "e"][ids, h].transpose(1, 2).reshape(len(ids) * page, -1)
    code = torch.stack([d % 16, d // 16], -1).flatten(-2)
    size = (code % 8).double()
    size = torch.where(size < 4, size / 2, torch.where(size < 6, size - 2, 2 * size - 8))
    size = size * torch.where(code >= 8, -1.0, 1.0) * torch.exp2(e.double() - 127).repeat_interleave(TILE, -1)
    return torch.where(e.repeat_interleave(TILE, -1) == E_NAN, torch.nan, size)


def _exact_bounds(state, case):
    page, out = case["page"], state["bounds"].double()
    for b, (new, n) in enumerate(zip(*_lengths(case))):
        for p in range(max(n - new, 0) // page, -(-n // page)):
            i = state["batch"]["table"][b, p].long().view(1)
            for h in range(case["hkv"]):
                k = _exact_held(state["cache"], "k", i, h, page)[:n - p * page]
                out[i, h, 0], out[i, h, 1] = k.min(0)[0], k.max(0)[0]
    return out


def _exact_attend(q, k, v, hidden):
    s = (q @ k.T / math.sqrt(q.shape[-1])).masked_fill(hidden, NEG)
    s = torch.where(hidden.all(-1, keepdim=True), 0.0, s)
    return torch.where(hidden.all(-1, keepdim=True), 0.0, torch.softmax(s, -1) @ v)


def _exact_shared(state, case):
    """Every sequence by itself over all of its tokens."""
    c, page, group = state["cache"], case["page"], case["hq"] // case["hkv"]
    q = _exact_values(state["q"])
    out = torch.zeros_like(q)
    news, lens, of = _shared_lengths(case)
    _, share = _groups(case)
    at = 0
    for b, (new, n) in enumerate(zip(news, lens)):
        if new and n:
            ids = state["batch"]["table"][b, :-(-n // page)].long()
            pos, key = torch.arange(n - new, n, device="cuda"), torch.arange(n, device="cuda")
            hidden = key[None] > pos[:, None]
            if case["window"]:
                hidden |= key[None] <= pos[:, None] - case["window"]
            for h in range(case["hkv"]):
                k, v = (_exact_held(c, x, ids, h, page)[:n] for x in "kv")
                for j in range(h * group, (h + 1) * group):
                    out[at:at + new, j] = _exact_attend(q[at:at + new, j], k, v, hidden)
        at += new
    return out


def _exact_sparse(state, case):
    """Row by row, by the definition: the score of every page, the pages that stay, attention over them."""
    news, lens = _lengths(case)
    if sum(news) * case["hkv"] > 10000:
        return None
    c, page, group, picks = state["cache"], case["page"], case["hq"] // case["hkv"], case["picks"]
    q = _exact_values(state["q"])
    out = torch.zeros_like(q)
    chosen = torch.full((sum(news), case["hkv"], picks), -1, dtype=torch.int64, device="cuda")
    t = -1
    for b, (new, n) in enumerate(zip(news, lens)):
        for p in range(n - new, n):
            t += 1
            if p < 0:
                continue
            ids = state["batch"]["table"][b, :p // page + 1].long()
            for h in range(case["hkv"]):
                x = q[t, h * group:(h + 1) * group]
                lo, hi = state["bounds"][ids, h].double().unbind(1)
                score = sum(torch.maximum(y * lo, y * hi).sum(-1) for y in x)
                score[:case["first"]] = POS
                score[max(0, len(ids) - case["last"]):] = POS
                keep = torch.sort(score, descending=True, stable=True)[1][:picks].sort()[0]
                chosen[t, h, :len(keep)] = keep
                key = (keep[:, None] * page + torch.arange(page, device="cuda")).flatten()
                hidden = (key > p)[None].expand(group, -1)
                out[t, h * group:(h + 1) * group] = _exact_attend(x, *(_exact_held(c, m, ids[keep], h, page) for m in "kv"), hidden)
    return out, chosen
