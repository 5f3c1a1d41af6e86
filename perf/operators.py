"""Measured cases of rotary positions, the paged key/value cache held in 4
bits, and the attention that reads it.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges,
``prepare`` makes a case's inputs, ``run`` makes one pass: in plain torch
where ``own`` is false, through ``bfp.rotary`` and ``bfp.kv4`` where it is
true.  ``exact`` is the result in 64 bits and ``work`` what a pass cannot do
without.

The cache holds tiles of 16 values: 16 four-bit E2M1 elements (0, 0.5, 1,
1.5, 2, 3, 4, 6 and their negatives) and one exponent byte E, value =
element * 2^(E-127), E = 255 for a tile with a NaN or an infinity in it.  The
exponent is the smallest at which the tile's largest element rounds to at
most 6.  A page holds ``page`` tokens of every KV head, tile by tile: k, v
(pages, heads, hd/16, page, 8) bytes, the lower half of a byte first, and ke,
ve (pages, heads, hd/16, page).
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
NEG = float("-inf")


# ------------------------------------------------------------------- cases
def listed():
    return [
        # the angles of the framework's own model: 2048 positions, heads of 64, base 10000, nothing scaled
        {"name": "table_short", "kind": "table", "n_pos": 2048, "rot": 64, "base": 10000.0, "scaling": "none",
         "factor": 1.0, "orig": 2048},
        # the angles of a context stretched 16 times, frequencies blended by how often they turn
        {"name": "table_long", "kind": "table", "n_pos": 131072, "rot": 128, "base": 500000.0, "scaling": "parts",
         "factor": 16.0, "orig": 8192},
        # one step of 64 sequences: the queries of one layer
        {"name": "rope_step", "kind": "rope", "rows": 64, "heads": 9, "hd": 64, "rot": 64, "n_pos": 2048,
         "interleaved": False, "dtype": "bf16", "fused": 0},
        # a prompt's queries inside the rows of a joined Q|K|V product, half of each head rotated, neighbours paired
        {"name": "rope_prompt", "kind": "rope", "rows": 4999, "heads": 32, "hd": 128, "rot": 64, "n_pos": 16384,
         "interleaved": True, "dtype": "f16", "fused": 16},
        # one step of 64 sequences as the matvec engine leaves it: Q, K and V as 16-bit tiles
        {"name": "append_step", "kind": "append", "seqs": 64, "new": 1, "ctx": 2048, "hq": 9, "hkv": 3, "hd": 64,
         "rot": 64, "page": 16, "interleaved": False, "dtype": "tile"},
        # three ragged prompts at once
        {"name": "append_prompt", "kind": "append", "seqs": 3, "new": 2500, "ctx": 4096, "hq": 32, "hkv": 8,
         "hd": 128, "rot": 128, "page": 64, "interleaved": False, "dtype": "bf16"},
        # the next token of one chat at the end of the framework's context: latency
        {"name": "token_single", "kind": "attend", "seqs": 1, "new": 1, "ctx": 2047, "hq": 9, "hkv": 3, "hd": 64,
         "page": 16, "dtype": "tile", "window": 0},
        # the next token of 64 sequences
        {"name": "token_batch", "kind": "attend", "seqs": 64, "new": 1, "ctx": 2048, "hq": 9, "hkv": 3, "hd": 64,
         "page": 16, "dtype": "bf16", "window": 0},
        # the next token of a few very long documents
        {"name": "token_long", "kind": "attend", "seqs": 8, "new": 1, "ctx": 131072, "hq": 32, "hkv": 8, "hd": 128,
         "page": 64, "dtype": "bf16", "window": 0},
        # a handful of short prompts in full precision
        {"name": "prompt_short", "kind": "attend", "seqs": 5, "new": 300, "ctx": 300, "hq": 9, "hkv": 3, "hd": 64,
         "page": 32, "dtype": "f32", "window": 0},
        # a piece of a long prompt behind what the cache holds already, looking back 16384 tokens
        {"name": "prompt_piece", "kind": "attend", "seqs": 1, "new": 509, "ctx": 32768, "hq": 16, "hkv": 4, "hd": 96,
         "page": 64, "dtype": "f16", "window": 16384},
        # two long prompts
        {"name": "prompt_long", "kind": "attend", "seqs": 2, "new": 8192, "ctx": 8192, "hq": 32, "hkv": 8, "hd": 128,
         "page": 64, "dtype": "bf16", "window": 0},
    ]


def _log_int(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    return min(max(v, lo), hi)


def draw(rng):
    kind = rng.choice(["table", "rope", "append", "append", "attend", "attend", "attend"])
    if kind == "table":
        return {"kind": kind, "n_pos": _log_int(rng, 64, 131072), "rot": rng.randrange(16, 130, 2),
                "base": rng.choice([10000.0, 100000.0, 500000.0]),
                "scaling": rng.choice(["none", "linear", "ntk", "parts", "bands"]),
                "factor": rng.choice([2.0, 4.0, 8.0, 16.0]), "orig": rng.choice([2048, 4096, 8192])}
    hd = rng.choice([32, 48, 64, 64, 80, 96, 112, 128, 128, 192, 256])
    page = rng.choice([16, 32, 64, 128])
    rot = rng.choice([hd, hd, hd // 2, hd // 4 + 2])
    inter = rng.random() < 0.5
    if kind == "rope":
        rows = _log_int(rng, 1, 8192)
        heads = min(rng.randint(1, 32), max(1, (20 << 20) // (rows * hd)))
        return {"kind": kind, "rows": rows, "heads": heads, "hd": hd, "rot": rot,
                "n_pos": _log_int(rng, 128, 32768), "interleaved": inter,
                "dtype": rng.choice(["bf16", "f16", "f32", "tile"]), "fused": rng.choice([0, 0, 2, 7])}
    hkv = rng.randint(1, 8)
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32", "tile"])
    if kind == "append":
        seqs = _log_int(rng, 1, 64)
        new = rng.choice([1, 1, _log_int(rng, 2, max(2, 8000 // seqs))])
        new = min(new, max(1, (6 << 20) // (seqs * hkv * hd)))
        return {"kind": kind, "seqs": seqs, "new": new, "ctx": new + _log_int(rng, 1, 4096), "hq": hq, "hkv": hkv,
                "hd": hd, "rot": rot, "page": page, "interleaved": inter, "dtype": dtype}
    seqs = _log_int(rng, 1, 64)
    # (a) one token a sequence, (b) a few, as a draft is checked, (c) prompts and pieces of them
    new = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 4096)])
    most = (1 << 30) // (seqs * new * hq)                      # a pass's scores
    ctx = new + min(_log_int(rng, 1, 65536), most, (1 << 29) // (seqs * hkv * hd))
    if new > 8:
        seqs = max(1, min(seqs, (1 << 31) // (new * hq * ctx)))
    return {"kind": kind, "seqs": seqs, "new": new, "ctx": ctx, "hq": hq, "hkv": hkv, "hd": hd, "page": page,
            "dtype": dtype, "window": rng.choice([0, 0, 0, _log_int(rng, 1, 4096)])}


def _lengths(case):
    """How many new tokens each sequence has and how long it is with them:
    ragged, the first the longest; past two sequences one that is empty.
    From the case alone, so that work() knows them."""
    n, new, ctx = case["seqs"], case["new"], case["ctx"]
    news, lens = [], []
    for b in range(n):
        part = 1.0 - 0.61 * ((b * 0.6180339887) % 1.0) if b else 1.0
        q = max(1, int(new * part))
        news.append(q)
        lens.append(max(q, int(ctx * part)))
    if n > 2:
        news[-1], lens[-1] = (1 if new == 1 else 0), 0
    return news, lens


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _tile16(v):
    """16-bit tiles of float32 values: (m int16, e int8), v ~ m 2^(e-15)."""
    t = v.double().unflatten(-1, (-1, TILE))
    e = torch.frexp(t.abs().amax(-1))[1].clamp(-127, 127)
    m = torch.round(torch.ldexp(t, (15 - e).unsqueeze(-1))).clamp(-32768, 32767)
    return m.flatten(-2).to(torch.int16), e.to(torch.int8)


def _typed(v, dtype):
    return _tile16(v) if dtype == "tile" else v.to(DTYPES[dtype])


def _cos_sin(n_pos, rot, base=10000.0):
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(n_pos, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def _batch(case, g):
    """The batch as the program describes it: where each sequence's new rows
    start, its length with them, and its pages in the order of its tokens."""
    news, lens = _lengths(case)
    page = case["page"]
    need = [-(-n // page) for n in lens]
    width = max(max(need), 1)
    pages = sum(need) + 3                                      # some that no sequence has
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([sum(need[:b]) for b in range(len(need))], device="cuda")
    at = torch.arange(width, device="cuda")
    held = at[None] < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(held, ids[(first[:, None] + at).clamp(max=pages - 1)], -1).to(torch.int32)
    cu = torch.tensor([0] + news, device="cuda").cumsum(0).to(torch.int32)
    return {"table": table, "cu": cu, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
            "max_q": max(news), "max_len": max(lens), "rows": sum(news), "pages": pages, "spare": ids[-1].long()}


def _empty_cache(case, pages):
    """Pages as they are found: whatever bytes were there."""
    g = _gen(pages)
    shape = (pages, case["hkv"], case["hd"] // TILE, case["page"])
    r = lambda *n: torch.randint(0, 256, (*shape, *n), generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
    return {"k": r(TILE // 2), "ke": r(), "v": r(TILE // 2), "ve": r()}


def _filled_cache(case, batch, g):
    """Keys with a few strong channels, as rotated keys have them, and
    plainer values; slots behind a sequence's end hold other bytes."""
    c = _empty_cache(case, batch["pages"])
    hd, hkv, page = case["hd"], case["hkv"], case["page"]
    strong = 1.0 + 3.0 * (torch.rand(hkv, 1, hd, generator=g, device="cuda") > 0.95)
    step = max(1, (1 << 27) // (hkv * page * hd))
    for p in range(0, batch["pages"], step):
        n = min(step, batch["pages"] - p)
        for data, exp, like in (("k", "ke", strong), ("v", "ve", 1.0)):
            d, e = _quant4(_randn(g, n, hkv, page, hd) * like)
            c[data][p:p + n], c[exp][p:p + n] = d.transpose(2, 3), e.transpose(2, 3)
    pos = torch.arange(batch["table"].shape[1] * page, device="cuda").view(1, -1, page)
    stale = (pos >= batch["lens"][:, None, None].long()) & (batch["table"][:, :, None] >= 0)
    b, w, off = stale.nonzero(as_tuple=True)
    ids = batch["table"][b, w].long()
    for name in ("k", "ke", "v", "ve"):
        old = c[name][ids, :, :, off]
        c[name][ids, :, :, off] = torch.randint(0, 256, old.shape, generator=g, device="cuda", dtype=torch.uint8)
    return c


def prepare(case, seed):
    kind = case["kind"]
    if kind == "table":
        # nothing in a table is random but where it starts
        return {"case": case, "first": seed % 64}
    g = _gen(seed)
    if kind == "rope":
        rows, heads, hd = case["rows"], case["heads"], case["hd"]
        x = _typed(_randn(g, rows, heads + case["fused"], hd), case["dtype"])
        x = tuple(t[:, :heads] for t in x) if case["dtype"] == "tile" else x[:, :heads]
        pos = torch.randint(0, case["n_pos"], (rows,), generator=g, device="cuda", dtype=torch.int32)
        return {"case": case, "x": x, "pos": pos, "cs": _cos_sin(case["n_pos"], case["rot"])}
    batch = _batch(case, g)
    if kind == "append":
        hq, hkv = case["hq"], case["hkv"]
        x = _typed(_randn(g, batch["rows"], hq + 2 * hkv, case["hd"]), case["dtype"])
        part = lambda a, b: tuple(t[:, a:b] for t in x) if case["dtype"] == "tile" else x[:, a:b]  # noqa: E731
        n_pos = batch["table"].shape[1] * case["page"]
        return {"case": case, "batch": batch, "cache": _empty_cache(case, batch["pages"]), "q": part(0, hq),
                "k": part(hq, hq + hkv), "v": part(hq + hkv, hq + 2 * hkv), "cs": _cos_sin(n_pos, case["rot"])}
    q = _typed(_randn(g, batch["rows"], case["hq"], case["hd"]), case["dtype"])
    return {"case": case, "batch": batch, "cache": _filled_cache(case, batch, g), "q": q}


# --------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["kind"] == "table":
        inv, mscale = _frequencies(case)
        pos = torch.arange(state["first"], state["first"] + case["n_pos"], dtype=torch.float64, device="cuda")
        a = pos[:, None] * inv
        return (torch.stack([a.cos(), a.sin()], -1) * mscale).float()
    if case["kind"] == "rope":
        x = _wide(state["x"], torch.float32)
        y = _rotate(x, state["cs"][state["pos"].long()], case["interleaved"])
        return y.to(DTYPES.get(case["dtype"], torch.float32))
    if case["kind"] == "append":
        return _append(state, case)
    return _attend(state, case)


def _run_own(state, case):
    from bfp import kv4, rotary
    if case["kind"] == "table":
        inv, mscale = rotary.rope_freqs(case["rot"], case["base"], case["scaling"], case["factor"], case["orig"])
        return rotary.rope_table(inv, case["n_pos"], mscale, first=state["first"])
    if case["kind"] == "rope":
        return rotary.rope(state["x"], state["pos"], state["cs"], interleaved=case["interleaved"])
    if "handle" not in state:      # what a serving loop keeps from call to call
        c, b = state["cache"], state["batch"]
        state["handle"] = (kv4.Fp4Cache.from_buffers(c["k"], c["ke"], c["v"], c["ve"]),
                           kv4.Batch(b["table"], b["cu"], b["lens"], max_q=b["max_q"], max_len=b["max_len"]))
    cache, batch = state["handle"]
    if case["kind"] == "append":
        q = cache.append(batch, state["k"], state["v"], state["cs"], interleaved=case["interleaved"], q=state["q"])
        k, v = cache.read(batch, state["batch"]["rows"], dtype=torch.bfloat16)
        return q, k, v
    return cache.attend(batch, state["q"], window=case["window"])


def _frequencies(case):
    """Angles per position and the factor on cos and sin, in 64 bits.
    linear: positions divided by the factor.  ntk: the base raised so that
    the slowest pair turns `factor` times slower.  parts: pairs that turn
    more than 32 times over the original context stay, those that turn less
    than once are divided, a straight line in the pair's index between; cos
    and sin grow by 0.1 ln(factor) + 1.  bands: the same by wavelength, from
    a quarter of the original context to all of it, a straight line in the
    turns between."""
    rot, base, kind, f, orig = case["rot"], case["base"], case["scaling"], case["factor"], case["orig"]
    j = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot
    if kind == "ntk":
        base = base * f ** (rot / (rot - 2))
    inv = base ** -j
    if kind == "linear":
        return inv / f, 1.0
    if kind == "parts":
        low = max(math.floor(rot * math.log(orig / (32 * 2 * math.pi)) / (2 * math.log(base))), 0)
        high = min(math.ceil(rot * math.log(orig / (2 * math.pi)) / (2 * math.log(base))), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64, device="cuda") - low) / max(high - low, 0.001)).clamp(0, 1)
        return inv / f * ramp + inv * (1 - ramp), 0.1 * math.log(f) + 1.0
    if kind == "bands":
        turns = orig * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return inv * keep + inv / f * (1 - keep), 1.0
    return inv, 1.0


def _wide(x, dtype):
    """Values of a tensor, or of 16-bit tiles, in a wider type (exact)."""
    if isinstance(x, tuple):
        m, e = x
        return torch.ldexp(m.to(dtype).unflatten(-1, (-1, TILE)), (e.to(torch.int32) - 15).unsqueeze(-1)).flatten(-2)
    return x.to(dtype)


def _rotate(x, cs, interleaved):
    """The first 2 * cs.shape[1] values of every head (rows, heads, hd)."""
    r = 2 * cs.shape[-2]
    c, s = cs[..., 0].to(x.dtype)[:, None], cs[..., 1].to(x.dtype)[:, None]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    y, z = a * c - b * s, b * c + a * s
    y = torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1)
    return torch.cat([y, x[..., r:]], -1)


def _quant4(v):
    """Values (..., hd) to the cache's tiles: bytes (..., hd/16, 8) and
    exponent bytes (..., hd/16)."""
    t = v.unflatten(-1, (-1, TILE))
    amax = t.abs().amax(-1)
    good = amax.isfinite()
    amax = torch.where(good, amax, torch.zeros_like(amax))
    f, x = torch.frexp(amax)                                   # amax = f 2^x, f in [0.5, 1)
    e = torch.where(amax > 0, x - 3 + (f >= 0.875).int(), torch.zeros_like(x)).clamp(E_MIN, E_MAX)
    t = torch.where(good.unsqueeze(-1), torch.ldexp(t, -e.unsqueeze(-1)), torch.zeros_like(t))
    a = t.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(a.dtype)
    a = (torch.round(a / step) * step).clamp(max=6)
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | ((t < 0).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.where(good, e + 127, E_NAN).to(torch.uint8)


def _values4(data, exp):
    """Tiles (..., hd/16, 8) and their exponents as float32 (..., hd)."""
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=data.device)
    v = lut[torch.stack([data & 15, data >> 4], -1).flatten(-2).int()]
    scale = torch.where(exp == E_NAN, torch.nan, torch.ldexp(torch.ones_like(exp, dtype=torch.float32), exp.int() - 127))
    return (v * scale.unsqueeze(-1)).flatten(-2)


def _slots(batch, page):
    """Of every new row: its sequence, its position, its page and its slot there."""
    cu, lens = batch["cu"].long(), batch["lens"].long()
    row = torch.arange(batch["rows"], device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    pos = lens[seq] - cu[seq + 1] + row
    ok = pos >= 0
    at = pos.clamp(min=0)
    return seq, pos, batch["table"][seq, at // page].long(), at % page, ok


def _append(state, case):
    """Rotated in 64 bits: a value next to a border between two elements
    would go to either otherwise."""
    batch, c = state["batch"], state["cache"]
    seq, pos, page, off, ok = _slots(batch, case["page"])
    cs = state["cs"][pos.clamp(min=0)]
    k = _rotate(_wide(state["k"], torch.float64), cs, case["interleaved"])
    v = _wide(state["v"], torch.float32)
    q = _rotate(_wide(state["q"], torch.float32), cs, case["interleaved"])
    kd, ke = _quant4(k)
    vd, ve = _quant4(v)
    at = torch.where(ok, page, batch["spare"])      # a row without a slot goes to a page that nobody has
    here = (at, slice(None), slice(None), off)
    c["k"][here], c["ke"][here], c["v"][here], c["ve"][here] = kd, ke, vd, ve
    w, zero = ok[:, None, None], torch.zeros((), device="cuda")
    rk = torch.where(w, _values4(c["k"][here], c["ke"][here]), zero)
    rv = torch.where(w, _values4(c["v"][here], c["ve"][here]), zero)
    q = torch.where(w, q, zero)
    return q.to(DTYPES.get(case["dtype"], torch.float32)), rk.bfloat16(), rv.bfloat16()


def _held_by(ids, data, exp):
    """The tiles of the pages `ids` (seqs, width), token after token."""
    return data[ids].permute(0, 2, 1, 4, 3, 5).flatten(2, 3), exp[ids].permute(0, 2, 1, 4, 3).flatten(2, 3)


def _attend(state, case):
    """Every sequence padded to the longest, float32 throughout."""
    batch, c, page = state["batch"], state["cache"], case["page"]
    hq, hkv, hd, n = case["hq"], case["hkv"], case["hd"], batch["max_q"]
    table, cu, lens = batch["table"].long(), batch["cu"].long(), batch["lens"].long()
    seqs, width = table.shape
    ids = table.clamp(min=0)
    key = torch.arange(width * page, device="cuda")
    there = (key[None] < lens[:, None])[:, None, :, None]                           # seqs, 1, keys, 1
    zero = torch.zeros((), device="cuda")
    k = torch.where(there, _values4(*_held_by(ids, c["k"], c["ke"])), zero)         # seqs, hkv, keys, hd
    v = torch.where(there, _values4(*_held_by(ids, c["v"], c["ve"])), zero)
    i = torch.arange(n, device="cuda")
    news = cu[1:] - cu[:-1]
    row = (cu[:-1, None] + i[None]).clamp(max=batch["rows"] - 1)                    # seqs, n
    q = _wide(state["q"], torch.float32)[row]                                       # seqs, n, hq, hd
    q = q.unflatten(2, (hkv, hq // hkv)).permute(0, 2, 3, 1, 4).flatten(2, 3)       # seqs, hkv, group * n, hd
    pos = (lens - news)[:, None] + i[None]
    seen = key[None, None] <= pos[:, :, None]
    if case["window"]:
        seen &= key[None, None] > pos[:, :, None] - case["window"]
    s = torch.matmul(q, k.transpose(-1, -2)).unflatten(2, (hq // hkv, n)) / math.sqrt(hd)
    s = s.masked_fill_(~seen[:, None, None], NEG)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == NEG, zero, m)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (hq // hkv, n))
    o = o / torch.where(total == 0, torch.ones_like(total), total)                  # seqs, hkv, group, n, hd
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)
    mine = i[None] < news[:, None]
    out = torch.zeros(batch["rows"], hq, hd, device="cuda")
    out[row[mine]] = o[mine]
    return out.to(DTYPES.get(case["dtype"], torch.float32))


# -------------------------------------------------------------------- work
def _held(n_values):
    return n_values // 2 + n_values // TILE


def _given(n_values, dtype):
    return {"f32": 4 * n_values, "bf16": 2 * n_values, "f16": 2 * n_values, "tile": 2 * n_values + n_values // TILE}[dtype]


def work(case):
    kind = case["kind"]
    if kind == "table":
        # a cosine and a sine in 64 bits: some 40 operations each
        n = case["n_pos"] * case["rot"] // 2
        return {"bytes": 8 * n, "flops": 80 * n}
    out = "f32" if case["dtype"] == "tile" else case["dtype"]
    if kind == "rope":
        n, rows = case["rows"] * case["heads"] * case["hd"], case["rows"]
        angles = min(rows, case["n_pos"]) * case["rot"] * 4
        return {"bytes": _given(n, case["dtype"]) + _given(n, out) + angles + 4 * rows,
                "flops": 3 * rows * case["heads"] * case["rot"]}
    news, lens = _lengths(case)
    rows = sum(news)
    nq, nkv = rows * case["hq"] * case["hd"], rows * case["hkv"] * case["hd"]
    if kind == "append":
        # in and out, the cache's rows written and read back once, the values read back
        return {"bytes": _given(nq + 2 * nkv, case["dtype"]) + _given(nq, out) + 4 * _held(nkv) + 4 * nkv
                + rows * case["rot"] * 4, "flops": 3 * rows * (case["hq"] + case["hkv"]) * case["rot"] + 8 * nkv}
    keys = read = 0
    for q, n in zip(news, lens):
        w = case["window"] or n + q
        first = max(n - q, 0)
        keys += sum(min(p + 1, w) for p in range(first, n))
        read += min(n, q + w - 1)
    return {"bytes": 2 * _held(read * case["hkv"] * case["hd"]) + _given(nq, case["dtype"]) + _given(nq, out),
            "flops": 4 * keys * case["hq"] * case["hd"]}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    state = prepare(case, seed)
    return {"table": _exact_table, "rope": _exact_rope, "append": _exact_append, "attend": _exact_attend}[case["kind"]](state, case)


def _exact_table(state, case):
    rot, base, f, orig = case["rot"], case["base"], case["factor"], case["orig"]
    mscale, inv = 1.0, []
    for j in range(rot // 2):
        b = base * f ** (rot / (rot - 2)) if case["scaling"] == "ntk" else base
        w = 1.0 / b ** (2 * j / rot)
        if case["scaling"] == "linear":
            w /= f
        if case["scaling"] == "parts":
            mscale = 1.0 + 0.1 * math.log(f)
            at = lambda turns: rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(math.floor(at(32)), 0), min(math.ceil(at(1)), rot - 1)
            share = min(max((j - lo) / (hi - lo if hi != lo else 0.001), 0.0), 1.0)
            w = w * (1 - share) + w / f * share
        if case["scaling"] == "bands":
            length = 2 * math.pi / w
            if length > orig:
                w /= f
            elif length >= orig / 4:
                share = (orig / length - 1) / 3
                w = (1 - share) * w / f + share * w
        inv.append(w)
    inv = torch.tensor(inv, dtype=torch.float64, device="cuda")
    a = torch.outer(torch.arange(case["n_pos"], dtype=torch.float64, device="cuda") + state["first"], inv)
    return torch.stack([torch.cos(a) * mscale, torch.sin(a) * mscale], 2)


def _exact_values(x):
    if not isinstance(x, tuple):
        return x.double()
    m, e = x
    return m.double() * torch.exp2(e.double() - 15).repeat_interleave(TILE, -1)


def _exact_turn(x, cs, interleaved):
    """As complex numbers."""
    r = 2 * cs.shape[1]
    pairs = x[..., :r].unflatten(-1, (r // 2, 2)) if interleaved else x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.view_as_complex(cs.double().contiguous())[:, None]
    y = torch.view_as_real(z)
    return torch.cat([(y if interleaved else y.transpose(-1, -2)).flatten(-2), x[..., r:]], -1)


def _exact_rope(state, case):
    return _exact_turn(_exact_values(state["x"]), state["cs"][state["pos"].long()], case["interleaved"])


def _exact_rows(state, case):
    news, lens = _lengths(case)
    return [(b, n - q + i) for b, (q, n) in enumerate(zip(news, lens)) for i in range(q)]


def _exact_append(state, case):
    where = torch.tensor([p for _, p in _exact_rows(state, case)], device="cuda")
    ok = (where >= 0)[:, None, None]
    cs = state["cs"][where.clamp(min=0)]
    turn = lambda x: _exact_turn(_exact_values(x), cs, case["interleaved"])  # noqa: E731

    def held(x):
        t = x.unflatten(-1, (-1, TILE))
        size = t.abs().amax(-1, keepdim=True)
        scale = torch.exp2(torch.floor(torch.log2(size.clamp(min=1e-300))) - 2)
        scale = torch.where(size >= 7 * scale, 2 * scale, scale)
        grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
        edge = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5], dtype=torch.float64, device="cuda")
        a = (t / scale).abs()
        # a value on an edge goes to the even element: down at the first, third, fifth and seventh
        i = torch.searchsorted(edge, a.contiguous())
        on = (i < 7) & (edge[i.clamp(max=6)] == a) & (i % 2 == 1)
        return (grid[(i + on).clamp(max=7)] * t.sign() * scale).flatten(-2)
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    return tuple(torch.where(ok, y, zero) for y in (turn(state["q"]), held(turn(state["k"])), held(_exact_values(state["v"]))))


def _exact_attend(state, case):
    batch, c = state["batch"], state["cache"]
    hq, hkv, hd, page = case["hq"], case["hkv"], case["hd"], case["page"]
    group = hq // hkv
    q = _exact_values(state["q"])
    out = torch.zeros(batch["rows"], hq, hd, dtype=torch.float64, device="cuda")
    news, lens = _lengths(case)
    at = 0

    def held(data, exp, ids, n, h):
        d = data[ids, h].transpose(1, 2).reshape(len(ids) * page, -1)[:n]
        e = exp[ids, h].transpose(1, 2).reshape(len(ids) * page, -1)[:n]
        code = torch.stack([d % 16, d // 16], -1).flatten(-2)
        size = (code % 8).double()
        size = torch.where(size < 4, size / 2, torch.where(size < 6, size - 2, 2 * size - 8))
        size = size * torch.where(code >= 8, -1.0, 1.0) * torch.exp2(e.double() - 127).repeat_interleave(TILE, -1)
        return torch.where(e.repeat_interleave(TILE, -1) == E_NAN, torch.nan, size)
    for b, (n_q, n) in enumerate(zip(news, lens)):
        if n_q and n:
            ids = batch["table"][b, :-(-n // page)].long()
            pos = torch.arange(n - n_q, n, device="cuda")
            key = torch.arange(n, device="cuda")
            hidden = key[None] > pos[:, None]
            if case["window"]:
                hidden |= key[None] <= pos[:, None] - case["window"]
            for h in range(hkv):
                k, v = held(c["k"], c["ke"], ids, n, h), held(c["v"], c["ve"], ids, n, h)
                for j in range(h * group, (h + 1) * group):
                    s = (q[at:at + n_q, j] @ k.T / math.sqrt(hd)).masked_fill(hidden, NEG)
                    out[at:at + n_q, j] = torch.softmax(s, -1) @ v
        at += n_q
    return out
