"""Plain 64-bit implementations of the rotary and 4-bit-cache operators for
the tests, on the CPU (numpy; nothing here comes from the package)."""
import math

import numpy as np

GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
MIDS = (GRID[1:] + GRID[:-1]) / 2
E_MIN, E_MAX, E_NAN = -100, 100, 255


def encode(v):
    """Tiles of 16 along the last axis: (codes 0..15, exponent bytes)."""
    t = np.asarray(v, np.float64).reshape(*v.shape[:-1], -1, 16)
    top = np.abs(t).max(-1)
    bad = ~np.isfinite(t).all(-1)
    e = np.zeros(top.shape, int)
    for i in np.ndindex(top.shape):
        if bad[i] or top[i] == 0:
            continue
        x = E_MIN
        while x < E_MAX and top[i] >= 7 * 2.0 ** x:   # 7 is where an element rounds past 6
            x += 1
        e[i] = x
    a = np.abs(np.where(bad[..., None], 0, t)) * 2.0 ** -e[..., None].astype(float)
    # nearest element, a tie to the even code
    code = np.searchsorted(MIDS, a)                   # MIDS[code-1] < a <= MIDS[code]
    tie = (code < 7) & (np.append(MIDS, np.inf)[code] == a) & (code % 2 == 1)
    code = np.minimum(code + tie, 7)
    code = code + 8 * (np.signbit(t) & (code > 0) & ~bad[..., None])
    return code.reshape(v.shape), np.where(bad, E_NAN, e + 127)


def value(codes, exps):
    c = np.asarray(codes)
    v = GRID[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.where(exps == E_NAN, np.nan, 2.0 ** (exps.astype(float) - 127))
    return (v.reshape(*c.shape[:-1], c.shape[-1] // 16, 16) * s[..., None]).reshape(c.shape)


def quant4(v):
    return value(*encode(np.asarray(v, np.float64)))


def freqs(rot, base=10000.0, scaling="none", factor=1.0, orig=0):
    out = []
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    at = lambda turns: rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    for j in range(rot // 2):
        w = 1.0 / base ** (2 * j / rot)
        if scaling == "linear":
            w /= factor
        if scaling == "parts":
            lo, hi = max(math.floor(at(32)), 0), min(math.ceil(at(1)), rot - 1)
            x = min(max((j - lo) / max(hi - lo, 0.001), 0), 1)
            w = w * (1 - x) + w / factor * x
        if scaling == "bands":
            x = min(max((orig * w / (2 * math.pi) - 1) / 3, 0), 1)
            w = w * x + w / factor * (1 - x)
        out.append(w)
    return np.array(out), (0.1 * math.log(factor) + 1 if scaling == "parts" else 1.0)


def angles(n_pos, rot, base=10000.0, first=0):
    a = np.outer(np.arange(first, first + n_pos, dtype=np.float64), freqs(rot, base)[0])
    return np.stack([np.cos(a), np.sin(a)], -1)


def rotate(x, pos, table, interleaved=False):
    """x (rows, heads, hd) by table[pos]; NaN where pos is not in it."""
    x = np.asarray(x, np.float64)
    h = table.shape[1]
    ok = (pos >= 0) & (pos < len(table))
    cs = np.where(ok[:, None, None], np.asarray(table, np.float64)[np.where(ok, pos, 0)], np.nan)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    y = x.copy()
    ia, ib = (np.arange(0, 2 * h, 2), np.arange(1, 2 * h, 2)) if interleaved else (np.arange(h), np.arange(h, 2 * h))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def attend(q, keys, values, start, lens, group, scale, window=0, there=None):
    """q (rows, heads, hd); keys, values: per sequence (tokens, kv heads,
    hd) float64, at least lens[b] tokens.  there: per sequence, which tokens
    have a page.  Returns (out, absolute weight of the values, largest score
    sum): the last two are what the error bounds are made of."""
    out, weight, big = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    for b in range(len(lens)):
        n = start[b + 1] - start[b]
        for i in range(n):
            p = max(lens[b], 0) - n + i
            t = start[b] + i
            see = np.arange(max(p + 1 - window, 0) if window else 0, p + 1)
            see = see[see < len(keys[b])]
            if there is not None:
                see = see[there[b][see]]
            if not len(see):
                continue
            for h in range(q.shape[1]):
                k, v = keys[b][see, h // group], values[b][see, h // group]
                s = (k * q[t, h]).sum(-1) * scale
                big[t, h] = (np.abs(k * q[t, h]).sum(-1) * abs(scale)).max()
                w = np.exp(s - s.max())
                out[t, h] = w @ v / w.sum()
                weight[t, h] = w @ np.abs(v) / w.sum()
    return out, weight, big


def attend_bound(out, weight, big, n_keys, hd, out_half, p_half):
    """How far float32 arithmetic on exact products may be off.  A score is
    a sum of at most 3 hd terms (a query in three pieces), its scaling and
    the subtraction of the maximum three roundings, taken as 2^-23 each
    (the matrix cores may cut); the exponential 2^-22.  That changes a
    probability relatively by d, and the quotient by 2 d; the two sums over
    the keys add 2^-23 a term, the probabilities' own rounding p_half, the
    result's out_half of its value."""
    d = big[..., None] * (3 * hd + 4) * 2.0 ** -23 + 2.0 ** -21
    return (2 * d + (2 * n_keys + 16) * 2.0 ** -23 + p_half) * weight + out_half * np.abs(out) + 1e-38


def attend_all(q, keys, values, start, lens, group, scale, window=0, there=None):
    """attend() a head at a time, for many rows or long contexts."""
    out, weight, big = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    for b in range(len(lens)):
        rows = slice(start[b], start[b + 1])
        n, m = start[b + 1] - start[b], len(keys[b])
        p = (max(lens[b], 0) - n + np.arange(n))[:, None]
        at = np.arange(m)[None]
        see = (at <= p) & ((at > p - window) if window else True) & (True if there is None else there[b][None, :m])
        some = see.any(-1)
        if not some.any():
            continue
        for h in range(q.shape[1]):
            k, v, x = keys[b][:, h // group], values[b][:, h // group], q[rows, h]
            s = np.where(see, x @ k.T * scale, -np.inf)
            w = np.exp(s - np.where(some, s.max(-1, initial=-np.inf), 0)[:, None])
            w /= np.where(some, w.sum(-1), 1)[:, None]
            out[rows, h], weight[rows, h] = w @ v, w @ np.abs(v)
            big[rows, h] = np.where(see, np.abs(x) @ np.abs(k).T * abs(scale), 0).max(-1, initial=0)
    return out, weight, big
