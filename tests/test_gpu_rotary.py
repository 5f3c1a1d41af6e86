"""Rotary tables and rotations on the GPU against plain 64-bit numpy."""
import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}   # half a step, of the value


def _dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _say(*a):
    print("[rotary]", *a, flush=True)


@pytest.mark.parametrize("rot,n_pos,first,scaling", [
    (64, 100, 0, "none"), (2, 1, 0, "none"), (34, 333, 131000, "linear"), (128, 65, 2 ** 31 - 65, "none"),
    (512, 3, 7, "parts"), (96, 1000, 100000, "bands"), (16, 257, 5, "ntk")])
def test_table(gpu, rot, n_pos, first, scaling):
    from bfp import rotary
    inv, ms = rotary.rope_freqs(rot, 10000.0, scaling, 8.0, 2048)
    got = rotary.rope_table(inv, n_pos, ms, first=first).cpu().numpy()
    # the same product position * frequency, then cos and sin within a few ulps of it
    a = np.arange(first, first + n_pos, dtype=np.float64)[:, None] * inv[None]
    want = np.stack([np.cos(a), np.sin(a)], -1) * ms
    assert got.shape == want.shape
    # float64 cos and sin 2^-50, one rounding to float32
    assert (np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -48 + 2.0 ** -149).all()


def test_table_into_and_empty(gpu):
    import torch
    from bfp import rotary
    inv, _ = rotary.rope_freqs(64)
    out = torch.full((10, 32, 2), 7.0, device="cuda")
    assert rotary.rope_table(inv, 10, out=out) is out
    assert torch.equal(out, rotary.rope_table(inv, 10)) and float(out[0, 0, 0]) == 1.0
    assert rotary.rope_table(inv, 0).shape == (0, 32, 2)
    with pytest.raises(ValueError):
        rotary.rope_table(inv, 11, out=out)


CASES = [  # rows, heads, hd, rot, interleaved, type in, type out, extra heads (stride), offset
    (1, 1, 64, 64, False, "f32", None, 0, 0),
    (5, 9, 64, 64, False, "bf16", None, 0, 0),
    (7, 3, 64, 64, True, "bf16", None, 2, 0),
    (33, 4, 128, 64, True, "f16", None, 4, 0),
    (33, 4, 128, 64, False, "f16", "f32", 4, 0),
    (3, 2, 96, 34, False, "f32", None, 0, 0),      # half 17: value by value
    (3, 2, 96, 34, True, "f32", "bf16", 0, 0),
    (4, 3, 20, 20, False, "bf16", None, 0, 0),
    (4, 3, 20, 6, True, "f16", None, 1, 0),
    (2, 5, 7, 4, False, "f32", None, 0, 0),        # odd width
    (6, 2, 64, 64, False, "f32", None, 0, 1),      # not 16-byte aligned
    (6, 2, 64, 32, True, "bf16", None, 0, 3),
    (5, 3, 64, 64, False, "tile", None, 0, 0),
    (5, 3, 64, 32, True, "tile", "bf16", 1, 0),
    (9, 1, 256, 256, False, "tile", "f16", 0, 0),
    (300, 17, 80, 40, False, "bf16", None, 0, 0),
]


def _typed(rng, rows, heads, hd, kind, extra, off):
    import torch
    full = rng.standard_normal((rows, heads + extra, hd)).astype(np.float32)
    if kind == "tile":
        from oracle import bfp_sim as sim
        m, e = sim.tile_quantize(full.astype(np.float64).reshape(-1))
        val = np.asarray(sim.tile_decode(m, e)).reshape(full.shape)
        m = torch.from_numpy(np.ascontiguousarray(np.asarray(m, np.int16).reshape(full.shape))).cuda()
        e = torch.from_numpy(np.ascontiguousarray(np.asarray(e, np.int8).reshape(rows, heads + extra, hd // 16))).cuda()
        return (m[:, :heads], e[:, :heads]), val[:, :heads]
    t = torch.from_numpy(full).to(_dt(kind))
    flat = torch.empty(t.numel() + off, dtype=t.dtype, device="cuda")
    x = flat[off:].view(t.shape)
    x.copy_(t)
    return x[:, :heads], t.double().numpy()[:, :heads]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_rope(gpu, case):
    import torch
    from bfp import rotary
    rows, heads, hd, rot, inter, kind, out_kind, extra, off = case
    rng = np.random.default_rng(rows * 1000 + hd)
    x, val = _typed(rng, rows, heads, hd, kind, extra, off)
    table = ref.angles(50, rot).astype(np.float32)
    pos = rng.integers(0, 50, rows).astype(np.int32)
    want = ref.rotate(val, pos, table, inter)
    _say(case)
    y = rotary.rope(x, torch.from_numpy(pos).cuda(), torch.from_numpy(table).cuda(), interleaved=inter,
                    dtype=_dt(out_kind) if out_kind else None)
    name = out_kind or ("f32" if kind == "tile" else kind)
    assert y.dtype == _dt(name)
    got = y.double().cpu().numpy()
    # products exact, one rounding in float64, one to the result
    tiny = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}[name] / 2
    assert (np.abs(got - want) <= HALF[name] * np.abs(want) + 2.0 ** -52 * 8 + tiny).all()
    # what is not turned is copied
    if kind == name:
        assert (got[..., rot:] == val[..., rot:]).all()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 32), (18, 10)])
def test_rope_in_place(gpu, inter, hd, rot):
    import torch
    from bfp import rotary
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(37, 3, hd, generator=g, device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(37, dtype=torch.int32, device="cuda")
    table = rotary.rope_table(rotary.rope_freqs(rot)[0], 37)
    want = rotary.rope(x, pos, table, interleaved=inter)
    assert rotary.rope(x, pos, table, interleaved=inter, out=x) is x
    assert torch.equal(x, want)


def test_rope_positions_outside_the_table(gpu):
    import torch
    from bfp import rotary
    for hd, rot in ((64, 32), (18, 10)):
        x = torch.ones(5, 2, hd, device="cuda")
        table = rotary.rope_table(rotary.rope_freqs(rot)[0], 8)
        pos = torch.tensor([0, -1, 8, 7, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
        y = rotary.rope(x, pos, table)
        bad = torch.isnan(y)
        assert bad[[1, 2, 4], :, :rot].all() and not bad[[0, 3]].any() and not bad[:, :, rot:].any()


def test_rope_other_layouts(gpu):
    """Heads before rows; a row used for all (stride 0); no rows."""
    import torch
    from bfp import rotary
    g = torch.Generator(device="cuda").manual_seed(4)
    table = rotary.rope_table(rotary.rope_freqs(64)[0], 20)
    pos = torch.arange(20, dtype=torch.int32, device="cuda")
    a = torch.randn(3, 20, 64, generator=g, device="cuda")
    want = rotary.rope(a.transpose(0, 1).contiguous(), pos, table)
    assert torch.equal(rotary.rope(a.transpose(0, 1), pos, table), want)
    out = torch.empty(3, 20, 64, device="cuda").transpose(0, 1)
    assert torch.equal(rotary.rope(a.transpose(0, 1), pos, table, out=out), want)
    one = torch.randn(1, 3, 64, generator=g, device="cuda").expand(20, 3, 64)
    assert torch.equal(rotary.rope(one, pos, table), rotary.rope(one.contiguous(), pos, table))
    assert rotary.rope(a[:, :0].transpose(0, 1), pos[:0], table).shape == (0, 3, 64)


def test_rope_extremes(gpu):
    """Infinities and NaN stay in their pair; the largest floats do not
    overflow on the way."""
    import torch
    from bfp import rotary
    table = torch.tensor([[[0.6, 0.8]] * 4], device="cuda")
    x = torch.zeros(1, 1, 8, device="cuda")
    x[0, 0, 1], x[0, 0, 2] = float("inf"), float("nan")
    big = torch.finfo(torch.float32).max
    x[0, 0, 3] = big
    y = rotary.rope(x, torch.zeros(1, dtype=torch.int32, device="cuda"), table)[0, 0]
    assert not torch.isfinite(y[[1, 5, 2, 6]]).any() and torch.isfinite(y[[0, 4, 3, 7]]).all()
    # the table's float32 factors, exactly
    assert abs(float(y[3]) / big - np.float32(0.6)) < 2e-7 and abs(float(y[7]) / big - np.float32(0.8)) < 2e-7


def test_rope_refuses(gpu):
    import torch
    from bfp import rotary
    from bfp._lib import BfpError
    x = torch.zeros(4, 2, 64, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    table = rotary.rope_table(rotary.rope_freqs(64)[0], 8)
    for bad in (lambda: rotary.rope(x[0], pos, table), lambda: rotary.rope(x.double(), pos, table),
                lambda: rotary.rope(x, pos[:3], table), lambda: rotary.rope(x, pos.long(), table),
                lambda: rotary.rope(x, pos, table[..., 0]), lambda: rotary.rope(x, pos, table.double()),
                lambda: rotary.rope(x, pos, table.cpu()), lambda: rotary.rope(x.cpu(), pos, table),
                lambda: rotary.rope(x.transpose(1, 2), pos, table),
                lambda: rotary.rope(x, pos, table, out=torch.zeros(4, 2, 32, device="cuda")),
                lambda: rotary.rope((x, x), pos, table)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(BfpError):
        rotary.rope(x[..., :32].contiguous(), pos, table)   # narrower than the table
    with pytest.raises(BfpError):                           # rows of the result on top of each other
        rotary.rope(x, pos, table, out=torch.zeros(1, 2, 64, device="cuda").expand(4, 2, 64))


def test_rope_captured(gpu):
    """Replays read what the buffers hold then."""
    import torch
    from bfp import rotary
    table = rotary.rope_table(rotary.rope_freqs(64)[0], 100)
    x, pos = torch.randn(6, 3, 64, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    y = torch.empty_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rotary.rope(x, pos, table, out=y)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotary.rope(x, pos, table, out=y)
    for step in range(4):
        x.copy_(torch.randn(6, 3, 64, device="cuda"))
        pos.fill_(17 * step)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, rotary.rope(x, pos, table)), step
