"""Attention over a shared prefix where the two parts of the work differ:
sequences outside every group with more rows than the groups have, scratch
that holds NaN before the call."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import HALF, _dt, _int, _say, _typed
from test_gpu_kv4_shared import Groups, _bound

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
