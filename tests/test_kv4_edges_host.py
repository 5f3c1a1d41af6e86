"""The ends of what the rotary and 4-bit-cache entry points take, on the CPU:
what they refuse at their own checks, and what they do not."""
import ctypes as C

import numpy as np
import pytest

from test_kv4_host import _batch, _cache, _lib, _refused, _rows


def test_in_place_forms_put_back_the_same_object():
    """t.lens += 1 writes into the tensor and then assigns it: no other
    object, so nothing to refuse; another one is."""
    import torch
    from bfp._rows import Fixed

    class Thing(Fixed):
        def __init__(self, lens):
            self.lens = lens
    lens = torch.tensor([3, 4])
    t = Thing(lens)
    t.lens += 1
    t.lens *= 2
    assert t.lens is lens and lens.tolist() == [8, 10]
    with pytest.raises(AttributeError):
        t.lens = t.lens + 1
    assert t.lens is lens and lens.tolist() == [8, 10]
