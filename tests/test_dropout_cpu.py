"""Argument checks of the counter-based dropout, without a GPU."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import myelin_b200 as mb
from myelin_b200 import _native as nat


def test_refusals():
    x, s = torch.zeros((4, 8)), torch.zeros(2, dtype=torch.int64)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="probability must be in"):
            mb.spike_dropout(x, p, s)
        with pytest.raises(ValueError, match="probability must be in"):
            mb.SpikeDropout(p)
    with pytest.raises(ValueError, match="CUDA devices only"):
        mb.spike_dropout(x, 0.5, s)
    with pytest.raises(ValueError, match="needs inputs shaped"):
        mb.spike_dropout(x[0, 0], 0.5, s, time_shared=True)
    assert mb.spike_dropout(x, 0.5, s, training=False) is x
    assert mb.spike_dropout(x, 0.0, s) is x
    with FakeTensorMode():
        c = torch.empty((4, 8), device="cuda")
        cs = torch.empty((2,), dtype=torch.int64, device="cuda")
        with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
            mb.spike_dropout(c.double(), 0.5, cs)
        with pytest.raises(ValueError, match=r"seed must be int64 shaped \[2\]"):
            mb.spike_dropout(c, 0.5, cs.int())
        with pytest.raises(ValueError, match=r"seed must be int64 shaped \[2\]"):
            mb.spike_dropout(c, 0.5, cs[:1])
        with pytest.raises(ValueError, match="same device"):
            mb.spike_dropout(c, 0.5, torch.empty((2,), dtype=torch.int64, device="cpu"))
        assert mb.spike_dropout(c, 0.5, cs).shape == (4, 8)


def test_c_entry():
    lib = nat.lib()
    assert lib.mb_dropout(0, None, None, 0, 8, 5, None, None) == 0
    for args, message in (((0, None, None, 1, 8, 65537, None, None), "threshold"),
                          ((7, None, None, 1, 8, 5, None, None), "unsupported dtype"),
                          ((0, None, None, -1, 8, 5, None, None), "negative"),
                          ((0, None, None, 1, 8, 5, None, None), "null tensor")):
        assert lib.mb_dropout(*args) != 0 and message in lib.mb_last_error().decode()
