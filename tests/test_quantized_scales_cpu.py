"""Gradients asked of a scale: refused, as those of the inputs are."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import myelin_b200 as mb


@pytest.mark.parametrize("of", ["rows", "weight", "bias"])
def test_a_scale_that_requires_a_gradient_is_refused(of):
    with FakeTensorMode():
        rows = mb.QuantizedRows(torch.empty((2, 8), dtype=torch.int8, device="cuda"),
                                torch.empty(2, device="cuda", requires_grad=of == "rows"))
        weight = mb.QuantizedWeight(torch.empty((6, 8), dtype=torch.int8, device="cuda"),
                                    torch.empty(6, device="cuda", requires_grad=of == "weight"))
        bias = torch.empty(6, device="cuda", requires_grad=of == "bias")
        with pytest.raises(NotImplementedError, match="forward only"):
            mb.quantized_linear(rows, weight, bias)
        with torch.no_grad():
            assert mb.quantized_linear(rows, weight, bias).shape == (2, 6)
