"""8-bit projections whose two scales multiply to a number outside fp32's range while
the results lie inside it, by the bound of ``test_quantized_gpu`` and 2^-150: a result
below 2^-126 is itself rounded to a multiple of 2^-149."""

from __future__ import annotations

import pytest
import torch

import myelin_b200 as mb
from tests.test_quantized_gpu import _randn, reference_rows, weights

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("M, N, K", [(2, 40, 200), (70, 100, 784), (300, 2600, 640)])
@pytest.mark.parametrize("rows, channels", [(1e-23, 1e-15), (1e-28, 1e-10), (1e25, 1e-30)])
def test_small_products_of_scales(M, N, K, rows, channels):
    x = _randn((M, K), 1) * rows
    w = weights(N, K, 2)
    w = mb.QuantizedWeight(w.data, w.scale * channels)
    q, scale = reference_rows(x)
    got = mb.quantized_linear(x, w).double().cpu()
    acc = q.double() @ w.data.double().cpu().t()
    want = acc * w.scale.double().cpu() * scale.double()[:, None]
    # 3 2^-24 for the scaling, half a step and 2^-24 for the rounding (2^-23 is fp32's eps)
    tol = (3 * 2.0**-24 + 2.0**-24 + 2.0**-24) * want.abs() + 2.0**-150
    assert ((got - want).abs() <= tol).all()
    assert float(want.abs().max()) > 2.0**-126


@pytest.mark.parametrize("M, N, K", [(2, 40, 200), (70, 100, 784), (300, 2600, 640)])
def test_sums_of_zero_by_large_scales(M, N, K):
    x = _randn((M, K), 1) * 1e32
    w = mb.QuantizedWeight(torch.zeros((N, K), dtype=torch.int8, device=DEV),
                           torch.full((N,), 1e12, device=DEV))
    bias = _randn((N,), 3)
    assert torch.equal(mb.quantized_linear(x, w, bias), bias.expand(M, N))
