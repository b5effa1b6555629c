"""Dropout on tensors whose first element is not where an allocation starts: the
result is that of a copy at an aligned address."""

from __future__ import annotations

import pytest
import torch

import myelin_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [1, 2, 4, 8, 12])
@pytest.mark.parametrize("shape, shared", [((6, 1024), False), ((6, 1024), True), ((5, 3, 8), True),
                                           ((7, 41), True), ((8192,), False)])
def test_views_at_any_element(shape, shared, offset, dtype):
    seed = torch.tensor([21, 3], device=DEV)
    x = torch.randn(shape, generator=torch.Generator(DEV).manual_seed(2), device=DEV).to(dtype)
    view = torch.zeros(x.numel() + offset, dtype=dtype, device=DEV)[offset:].view(shape)
    view.copy_(x)
    assert view.storage_offset() == offset and view.is_contiguous()
    want = mb.spike_dropout(x, 0.3, seed, time_shared=shared)
    assert torch.equal(mb.spike_dropout(view, 0.3, seed, time_shared=shared), want)
    # the gradient's kernel reads the gradient where it lies
    leaf = x.clone().requires_grad_(True)
    out = mb.spike_dropout(leaf, 0.3, seed, time_shared=shared)
    (got,) = torch.autograd.grad(out, [leaf], view)
    assert torch.equal(got, want)
