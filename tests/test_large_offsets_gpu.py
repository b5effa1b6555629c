"""Offsets that pass 32 bits: elements of a tensor that lie more than 2^31 apart give
what the same values give close together."""

from __future__ import annotations

import pytest
import torch

import myelin_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"
FAR = 1 << 27  # elements between two steps: 17 of them pass 2^31


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def _randn(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV).to(dtype)


@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float16, 128),
                                      (torch.bfloat16, 136)])
def test_attention_over_far_steps(dtype, D):
    T, B, H = 20, 2, 3
    decay = torch.tensor([0.5, 0.9, 0.99], device=DEV)
    near = [_randn((T, B, H, D), s, dtype) for s in (1, 2, 3)]
    base = torch.empty((T - 1) * FAR + 3 * B * H * D, dtype=dtype, device=DEV)
    far = []
    for i, x in enumerate(near):
        view = base.as_strided((T, B, H, D), (FAR, H * D, D, 1), i * B * H * D)
        view.copy_(x)
        far.append(view)
    want = mb.decay_attention_forward(*near, decay, scale=0.1)
    got = mb.decay_attention_forward(*far, decay, scale=0.1)
    assert torch.equal(got[1], want[1]) and torch.equal(got[0].memory, want[0].memory)


def test_dropout_of_more_than_32_bits_of_elements():
    n = (1 << 31) + 4096
    seed = torch.tensor([5, 6], device=DEV)
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = mb.spike_dropout(x, 0.5, seed)
    rows = mb.spike_dropout(x.view(2, n // 2), 0.5, seed, time_shared=True)
    assert torch.equal(y[: n // 2], rows[0]) and torch.equal(rows[0], rows[1])
    tail = y[1 << 31:]
    assert set(tail.unique().tolist()) == {0.0, 2.0}
    assert abs(float((tail == 0).float().mean()) - 0.5) < 4 * 0.5 / 64


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8])
def test_integer_product_over_far_rows(dtype):
    M, K, N = 160, 64, 48
    g = torch.Generator(DEV).manual_seed(1)
    near = torch.randint(-100, 100, (M, K), generator=g, device=DEV).to(dtype)
    pitch = 1 << 24
    base = torch.empty((M - 1) * pitch + K, dtype=dtype, device=DEV)
    far = base.as_strided((M, K), (pitch, 1))
    far.copy_(near)
    weight = mb.QuantizedWeight(torch.randint(-127, 128, (N, K), generator=g, device=DEV).to(
        torch.int8), torch.rand(N, generator=g, device=DEV))
    assert torch.equal(mb.quantized_linear(far, weight), mb.quantized_linear(near, weight))
    rows = mb.quantize_rows(far.float() if dtype == torch.int8 else far)
    want = mb.quantize_rows(near.float() if dtype == torch.int8 else near)
    assert torch.equal(rows.data, want.data) and torch.equal(rows.scale, want.scale)
