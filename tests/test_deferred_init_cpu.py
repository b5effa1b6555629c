"""Modules made on the meta device and given storage afterwards, and casts that
leave fp32 buffers alone."""

from __future__ import annotations

import pytest
import torch

import myelin_b200 as mb


def _synapse():
    data = torch.arange(60, dtype=torch.int8).view(6, 10)
    return mb.QuantizedLinearSynapse(mb.QuantizedWeight(data, torch.rand(6)), torch.rand(6))


@pytest.mark.parametrize("make", [lambda: mb.DecayAttention(12, 2, 4, dropout=0.5), _synapse,
                                  lambda: mb.SpikeDropout(0.5)])
def test_meta_then_storage_then_state(make):
    ready = make()
    with torch.device("meta"):
        late = make()
    late = late.to("meta").to_empty(device="cpu")
    late.load_state_dict(ready.state_dict())
    for (name, a), (_, b) in zip(ready.state_dict().items(), late.state_dict().items()):
        assert a.dtype == b.dtype and torch.equal(a, b), name
    if isinstance(late, mb.QuantizedLinearSynapse):
        assert late.data.stride(0) % 16 == 0


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.to(torch.bfloat16),
                                  lambda m: m.to("meta").to(torch.bfloat16)])
def test_casts_leave_scales_and_decays(cast):
    layer = cast(mb.DecayAttention(12, 2, 4))
    assert layer.decay.dtype == torch.float32 and layer.keys.weight.dtype != torch.float32
    if not layer.decay.is_meta:
        assert torch.equal(layer.decay, mb.DecayAttention(12, 2, 4).decay)
    synapse = cast(_synapse())
    assert synapse.scale.dtype == torch.float32 and synapse.bias.dtype != torch.float32
    assert synapse.scale.device == synapse.bias.device
