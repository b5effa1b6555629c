"""Which synapses a streaming layer hands to the fused function: any that has a
weight and a bias, but not 8-bit ones."""

from __future__ import annotations

import torch
from torch import nn

import myelin_b200 as mb
from myelin_b200 import modules


class OwnSynapse(nn.Module):
    def __init__(self):
        super().__init__()
        self.weight, self.bias = nn.Parameter(torch.zeros((4, 6))), None

    def forward(self, inputs):
        raise AssertionError("the fused function takes the weight")


def test_a_synapse_of_the_users_own_is_streamed(monkeypatch):
    seen = []

    def fused(inputs, weight, bias, *args, **kw):
        seen.append((weight, bias))
        return None, inputs

    monkeypatch.setattr(modules, "linear_surrogate_lif_forward", fused)
    layer = mb.LinearSurrogateLIF(4, 6, stream_synapse=True)
    x = torch.zeros((3, 2, 4))
    for synapse in (layer.synapse, OwnSynapse()):
        layer.synapse = synapse
        assert layer(x) is x
        assert seen.pop() == (synapse.weight, synapse.bias)
    layer.synapse = mb.QuantizedLinearSynapse(
        mb.QuantizedWeight(torch.zeros((6, 4), dtype=torch.int8), torch.ones(6)))
    monkeypatch.setattr(layer.synapse, "forward", lambda z: z)
    layer.unroll = nn.Module()
    layer.unroll.cell, layer.unroll.forward = None, lambda z: (None, z)
    assert layer(x) is x and not seen
