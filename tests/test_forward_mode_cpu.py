"""Tangents of forward-mode differentiation: refused, since a launch would drop them
and the derivative would read as zero."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode

import myelin_b200 as mb
from myelin_b200.autograd import DecayAttentionFunction, DropoutFunction

MODE = FakeTensorMode(allow_non_fake_inputs=True)
SHAPES = {"q": (4, 2, 3, 8), "k": (4, 2, 3, 8), "v": (4, 2, 3, 16), "m": (2, 3, 8, 16)}


def _calls():
    def forward(a):
        mb.decay_attention_forward(a["q"], a["k"], a["v"], a["decay"],
                                   mb.DecayAttentionState(a["m"]))

    def step(inplace):
        def call(a):
            mb.decay_attention_step(a["q"][0], a["k"][0], a["v"][0], a["decay"],
                                    mb.DecayAttentionState(a["m"]), inplace=inplace)
        return call

    def dropout(a):
        mb.spike_dropout(a["q"], 0.5, a["seed"])

    def rows(a):
        mb.quantize_rows(a["q"])

    def weight(a):
        mb.quantize_weight(a["q"][0, 0])

    def linear(a):
        mb.quantized_linear(a["q"], mb.QuantizedWeight(a["w"], a["scale"]), a["bias"])

    return [(forward, n) for n in "qkvm"] + [(step(i), n) for i in (False, True) for n in "qkvm"] + [
        (dropout, "q"), (rows, "q"), (weight, "q"), (linear, "q"), (linear, "scale"), (linear, "bias")]


@pytest.mark.parametrize("call, name", _calls())
def test_tangents_are_refused(call, name):
    with MODE:
        a = {n: torch.empty(s, device="cuda") for n, s in SHAPES.items()}
        a |= {"decay": torch.empty(3, device="cuda"), "scale": torch.empty(6, device="cuda"),
              "seed": torch.empty(2, dtype=torch.int64, device="cuda"),
              "w": torch.empty((6, 8), dtype=torch.int8, device="cuda"),
              "bias": torch.empty(6, device="cuda")}
        call(a)
        with fwd.dual_level():
            call(a)  # tensors without a tangent run as ever
            a[name] = fwd.make_dual(a[name], torch.empty_like(a[name]))
            with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                call(a)


@pytest.mark.parametrize("function, grads", [(DecayAttentionFunction, 2), (DropoutFunction, 1)])
def test_tangents_of_a_gradient_are_refused(function, grads):
    with fwd.dual_level():
        g = fwd.make_dual(torch.ones(3), torch.ones(3))
        with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
            function.backward(SimpleNamespace(), g, *[None] * (grads - 1))
