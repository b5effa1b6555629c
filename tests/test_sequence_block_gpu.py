"""The new operators in one run, as a model uses them: train a layer of decayed
attention with dropout, then serve it with 8-bit synapses, a prompt and single steps."""

from __future__ import annotations

import pytest
import torch

import myelin_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _plain(layer, x, mask=None, projections=None):
    """The layer from its recurrence, in float64 (differentiable)."""

    T, B, _ = x.shape
    H, Dk, Dv = layer.heads, layer.key_size, layer.value_size
    project = projections or (lambda name, y: y @ getattr(layer, name).weight.double()
                              + getattr(layer, name).bias.double())
    q = project("queries", x).view(T, B, H, Dk)
    k = project("keys", x).view(T, B, H, Dk)
    v = project("values", x).view(T, B, H, Dv)
    g = layer.decay.double()[None, :, None, None]
    S = torch.zeros((B, H, Dk, Dv), dtype=torch.float64, device=x.device)
    outs = []
    for t in range(T):
        S = g * S + k[t][..., :, None] * v[t][..., None, :]
        outs.append(Dk**-0.5 * torch.einsum("bhd,bhde->bhe", q[t], S).flatten(-2))
    y = torch.stack(outs)
    return S, project("output", y if mask is None else y * mask)


def test_training_step_matches_the_plain_layer():
    torch.manual_seed(0)
    layer = mb.DecayAttention(48, 4, 16, 24, 20, dropout=0.25).to(DEV)
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(0, 0.15)
    x = torch.randn((70, 3, 48), device=DEV, requires_grad=True)
    seed = layer.dropout.rng.clone()
    state, out = layer(x)
    mask = mb.spike_dropout(torch.ones((70, 3, 96), device=DEV), 0.25, seed, time_shared=True)
    S, want = _plain(layer, x.double(), mask.double())
    g = torch.randn(out.shape, device=DEV)
    leaves = [x, *layer.parameters()]
    mine = torch.autograd.grad((out * g).sum() + state.memory.sum(), leaves)
    plain = torch.autograd.grad((want * g.double()).sum() + S.sum(), leaves)
    assert torch.equal(mask[0], mask[69]) and 0 < float((mask[0] == 0).double().mean()) < 1
    # fp32 against fp64: sums of up to 70 x 48 x 48 terms, relative to their norms
    assert (out.double() - want).norm() <= 1e-5 * want.norm()
    assert (state.memory.double() - S).norm() <= 1e-5 * S.norm()
    for a, b in zip(mine, plain):
        assert (a.double() - b).norm() <= 1e-5 * b.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_serving_in_8_bits_prompt_then_steps(dtype):
    torch.manual_seed(1)
    layer = mb.DecayAttention(64, 2, 32).to(DEV)
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(0, 0.1)
    layer = mb.quantize_synapses(layer).to(dtype).eval()
    assert layer.decay.dtype == torch.float32 and layer.values.scale.dtype == torch.float32
    x = torch.randn((150, 3, 64), device=DEV).to(dtype)
    lengths = torch.tensor([130, 1, 130], dtype=torch.int32, device=DEV)
    with torch.inference_mode():
        state, out = layer(x[:130], lengths=lengths)
        active = torch.tensor([True, False, True], device=DEV)
        steps = []
        before = state.memory.clone()
        for t in range(130, 150):
            state, y = layer.step(x[t], state, active, inplace=True)
            steps.append(y)
        whole_state, whole = layer(x)
    # the padded row stays where its prompt ended
    assert torch.equal(state.memory[1], before[1])
    got = torch.cat([out, torch.stack(steps)])[:, [0, 2]].double()
    want = whole[:, [0, 2]].double()
    # Two routes of the same definition: per 16-bit output of the attention they differ by
    # a few half steps u of its terms; an 8-bit row step is 1 / 254 of its largest value, so a
    # value near a border may land on the next one. Both are far below the layer's own
    # quantisation error, 1 / 127 of the terms.
    assert (got - want).norm() <= (1 / 127) * want.norm()
    S, Sw = state.memory[[0, 2]].double(), whole_state.memory[[0, 2]].double()
    assert (S - Sw).norm() <= 2.0**-16 * Sw.norm()


def test_refusals():
    with pytest.raises(ValueError, match="heads and key_size"):
        mb.DecayAttention(8, 0, 4)
    with pytest.raises(ValueError, match="tau_min"):
        mb.DecayAttention(8, 1, 4, tau_min=0.5)
