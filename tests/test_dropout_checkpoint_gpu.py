"""Layers with SpikeDropout under activation checkpointing and compilation: the same
outputs and gradients as the plain call with the same seed."""

from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import myelin_b200 as mb

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _grads(net, x, run):
    y = run(x)
    (y + y.square()).sum().backward()  # (rates may be zero: their gradient is not)
    got = [x.grad, *(p.grad for p in net.parameters())]
    x.grad = None
    net.zero_grad(set_to_none=True)
    return y.detach(), got


@pytest.mark.parametrize("use_reentrant", [False, True])
@pytest.mark.parametrize("kind", ["attention", "classifier"])
def test_checkpointed_layer(kind, use_reentrant):
    torch.manual_seed(0)
    if kind == "attention":
        net = mb.DecayAttention(32, 2, 16, dropout=0.4).to(DEV)
        call = lambda z, s: net(z, None, None, s)[1]  # noqa: E731
    else:
        net = mb.RateReadoutClassifier(32, 48, 5, dropout=0.4, time_shared_dropout=True).to(DEV)
        call = net
    x = torch.randn((30, 3, 32), device=DEV, requires_grad=True)
    seed = net.dropout.next_seed()
    y, got = _grads(net, x, lambda z: checkpoint(call, z, seed, use_reentrant=use_reentrant))
    want_y, want = _grads(net, x, lambda z: call(z, seed))
    assert torch.equal(y, want_y)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.count_nonzero(got[0])
    assert net.dropout.rng[1] == 1
    with pytest.raises(RuntimeError, match="run again inside a backward pass"):
        checkpoint(lambda z: call(z, None), x, use_reentrant=use_reentrant).sum().backward()


def test_compiled_layer_counts_its_calls():
    torch.manual_seed(0)
    net = mb.DecayAttention(32, 2, 16, dropout=0.5).to(DEV)
    x = torch.randn((20, 2, 32), device=DEV)
    fast = torch.compile(net, fullgraph=True)
    outs = [fast(x)[1] for _ in range(2)]
    assert net.dropout.rng[1] == 2
    net.dropout.rng[1] = 0
    for out in outs:
        want = net(x)[1]
        assert (out - want).abs().max() <= 1e-4 * want.abs().max()
    assert not torch.equal(outs[0], outs[1])


def test_compiled_training_step_has_the_forwards_mask():
    torch.manual_seed(0)
    net = mb.DecayAttention(32, 2, 16, dropout=0.5).to(DEV)
    x = torch.randn((20, 2, 32), device=DEV, requires_grad=True)
    fast = torch.compile(net, fullgraph=True)
    y, got = _grads(net, x, lambda z: fast(z)[1])
    assert net.dropout.rng[1] == 1
    net.dropout.rng[1] = 0
    want_y, want = _grads(net, x, lambda z: net(z)[1])
    for a, b in zip((y, *got), (want_y, *want)):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max()


def test_compiled_checkpoint_is_right_or_refused():
    torch.manual_seed(0)
    net = mb.DecayAttention(32, 2, 16, dropout=0.5).to(DEV)
    x = torch.randn((20, 2, 32), device=DEV, requires_grad=True)
    fast = torch.compile(lambda z: checkpoint(lambda w: net(w)[1], z, use_reentrant=False))
    try:
        y, got = _grads(net, x, fast)
    except Exception as error:  # noqa: BLE001  (the compiler may wrap it)
        assert "run again inside a backward pass" in str(error) or "HigherOrder" in str(error) \
            or "side effect" in str(error).lower()
        return
    net.dropout.rng[1] = 0
    want_y, want = _grads(net, x, lambda z: net(z)[1])
    for a, b in zip((y, *got), (want_y, *want)):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max()
