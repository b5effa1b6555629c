"""SpikeDropout where its forward runs again in the backward pass, with a plain
dropout in place of the kernel: a mask is the forward's, or the call is refused."""

from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import myelin_b200 as mb
from myelin_b200 import compile_ops as cops
from myelin_b200 import modules


@pytest.fixture(autouse=True)
def plain_dropout(monkeypatch):
    def plain(x, p, seed, *, time_shared=False, training=True):
        g = torch.Generator().manual_seed(int(seed[0]) * 1009 + int(seed[1]))
        return torch.where(torch.rand(x.shape, generator=g) < p, 0.0, x / (1 - p))

    monkeypatch.setattr(modules, "spike_dropout", plain)


def _loss(y):
    return y.exp().sum()


@pytest.mark.parametrize("use_reentrant", [False, True])
def test_a_second_run_without_the_first_ones_seed_is_refused(use_reentrant):
    drop = mb.SpikeDropout(0.5, seed=5)
    x = torch.randn((4, 64), requires_grad=True)
    # exp saves what it needs inside the checkpointed part, so the backward runs it again
    y = checkpoint(lambda z: drop(z).exp(), x, use_reentrant=use_reentrant)
    with pytest.raises(RuntimeError, match="run again inside a backward pass"):
        y.sum().backward()
    assert drop.rng.tolist() == [5, 1]


@pytest.mark.parametrize("use_reentrant", [False, True])
def test_a_second_run_with_its_seed_gives_the_gradients_of_the_plain_call(use_reentrant):
    drop, twin = mb.SpikeDropout(0.5, seed=5), mb.SpikeDropout(0.5, seed=5)
    x = torch.randn((4, 64), requires_grad=True)
    for _ in range(2):
        y = checkpoint(lambda z, s: drop(z, s).exp(), x, drop.next_seed(),
                       use_reentrant=use_reentrant)
        (got,) = torch.autograd.grad(y.sum(), [x]) if not use_reentrant else (None,)
        if use_reentrant:
            x.grad = None
            y.sum().backward()
            got = x.grad
        want_y = twin(x).exp()
        (want,) = torch.autograd.grad(want_y.sum(), [x])
        assert torch.equal(y, want_y) and torch.equal(got, want)
    assert drop.rng.tolist() == twin.rng.tolist() == [5, 2]


def test_seeds_and_modes():
    drop = mb.SpikeDropout(0.5, seed=3)
    x = torch.randn((4, 64))
    seed = drop.next_seed()
    assert seed.tolist() == [3, 0] and drop.rng.tolist() == [3, 1]
    assert torch.equal(drop(x, seed), drop(x, seed)) and drop.rng.tolist() == [3, 1]
    assert drop.eval()(x, seed) is x and drop(x) is x and drop.rng.tolist() == [3, 1]
    net = mb.RateReadoutClassifier(4, 8, 2)
    with pytest.raises(ValueError, match="needs a SpikeDropout"):
        modules._drop(net.dropout, x, seed)


def test_seed_op():
    torch.library.opcheck(cops.next_seed_op, (torch.tensor([7, 2]),))
