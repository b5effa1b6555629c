"""Dropout from the counter-based generator, against Philox 4x32-10 in Python integers.

The mask has to be exact; a kept value is x times an fp32 scale (one rounding)
and one more rounding to the dtype, against the product in 64 bits: within
(eps / 2 + 2^-23) of it.
"""

from __future__ import annotations

import pytest
import torch

import myelin_b200 as mb
from myelin_b200 import compile_ops as cops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def philox(counter, key):
    """Philox 4x32-10 on Python integers: four words in, four words out."""

    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep_mask(n, p, seed, offset):
    threshold = round(p * 65536)
    seed, offset = seed % 2**64, offset % 2**64
    keep = []
    for g in range((n + 7) // 8):
        w = philox([g & 0xFFFFFFFF, g >> 32, offset & 0xFFFFFFFF, offset >> 32],
                   [seed & 0xFFFFFFFF, seed >> 32])
        keep += [((w[j // 2] >> (16 * (j % 2))) & 0xFFFF) >= threshold for j in range(8)]
    return torch.tensor(keep[:n])


def test_philox_known_answer():
    """The published known answers of Philox 4x32-10 (all-zero and all-one inputs)."""

    assert philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert philox([ones] * 4, [ones] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape, shared", [
    ((1,), False), ((7,), True), ((3, 5), False), ((40, 3, 33), True), ((9, 2, 64), True),
    ((5, 1000), False), ((2, 8, 1024), True), ((300, 1, 8), True),
])
@pytest.mark.parametrize("p", [0.0001, 0.3, 0.999, 1.0])
def test_matches_the_generator(shape, shared, dtype, p):
    seed, offset = -5 if p == 0.3 else 2**61 + 12345, 2**40 + 7
    x = torch.randn(shape, generator=torch.Generator(DEV).manual_seed(1), device=DEV).to(dtype)
    s = torch.tensor([seed, offset], device=DEV)
    y = mb.spike_dropout(x, p, s, time_shared=shared)
    n = x[0].numel() if shared else x.numel()
    keep = keep_mask(n, p, seed, offset).to(DEV)
    keep = (keep.view(shape[1:]).expand(shape) if shared else keep.view(shape))
    threshold = round(p * 65536)
    assert torch.equal(y == 0, ~keep | (x == 0)) and y.dtype == dtype
    if threshold < 65536:
        want = torch.where(keep, x.double() * 65536 / (65536 - threshold), 0.0)
        finite = want.abs() <= torch.finfo(dtype).max
        tol = (torch.finfo(dtype).eps / 2 + 2.0**-23) * want.abs() + 2.0**-25
        assert ((y.double() - want).abs() <= tol)[finite].all()
    else:
        assert torch.count_nonzero(y) == 0


def test_dropped_values_vanish_whatever_they_were():
    x = torch.full((4096,), float("nan"), device=DEV)
    s = torch.tensor([3, 4], device=DEV)
    y = mb.spike_dropout(x, 0.5, s)
    keep = keep_mask(4096, 0.5, 3, 4).to(DEV)
    assert torch.equal(torch.isnan(y), keep) and torch.equal(y == 0, ~keep)


@pytest.mark.parametrize("shared", [False, True])
def test_gradient_uses_the_same_mask(shared):
    x = torch.randn((6, 3, 41), device=DEV, requires_grad=True)
    s = torch.tensor([11, 5], device=DEV)
    y = mb.spike_dropout(x, 0.4, s, time_shared=shared)
    g = torch.randn(x.shape, device=DEV)
    (dx,) = torch.autograd.grad(y, [x], g, create_graph=True)
    mask = mb.spike_dropout(torch.ones_like(x.detach()), 0.4, s, time_shared=shared)
    torch.testing.assert_close(dx, g * mask, rtol=2.0**-22, atol=0)
    # against differences: the operator is linear
    d = torch.randn(x.shape, device=DEV)
    f = lambda z: (mb.spike_dropout(z, 0.4, s, time_shared=shared).double() * g.double()).sum()  # noqa: E731
    with torch.no_grad():
        diff = (f(x + d) - f(x - d)) / 2
    inner = (dx.detach().double() * d.double()).sum()
    assert (diff - inner).abs() <= 2.0**-22 * (g.abs() * (x.abs() + d.abs()) * mask).double().sum()
    # a seed that changes before the backward is noticed
    y = mb.spike_dropout(x, 0.4, s, time_shared=shared)
    s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_strided_inputs_and_share_of_zeros():
    base = torch.randn((512, 1024), device=DEV)
    s = torch.tensor([1, 2], device=DEV)
    assert torch.equal(mb.spike_dropout(base.t(), 0.25, s),
                       mb.spike_dropout(base.t().contiguous(), 0.25, s))
    y = mb.spike_dropout(torch.ones((1 << 22,), device=DEV), 0.25, s)
    share = (y == 0).double().mean()
    # four standard deviations of a binomial share
    assert abs(float(share) - 0.25) <= 4 * (0.25 * 0.75 / (1 << 22)) ** 0.5


def test_module_counts_its_calls_and_replays():
    drop = mb.SpikeDropout(0.5, seed=9).to(DEV)
    x = torch.ones((4, 8, 64), device=DEV)
    first, second = drop(x), drop(x)
    assert drop.rng.tolist() == [9, 2] and not torch.equal(first, second)
    assert torch.equal(first[0], first[3])  # one mask for all steps
    assert torch.equal(first, mb.spike_dropout(x, 0.5, torch.tensor([9, 0], device=DEV),
                                               time_shared=True))
    assert drop.eval()(x) is x
    drop.train()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        drop(x)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        held = drop(x)
    at = int(drop.rng[1])
    for i in range(3):
        graph.replay()
        want = mb.spike_dropout(x, 0.5, torch.tensor([9, at + i], device=DEV), time_shared=True)
        assert torch.equal(held, want)


def test_classifier_drops_neurons_for_the_whole_window():
    torch.manual_seed(0)
    net = mb.RateReadoutClassifier(12, 64, 4, dropout=0.5, time_shared_dropout=True).to(DEV)
    x = torch.randn((10, 3, 12), device=DEV)
    rates = net(x)
    rates.sum().backward()
    assert rates.shape == (3, 4) and torch.isfinite(net.hidden.synapse.weight.grad).all()
    assert int(net.dropout.rng[1]) == 1
    plain = mb.RateReadoutClassifier(12, 64, 4, dropout=0.5)
    assert isinstance(plain.dropout, torch.nn.Dropout)


def test_opcheck():
    x = torch.randn((4, 40), device=DEV)
    torch.library.opcheck(cops.dropout_op, (x, torch.tensor([1, 2], device=DEV), 20000, True))


def test_empty():
    s = torch.tensor([1, 2], device=DEV)
    assert mb.spike_dropout(torch.zeros((0, 4), device=DEV), 0.5, s, time_shared=True).shape == (0, 4)
    assert mb.spike_dropout(torch.zeros((4, 0), device=DEV), 0.5, s).shape == (4, 0)
