"""Decayed attention far from magnitude 1, against its recurrence in 64 bits.

The bounds are those of ``test_decay_attention_gpu`` (relative to A, the recurrence
over absolute values), without any floor for small operands: 16-bit operands that
the kernels make themselves carry a common power of two, so that an input's own
magnitude costs nothing.

A memory of one term S = g^n k v^T has no sum in it and takes a sharper bound.
Relative to its value, with x = n |log2 g|: the weight g^n is good to
(1.04 x + 2.5) 2^-23 per chunk that it passes (log2f within 1 ulp, one product,
exp2f within 2 ulp, one FMA), the weighed key's own rounding is 2^-24, its parts
leave 2^-22 (two of fp16; three of bf16 leave 2^-24) and their sum in the tensor cores
truncates at most 3 times by 2^-23, the scale's FMA 2^-24. Two parts of fp16 also leave
2^-38 of the chunk's largest weighed key: the second is a number below 2^-11 times the
scaled key, itself rounded no finer than 2^-25 where the largest is 2^13.
"""

from __future__ import annotations

import pytest
import torch

import myelin_b200 as mb
from tests.test_decay_attention_gpu import (
    _live, _randn, check, magnitude, memory_bound, out_bound, reference)

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALVES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-5, 3e-7])
@pytest.mark.parametrize("at", [0, 61, 100, 126, 127])
@pytest.mark.parametrize("Dk, Dv", [(64, 64), (128, 128), (40, 96)])
def test_a_memory_of_one_term_is_good_to_fp32(Dk, Dv, at, size, dtype):
    T, H = 128, 3
    decay = torch.tensor([0.98, 0.995, 0.9999], device=DEV)
    q, v = _randn((T, 1, H, Dk), 1, dtype), _randn((T, 1, H, Dv), 3, dtype)
    k = torch.zeros((T, 1, H, Dk), dtype=dtype, device=DEV)
    k[at] = (_randn((1, H, Dk), 2) * size).to(dtype)
    state, _ = mb.decay_attention_forward(q, k, v, decay)
    n = T - 1 - at
    w = decay.double()[None, :, None, None] ** n
    want = w * k[at].double()[..., :, None] * v[at].double()[..., None, :]
    x = n * torch.log2(decay.double()).abs()[None, :, None, None]
    relative = 2.0**-23 * (1.04 * x + 2.5 + 0.5 + 2 + 3 + 0.5)
    bound = relative * want.abs()
    if dtype == torch.float16:
        top = (w * k[at].double().abs().amax(-1)[..., None, None])
        bound = bound + 2.0**-38 * top * v[at].double().abs()[..., None, :]
    check(state.memory, want, bound, "memory")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("size", [1e-3, 1e-5, 1e2])
@pytest.mark.parametrize("Dk, Dv", [(64, 64), (128, 128)])
@pytest.mark.parametrize("ragged", [False, True])
def test_keys_of_any_size(Dk, Dv, size, ragged, dtype):
    T, B, H = 700, 3, 2
    decay = torch.tensor([0.75, 0.998], device=DEV)
    lengths = (torch.tensor([T, 130, 333], dtype=torch.int32, device=DEV) if ragged else None)
    q, v = _randn((T, B, H, Dk), 1, dtype), _randn((T, B, H, Dv), 3, dtype)
    k = (_randn((T, B, H, Dk), 2) * size).to(dtype)
    scale = 1.0 / (size * Dk)
    state, out = mb.decay_attention_forward(q, k, v, decay, scale=scale, lengths=lengths)
    S, o = reference(q, k, v, decay, None, scale, lengths)
    A_S, A_o = magnitude(q, k, v, decay, None, scale, lengths)
    check(out, o, out_bound(A_o, dtype, T, Dk), "outputs")
    check(state.memory, S, memory_bound(A_S, dtype, T, Dk), "memory")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("size", [1e-3, 1e-5])
@pytest.mark.parametrize("Dk, Dv", [(64, 64), (128, 128), (64, 128), (128, 40)])
def test_gradients_of_any_size(Dk, Dv, size, dtype):
    """The outputs' gradient is the key operand of the keys' gradient."""

    T, B, H = 400, 2, 2
    decay = torch.tensor([0.75, 0.998], device=DEV)
    lengths = torch.tensor([T, 290], dtype=torch.int32, device=DEV)
    leaves = [_randn((T, B, H, Dk), 1, dtype), _randn((T, B, H, Dk), 2, dtype),
              _randn((T, B, H, Dv), 3, dtype), _randn((B, H, Dk, Dv), 4)]
    go = (_randn((T, B, H, Dv), 5) * size).to(dtype)
    scale = 1.0 / (size * Dk)
    mine = [x.clone().requires_grad_(True) for x in leaves]
    _, out = mb.decay_attention_forward(*mine[:3], decay, mb.DecayAttentionState(mine[3]),
                                        scale=scale, lengths=lengths)
    got = torch.autograd.grad(out, mine, go)

    def grads(values, g):
        ls = [x.double().requires_grad_(True) for x in values]
        _, o = reference(*ls[:3], decay, ls[3], scale, lengths)
        return torch.autograd.grad(o, ls, g.double())

    want = grads(leaves, go)
    sizes = grads([x.abs() for x in leaves], go.abs())
    for name, a, w, A in zip(("dq", "dk", "dv"), got, want, sizes):
        check(a, w, out_bound(A, dtype, T, max(Dk, Dv)), name)
    check(got[3], want[3], memory_bound(sizes[3], dtype, T, max(Dk, Dv)), "dmemory")
    assert torch.equal(got[1].masked_fill(_live(T, lengths), 0), torch.zeros_like(got[1]))


@pytest.mark.parametrize("dtype", HALVES)
def test_a_memory_that_grows(dtype):
    """Decays above 1: the weights of a chunk's first keys pass fp16's range."""

    T, B, H, D = 300, 1, 2, 64
    decay = torch.tensor([1.1, 1.02], device=DEV)
    q, k, v = (_randn((T, B, H, D), s, dtype) for s in (1, 2, 3))
    S, o = reference(q, k, v, decay, None, 1e-13)
    A_S, A_o = magnitude(q, k, v, decay, None, 1e-13)
    state, out = mb.decay_attention_forward(q, k, v, decay, scale=1e-13)
    check(out, o, out_bound(A_o, dtype, T, D), "outputs")
    check(state.memory, S, memory_bound(A_S, dtype, T, D), "memory")


@pytest.mark.parametrize("dtype, T", [(torch.float32, 45), (torch.float32, 1030),
                                      (torch.bfloat16, 13)])
@pytest.mark.parametrize("size", [1e16, 1.0, 1e-15])
@pytest.mark.parametrize("D", [32, 80, 200])
def test_fast_leaks_keep_the_range_of_fp32(D, size, dtype, T):
    """The recurrent kernel, whose bursts of steps must not leave the range that the
    memory itself stays in: products of 1e32 and of 1e-30 with decays down to 0.

    Below fp32's normal range a kept value is rounded to a multiple of 2^-149, and it is
    at least 2^-15 of the memory: 2^-135 of memory per step, at most T of them, for each
    element of the operand that reads it. (1e16 puts the memory of dk at 1e-34.)"""

    decay = torch.tensor([0.0, 1e-5, 0.02, 0.1, 0.24, 0.4, 0.55, 1.0], device=DEV)
    H, scale = decay.numel(), 1.0 / (size * size * D)
    q, k, v = ((_randn((T, 1, H, D), s) * m).to(dtype) for s, m in ((1, 1.0), (2, size), (3, size)))
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    state, out = mb.decay_attention_forward(*leaves, decay, scale=scale)
    S, o = reference(q, k, v, decay, None, scale)
    A_S, A_o = magnitude(q, k, v, decay, None, scale)
    u = 2.0**-8 if dtype == torch.bfloat16 else 0.0  # the outputs' own rounding
    fp32 = (2 * T + D + 8) * 2.0**-24
    floor = lambda x, c: T * 2.0**-135 * c * x.detach().double().abs().sum(-1, keepdim=True)  # noqa: E731
    check(out.detach(), o.detach(), (fp32 + u) * A_o.detach() + floor(q, scale), "outputs")
    check(state.memory.detach(), S.detach(), fp32 * A_S.detach() + T * 2.0**-135, "memory")
    go = _randn(out.shape, 5, dtype)
    got = torch.autograd.grad(out, leaves, go)
    doubles = [x.detach().double().requires_grad_(True) for x in leaves]
    want = torch.autograd.grad(reference(*doubles, decay, None, scale)[1], doubles, go.double())
    parts = [x.detach().double().abs().requires_grad_(True) for x in leaves]
    sizes = torch.autograd.grad(reference(*parts, decay, None, scale)[1], parts, go.double().abs())
    reads = (floor(go, scale), floor(v, 1.0), floor(k, 1.0))
    for name, a, w, A, low in zip(("dq", "dk", "dv"), got, want, sizes, reads):
        check(a, w, (fp32 + u) * A + low, name)


def test_a_memory_that_grows_fast():
    T, D = 20, 48
    decay = torch.tensor([1.5, 4.0, 30.0], device=DEV)
    q, k, v = (_randn((T, 1, 3, D), s) for s in (1, 2, 3))
    S, o = reference(q, k, v, decay, None, 1e-3)
    A_S, A_o = magnitude(q, k, v, decay, None, 1e-3)
    state, out = mb.decay_attention_forward(q, k, v, decay, scale=1e-3)
    check(out, o, out_bound(A_o, q.dtype, T, D), "outputs")
    check(state.memory, S, memory_bound(A_S, q.dtype, T, D), "memory")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("size", [1e-30, 1e25])
def test_memories_of_any_size(size, dtype):
    """A first memory far from 1, brought back by the outputs' scale (no keys, so that
    it is all there is to read)."""

    T, B, H, D = 300, 2, 2, 64
    decay = torch.tensor([0.98, 0.999], device=DEV)
    q, v = _randn((T, B, H, D), 1, dtype), _randn((T, B, H, D), 3, dtype)
    k, memory = torch.zeros_like(q), _randn((B, H, D, D), 4) * size
    scale = 1.0 / (size * D)
    state, out = mb.decay_attention_forward(q, k, v, decay, mb.DecayAttentionState(memory),
                                            scale=scale)
    S, o = reference(q, k, v, decay, memory, scale)
    A_S, A_o = magnitude(q, k, v, decay, memory, scale)
    check(out, o, out_bound(A_o, dtype, T, D), "outputs")
    check(state.memory, S, memory_bound(A_S, dtype, T, D), "memory")
