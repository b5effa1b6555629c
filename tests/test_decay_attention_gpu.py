"""Attention with a decay for each head, against its recurrence in 64 bits.

Error bounds, elementwise, with u the output type's half step
(``finfo.eps / 2``) and A the same recurrence over absolute values (the sum of
the magnitudes of every term):

- outputs and 16-bit gradients: u |o| for the final rounding, u A for the
  rounding of the scores and u A for the rounding of the memory where they
  become 16-bit operands, doubled for second-order terms: 4 u A in all (|o| <= A);
- fp32 outputs and memories of fp32 inputs: two roundings per step of the
  recurrence and one per term of the products: (2 T + D + 8) 2^-24 A;
- the fp32 memory of 16-bit inputs: the weighted keys go as two 16-bit parts,
  which leaves u^2 <= 2^-16 of each term, plus the sums: 2^-16 A +
  (T + 16) 2^-23 A (the tensor cores truncate where they add).
"""

from __future__ import annotations

import pytest
import torch

import myelin_b200 as mb
from myelin_b200 import _native as nat
from myelin_b200 import compile_ops as cops

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=_gen(seed), device=DEV).to(dtype)


def _decay(H):
    return (1.0 - 1.0 / torch.logspace(0.5, 8, H, base=2.0, dtype=torch.float64)).float().to(DEV)


def _live(T, lengths):
    if lengths is None:
        return None
    t = torch.arange(T, device=DEV)[:, None]
    return (t < lengths.to(torch.int64)[None, :])[:, :, None, None]


def reference(q, k, v, decay, memory, scale, lengths=None):
    """The recurrence in float64 (differentiable)."""

    q, k, v = q.double(), k.double(), v.double()
    T, B, H, Dk = q.shape
    live = _live(T, lengths)
    if live is not None:
        q, k, v = (torch.where(live, x, torch.zeros_like(x)) for x in (q, k, v))
    g = decay.double()[None, :, None, None]
    S = (torch.zeros((B, H, Dk, v.shape[3]), dtype=torch.float64, device=q.device)
         if memory is None else memory.double())
    outs = []
    for t in range(T):
        step = g * S + k[t][..., :, None] * v[t][..., None, :]
        S = step if live is None else torch.where(live[t][..., None], step, S)
        outs.append(scale * torch.einsum("bhd,bhde->bhe", q[t], S))
    out = torch.stack(outs) if outs else v.new_zeros(v.shape)
    return S, out


def magnitude(q, k, v, decay, memory, scale, lengths=None):
    return reference(q.abs(), k.abs(), v.abs(), decay, None if memory is None else memory.abs(),
                     abs(scale), lengths)


def check(got, want, bound, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    worst = ((got - want).abs() - bound).max() if got.numel() else torch.tensor(-1.0)
    assert worst <= 1e-30, (what, float(worst), float((got - want).abs().max()))


def out_bound(A, dtype, T, D):
    if dtype == torch.float32:
        return (2 * T + D + 8) * 2.0**-24 * A
    u = torch.finfo(dtype).eps / 2
    tiny = 2.0**-24 if dtype == torch.float16 else 0.0  # half a step of the subnormals
    return 4 * u * A + tiny


def memory_bound(A, dtype, T, D):
    if dtype == torch.float32:
        return (2 * T + D + 8) * 2.0**-24 * A
    return (2.0**-16 + (T + 16) * 2.0**-23) * A


def run_and_check(q, k, v, decay, memory, scale, lengths=None):
    T, _, _, D = q.shape
    first = None if memory is None else mb.DecayAttentionState(memory)
    state, out = mb.decay_attention_forward(q, k, v, decay, first, scale=scale, lengths=lengths)
    S, o = reference(q, k, v, decay, memory, scale, lengths)
    A_S, A_o = magnitude(q, k, v, decay, memory, scale, lengths)
    assert out.dtype == q.dtype and state.memory.dtype == torch.float32
    check(out, o, out_bound(A_o, q.dtype, T, D), "outputs")
    check(state.memory, S, memory_bound(A_S, q.dtype, T, D), "memory")
    return state, out


SHAPES = [
    (1, 1, 1, 1, 1),
    (1, 2, 3, 64, 64),
    (2, 1, 2, 16, 8),
    (7, 2, 2, 40, 72),
    (64, 1, 3, 128, 64),
    (127, 2, 1, 64, 128),
    (128, 1, 2, 128, 128),
    (129, 2, 2, 64, 64),
    (65, 3, 2, 33, 17),
    (300, 2, 3, 96, 40),
    (257, 1, 2, 128, 120),
    (70, 1, 1, 256, 200),
    (40, 1, 2, 24, 256),
    (2100, 1, 1, 64, 64),
    (1500, 1, 2, 128, 128),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_matches_the_recurrence(shape, dtype):
    T, B, H, Dk, Dv = shape
    q, k = _randn((T, B, H, Dk), 1, dtype), _randn((T, B, H, Dk), 2, dtype)
    v = _randn((T, B, H, Dv), 3, dtype)
    memory = _randn((B, H, Dk, Dv), 4) if T % 2 else None
    run_and_check(q, k, v, _decay(H), memory, Dk**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 130, 700])
def test_ragged_rows_ignore_what_lies_past_them(T, dtype):
    B, H, Dk, Dv = 6, 2, 64, 48
    lengths = torch.tensor([T, 0, 1, T // 2, T + 9, -3], dtype=torch.int32, device=DEV)
    clamped = lengths.clamp(0, T)
    q, k = _randn((T, B, H, Dk), 1, dtype), _randn((T, B, H, Dk), 2, dtype)
    v, memory = _randn((T, B, H, Dv), 3, dtype), _randn((B, H, Dk, Dv), 4)
    live = _live(T, clamped).expand_as(q)
    clean = [x.clone() for x in (q, k, v)]
    for x, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan"))):
        x.masked_fill_(~live[..., :1], bad)
    state, out = mb.decay_attention_forward(q, k, v, _decay(H), mb.DecayAttentionState(memory),
                                            scale=0.25, lengths=lengths)
    S, o = reference(*clean, _decay(H), memory, 0.25, clamped)
    A_S, A_o = magnitude(*clean, _decay(H), memory, 0.25, clamped)
    check(out, o, out_bound(A_o, dtype, T, Dk), "outputs")
    check(state.memory, S, memory_bound(A_S, dtype, T, Dk), "memory")
    assert torch.equal(out[:, 1], torch.zeros_like(out[:, 1]))
    assert torch.equal(state.memory[1], memory[1]) and torch.equal(state.memory[5], memory[5])


@pytest.mark.parametrize("dtype", DTYPES)
def test_decay_of_zero_and_one(dtype):
    T, B, D = 200, 2, 64
    decay = torch.tensor([0.0, 1.0, 1e-30], device=DEV)
    q, k, v = (_randn((T, B, 3, D), s, dtype) for s in (1, 2, 3))
    run_and_check(q, k, v, decay, _randn((B, 3, D, D), 4), 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e-3, 200.0])
def test_small_and_large_values(dtype, size):
    """Magnitudes away from 1: products that leave the range of 16 bits on the way."""

    T, B, H, D = 300, 1, 2, 64
    q, k = (_randn((T, B, H, D), s) .mul(size).to(dtype) for s in (1, 2))
    v = _randn((T, B, H, D), 3, dtype)
    scale = 1.0 / (size * size * D)
    first = None
    state, out = mb.decay_attention_forward(q, k, v, _decay(H), first, scale=scale)
    S, o = reference(q, k, v, _decay(H), None, scale)
    A_S, A_o = magnitude(q, k, v, _decay(H), None, scale)
    # fp16 keys of 1e-3 have weighted parts below its normal range: 2^-25 absolute
    floor = 2.0**-25 * T * float(v.abs().max()) if dtype == torch.float16 else 0.0
    check(out, o, out_bound(A_o, dtype, T, D) + floor * D * scale * float(q.abs().max()),
          "outputs")
    check(state.memory, S, memory_bound(A_S, dtype, T, D) + floor, "memory")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_are_read_in_place(dtype):
    T, B, H, D = 150, 3, 4, 64
    fused = _randn((T, B, 3, H, D), 1, dtype)
    q, k, v = fused.unbind(2)
    base = run_and_check(q, k, v, _decay(H), None, 0.125)
    for layout in ("batch_first", "odd_offset", "inner_stride"):
        def view(x):
            if layout == "batch_first":
                return x.permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3)
            if layout == "odd_offset":
                wide = torch.zeros((T, B, H, D + 3), dtype=dtype, device=DEV)
                wide[..., 1:D + 1] = x
                return wide[..., 1:D + 1]
            return x.transpose(-1, -2).contiguous().transpose(-1, -2)
        state, out = run_and_check(view(q), view(k), view(v), _decay(H), None, 0.125)
        if layout == "batch_first":  # the same kernel on other strides: the same bits
            assert torch.equal(out, base[1]) and torch.equal(state.memory, base[0].memory)


def test_shared_heads_and_broadcast_inputs():
    T, B, H, D = 140, 2, 4, 64
    q = _randn((T, B, H, D), 1, torch.bfloat16).requires_grad_(True)
    k1 = _randn((T, B, 1, D), 2, torch.bfloat16).requires_grad_(True)
    v1 = _randn((1, B, H, D), 3, torch.bfloat16).requires_grad_(True)
    run_and_check(q.detach(), k1.detach().expand(T, B, H, D), v1.detach().expand(T, B, H, D),
                  _decay(H), None, 0.1)
    _, out = mb.decay_attention_forward(q, k1.expand(T, B, H, D), v1.expand(T, B, H, D),
                                        _decay(H), scale=0.1)
    g = _randn(out.shape, 5, torch.bfloat16)
    dk, dv = torch.autograd.grad(out, [k1, v1], g)
    k2, v2 = (x.detach().double().requires_grad_(True) for x in (k1, v1))
    _, o = reference(q.detach(), k2.expand(T, B, H, D), v2.expand(T, B, H, D), _decay(H), None,
                     0.1)
    wk, wv = torch.autograd.grad(o, [k2, v2], g.double())
    # sums of H (of T) bf16 gradients, each within 4 u of its terms and summed in bf16's
    # own sum (fp32 inside, one rounding): bounded by the norms here
    assert dk.shape == k1.shape and dv.shape == v1.shape
    assert (dk.double() - wk).norm() <= 2.0**-7 * wk.norm()
    assert (dv.double() - wv).norm() <= 2.0**-7 * wv.norm()


GRAD_SHAPES = [(1, 1, 1, 8, 8), (5, 2, 2, 64, 32), (130, 2, 2, 64, 64), (129, 1, 2, 128, 72),
               (260, 2, 1, 40, 128), (61, 2, 3, 33, 65), (1200, 1, 1, 64, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", GRAD_SHAPES)
@pytest.mark.parametrize("ragged", [False, True])
def test_gradients_match_the_recurrence(shape, dtype, ragged):
    T, B, H, Dk, Dv = shape
    scale = Dk**-0.5
    lengths = None
    if ragged:
        lengths = torch.tensor([max(T - 3, 0), T][:B], dtype=torch.int32, device=DEV)
    leaves = [_randn((T, B, H, Dk), 1, dtype), _randn((T, B, H, Dk), 2, dtype),
              _randn((T, B, H, Dv), 3, dtype), _randn((B, H, Dk, Dv), 4)]
    go, gm = _randn((T, B, H, Dv), 5, dtype), _randn((B, H, Dk, Dv), 6)
    if ragged:  # gradients that arrive past a row's end are not used either
        go = go.masked_fill(~_live(T, lengths), float("nan"))
    mine = [x.clone().requires_grad_(True) for x in leaves]
    state, out = mb.decay_attention_forward(*mine[:3], _decay(H), mb.DecayAttentionState(mine[3]),
                                            scale=scale, lengths=lengths)
    got = torch.autograd.grad((out, state.memory), mine, (go, gm))

    def grads(values, g_out, g_mem):
        ls = [x.double().requires_grad_(True) for x in values]
        S, o = reference(*ls[:3], _decay(H), ls[3], scale, lengths)
        return torch.autograd.grad((o, S), ls, (torch.nan_to_num(g_out).double(),
                                                g_mem.double()))

    want = grads(leaves, go, gm)
    sizes = grads([x.abs() for x in leaves], go.abs(), gm.abs())
    for name, a, w, A in zip(("dq", "dk", "dv", "dmemory"), got, want, sizes):
        if name == "dmemory":
            check(a, w, memory_bound(A, dtype, T, max(Dk, Dv)), name)
        else:
            assert a.dtype == dtype
            check(a, w, out_bound(A, dtype, T, max(Dk, Dv)), name)


def test_gradients_match_differences():
    """The operator is linear in each input alone, so central differences are
    exact but for fp32 rounding of the outputs (about 2^-24 of their magnitude
    times their number, divided by the step)."""

    T, B, H, D = 40, 1, 2, 16
    xs = [_randn((T, B, H, D), s) for s in (1, 2, 3)] + [_randn((B, H, D, D), 4)]
    go, gm = _randn((T, B, H, D), 5), _randn((B, H, D, D), 6)

    def loss(vals):
        state, out = mb.decay_attention_forward(*vals[:3], _decay(H),
                                                mb.DecayAttentionState(vals[3]), scale=0.25)
        return ((out.double() * go.double()).sum() + (state.memory.double() * gm.double()).sum())

    mine = [x.clone().requires_grad_(True) for x in xs]
    grads = torch.autograd.grad(loss(mine), mine)
    for i, g in enumerate(grads):
        d = _randn(xs[i].shape, 20 + i)
        up, down = list(xs), list(xs)
        up[i], down[i] = xs[i] + d, xs[i] - d
        diff = (loss(up) - loss(down)) / 2
        inner = (g.double() * d.double()).sum()
        _, A = magnitude(*xs[:3], _decay(H), xs[3], 0.25)
        # rounding of the shifted inputs and of ~80 steps' sums, over all outputs
        assert (diff - inner).abs() <= 2.0**-24 * 400 * (A.norm() + gm.norm() * 40) * go.norm()


def test_only_requested_gradients_flow():
    T, B, H, D = 20, 1, 1, 16
    q, k, v = (_randn((T, B, H, D), s) for s in (1, 2, 3))
    v.requires_grad_(True)
    state, out = mb.decay_attention_forward(q, k, v, _decay(H), scale=1.0)
    (dv,) = torch.autograd.grad(state.memory.sum(), [v])  # no gradient from the outputs
    w = _decay(H).double() ** torch.arange(T - 1, -1, -1, device=DEV).double()
    want = (k.double().sum(-1)[:, 0, 0] * w)[:, None].expand(T, D)
    check(dv[:, 0, 0], want, 1e-4 * k.abs().sum(-1)[:, 0].double(), "dv")
    out, = [mb.decay_attention_forward(q, k, v.detach(), _decay(H))[1]]
    assert not out.requires_grad
    with pytest.raises(RuntimeError):  # a second derivative is refused, not wrong
        x = q.clone().requires_grad_(True)
        _, o = mb.decay_attention_forward(x, k, v.detach(), _decay(H))
        (dx,) = torch.autograd.grad(o.square().sum(), [x], create_graph=True)
        dx.sum().backward()


def test_empty_sizes():
    for T, B, H in ((0, 2, 3), (4, 0, 3), (4, 2, 0)):
        q, v = torch.zeros((T, B, H, 16), device=DEV), torch.zeros((T, B, H, 8), device=DEV)
        memory = torch.ones((B, H, 16, 8), device=DEV)
        state, out = mb.decay_attention_forward(q, q, v, torch.zeros(H, device=DEV),
                                                mb.DecayAttentionState(memory))
        assert out.shape == v.shape and state.memory.shape == memory.shape
        assert torch.equal(state.memory, memory)


STEP_SHAPES = [(1, 1, 1, 1), (1, 8, 64, 64), (3, 2, 33, 17), (2, 5, 128, 128), (40, 9, 128, 128),
               (2, 2, 256, 200), (70, 7, 40, 36), (1, 1, 7, 256)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", STEP_SHAPES)
@pytest.mark.parametrize("inplace", [False, True])
def test_step_matches_the_recurrence(shape, dtype, inplace):
    B, H, Dk, Dv = shape
    q, k = _randn((B, H, Dk), 1, dtype), _randn((B, H, Dk), 2, dtype)
    v, memory = _randn((B, H, Dv), 3, dtype), _randn((B, H, Dk, Dv), 4)
    before = memory.clone()
    active = torch.ones(B, dtype=torch.bool, device=DEV)
    active[B // 2] = B == 1
    state, out = mb.decay_attention_step(q, k, v, _decay(H), mb.DecayAttentionState(memory),
                                         scale=0.5, active=active, inplace=inplace)
    S, o = reference(q[None], k[None], v[None], _decay(H), before, 0.5, active.to(torch.int32))
    A_S, A_o = magnitude(q[None], k[None], v[None], _decay(H), before, 0.5)
    u = torch.finfo(dtype).eps / 2
    check(state.memory, S, 2.0**-22 * A_S, "memory")
    check(out, o[0], (u + (Dk + 8) * 2.0**-24) * A_o[0] + 2.0**-24 * (dtype == torch.float16),
          "outputs")
    assert (state.memory is memory) == inplace
    if not inplace:
        assert torch.equal(memory, before)


def test_steps_and_chunks_agree_over_a_sequence():
    """A prompt, then single steps, against the whole sequence at once."""

    T, P, B, H, D = 180, 150, 3, 2, 64
    q, k, v = (_randn((T, B, H, D), s, torch.bfloat16) for s in (1, 2, 3))
    S, o = reference(q, k, v, _decay(H), None, 0.125)
    A_S, A_o = magnitude(q, k, v, _decay(H), None, 0.125)
    state, out = mb.decay_attention_forward(q[:P], k[:P], v[:P], _decay(H), scale=0.125)
    outs = [out]
    for t in range(P, T):
        state, y = mb.decay_attention_step(q[t], k[t], v[t], _decay(H), state, scale=0.125,
                                           inplace=t % 2 == 0)
        outs.append(y[None])
    check(torch.cat(outs), o, out_bound(A_o, torch.bfloat16, T, D), "outputs")
    check(state.memory, S, memory_bound(A_S, torch.bfloat16, T, D), "memory")


def test_step_is_differentiable():
    B, H, D = 2, 2, 32
    xs = [_randn((B, H, D), s).requires_grad_(True) for s in (1, 2, 3)]
    m = _randn((B, H, D, D), 4).requires_grad_(True)
    active = torch.tensor([True, False], device=DEV)
    state, out = mb.decay_attention_step(*xs, _decay(H), mb.DecayAttentionState(m), active=active)
    got = torch.autograd.grad(out.sum() + state.memory.square().sum(), [*xs, m])
    ys = [x.detach().double().requires_grad_(True) for x in (*xs, m)]
    S, o = reference(ys[0][None], ys[1][None], ys[2][None], _decay(H), ys[3], 1.0,
                     active.to(torch.int32))
    want = torch.autograd.grad(o.sum() + S.square().sum(), ys)
    for a, w in zip(got, want):
        assert (a.double() - w).norm() <= 1e-5 * (1 + w.norm())


def test_another_stream_and_graph_replay():
    T, B, H, D = 200, 2, 2, 64
    decay = _decay(H)
    q, k, v = (_randn((T, B, H, D), s, torch.bfloat16) for s in (1, 2, 3))
    memory = torch.zeros((B, H, D, D), device=DEV)

    def work():
        state, out = mb.decay_attention_forward(q, k, v, decay, mb.DecayAttentionState(memory),
                                                scale=0.125)
        _, y = mb.decay_attention_step(q[0], k[0], v[0], decay, state, inplace=True)
        return out, y, state.memory

    eager = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for seed in (11, 12):
        for x, s in ((q, seed), (k, seed + 1), (v, seed + 2)):
            x.copy_(_randn(x.shape, s, torch.bfloat16))
        graph.replay()
        for a, b in zip(held, work()):
            assert torch.equal(a, b)


def test_inference_mode_and_versions():
    B, H, D = 1, 1, 16
    q, m = _randn((B, H, D), 1), _randn((B, H, D, D), 2)
    with torch.inference_mode():
        inner = torch.zeros((B, H, D, D), device=DEV)
        mb.decay_attention_step(q, q, q, _decay(H), mb.DecayAttentionState(inner), inplace=True)
    w = torch.ones((), device=DEV, requires_grad=True)
    y = (w * m).sum()  # saves m for its backward
    mb.decay_attention_step(q, q, q, _decay(H), mb.DecayAttentionState(m), inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_wait_timeout_is_reported():
    nat.device_status()
    nat.debug_wait_timeout(nat.MB_UNIT_ATTENTION)
    torch.cuda.synchronize()
    assert nat.device_status() == 1 and nat.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_and_heads_do_not_touch_one_another(dtype):
    """A row's result is the same bits whatever its neighbours hold, NaN included,
    and however many there are."""

    T, B, H, D = 300, 4, 3, 64
    q, k, v = (_randn((T, B, H, D), s, dtype) for s in (1, 2, 3))
    memory = _randn((B, H, D, D), 4)
    base, out = mb.decay_attention_forward(q, k, v, _decay(H), mb.DecayAttentionState(memory),
                                           scale=0.1)
    for x in (q, k, v):
        x[:, 1, 2] = float("nan")
        x[:, 3, 0] = float("inf")
    state, got = mb.decay_attention_forward(q, k, v, _decay(H), mb.DecayAttentionState(memory),
                                            scale=0.1)
    keep = torch.ones((B, H), dtype=torch.bool, device=DEV)
    keep[1, 2] = keep[3, 0] = False
    assert torch.equal(got[:, keep], out[:, keep])
    assert torch.equal(state.memory[keep], base.memory[keep])
    state, got = mb.decay_attention_forward(q[:, :1], k[:, :1], v[:, :1], _decay(H),
                                            mb.DecayAttentionState(memory[:1]), scale=0.1)
    assert torch.equal(got, out[:, :1]) and torch.equal(state.memory, base.memory[:1])


def test_a_later_value_does_not_reach_earlier_chunks():
    T, D = 400, 64
    q, k, v = (_randn((T, 1, 1, D), s, torch.bfloat16) for s in (1, 2, 3))
    _, out = mb.decay_attention_forward(q, k, v, _decay(1), scale=0.1)
    k2, v2 = k.clone(), v.clone()
    k2[300], v2[300] = float("nan"), float("inf")
    _, got = mb.decay_attention_forward(q, k2, v2, _decay(1), scale=0.1)
    assert torch.equal(got[:256], out[:256])  # chunks of 128 steps before the one that holds it
    assert not torch.isfinite(got[300:]).any()


def test_opcheck():
    T, B, H, D = 20, 2, 2, 16
    q, k, v = (_randn((T, B, H, D), s, torch.bfloat16) for s in (1, 2, 3))
    m, lengths = _randn((B, H, D, D), 4), torch.tensor([20, 7], dtype=torch.int32, device=DEV)
    args = (q, k, v, _decay(H), m, lengths, 0.5)
    torch.library.opcheck(cops.decay_attention_op, args)
    torch.library.opcheck(cops.decay_attention_backward_op,
                          (*args[:6], q, m, 0.5, True, False, True, True))
    step = (q[0], k[0], v[0], _decay(H), m, None, 0.5)
    torch.library.opcheck(cops.decay_attention_step_op, step)
    torch.library.opcheck(cops.decay_attention_step_inplace_op, step)


def test_compiled_layer_matches_eager():
    torch.manual_seed(0)
    layer = mb.DecayAttention(32, 2, 16).to(DEV)
    x = torch.randn((40, 2, 32), device=DEV)
    fast = torch.compile(layer, fullgraph=True)
    state, out = layer(x)
    state2, out2 = fast(x)
    assert (out - out2).abs().max() <= 1e-4 * out.abs().max()
    g1 = torch.autograd.grad(out.sum(), list(layer.parameters()), allow_unused=True)
    g2 = torch.autograd.grad(out2.sum(), list(layer.parameters()), allow_unused=True)
    for a, b in zip(g1, g2):
        assert (a - b).abs().max() <= 1e-4 * a.abs().max()


def test_calls_on_two_streams_at_once():
    """Split time axes with workspaces of their own, both in flight."""

    T, B, H, D = 4096, 1, 2, 64
    sets = [[_randn((T, B, H, D), s + 10 * i, torch.bfloat16) for s in (1, 2, 3)] for i in (0, 1)]
    want = [mb.decay_attention_forward(*x, _decay(H), scale=0.1) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for stream, x in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(mb.decay_attention_forward(*x, _decay(H), scale=0.1))
    torch.cuda.synchronize()
    for i, (state, out) in enumerate(got):
        assert torch.equal(out, want[i % 2][1])
        assert torch.equal(state.memory, want[i % 2][0].memory)


def test_training_step_in_a_graph():
    T, B, H, D = 150, 2, 2, 64
    q, k, v = (_randn((T, B, H, D), s, torch.bfloat16) for s in (1, 2, 3))
    go = _randn((T, B, H, D), 5, torch.bfloat16)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]

    def step():
        _, out = mb.decay_attention_forward(*leaves, decay, scale=0.1)
        return (out, *torch.autograd.grad(out, leaves, go))

    decay = _decay(H)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        leaves[0].copy_(_randn((T, B, H, D), 9, torch.bfloat16))
    graph.replay()
    held = [x.detach().clone() for x in held]
    for a, b in zip(held, step()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("B, H", [(30, 12), (37, 4), (128, 3), (129, 2)])
def test_many_ragged_rows_in_any_order(B, H):
    """More rows than SMs, ranked by length inside the kernel (up to 128 batch
    rows): each row's bits are those it has on its own; every output is written."""

    T, D = 400, 32
    g = _gen(7)
    lengths = torch.randint(0, T + 1, (B,), generator=g, device=DEV).to(torch.int32)
    lengths[B // 2 :: 5] = 128  # ties
    q, k, v, go = (_randn((T, B, H, D), s, torch.bfloat16) for s in (1, 2, 3, 5))
    first = mb.DecayAttentionState(_randn((B, H, D, D), 4))
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    torch.full((T, B, H, D), float("nan"), dtype=torch.bfloat16, device=DEV)  # stale memory
    state, out = mb.decay_attention_forward(*leaves, _decay(H), first, scale=0.2, lengths=lengths)
    grads = torch.autograd.grad(out, leaves, go)
    for b in range(0, B, 7):
        own = [x[:, b : b + 1].contiguous().requires_grad_(True) for x in (q, k, v)]
        s1, o1 = mb.decay_attention_forward(
            *own, _decay(H), mb.DecayAttentionState(first.memory[b : b + 1]), scale=0.2,
            lengths=lengths[b : b + 1])
        g1 = torch.autograd.grad(o1, own, go[:, b : b + 1].contiguous())
        assert torch.equal(out[:, b], o1[:, 0])
        assert torch.equal(state.memory[b], s1.memory[0])
        for x, y in zip(grads, g1):
            assert torch.equal(x[:, b], y[:, 0])
    live = _live(T, lengths)
    for x in (out, *grads):
        assert torch.equal(x.masked_fill(live, 0), torch.zeros_like(x))
