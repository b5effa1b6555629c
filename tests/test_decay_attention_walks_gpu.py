"""Decayed attention where a CTA walks several (segment, row, head) units: every tile
layout, both 16-bit types, equal and ragged rows, with and without a first memory,
split and whole time axes. Rows are compared with their recurrence in 64 bits, by the
bounds of ``test_decay_attention_gpu``."""

from __future__ import annotations

import pytest
import torch

import myelin_b200 as mb
from myelin_b200 import _native as nat
from tests.test_decay_attention_gpu import (
    _gen, _live, _randn, check, magnitude, memory_bound, out_bound, reference)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _decays(H):
    return (1.0 - 1.0 / torch.logspace(1, 9, H, base=2.0, dtype=torch.float64)).float().to(DEV)


def run_and_check_rows(T, B, H, Dk, Dv, dtype, ragged, memory, rows):
    scale = Dk**-0.5
    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=_gen(7), device=DEV).to(torch.int32)
        lengths[rows[0]], lengths[rows[-1]] = T, T - 100
    leaves = [_randn((T, B, H, Dk), 1, dtype), _randn((T, B, H, Dk), 2, dtype),
              _randn((T, B, H, Dv), 3, dtype)]
    if memory:
        leaves.append(_randn((B, H, Dk, Dv), 4))
    go, gm = _randn((T, B, H, Dv), 5, dtype), _randn((B, H, Dk, Dv), 6)
    mine = [x.clone().requires_grad_(True) for x in leaves]
    first = mb.DecayAttentionState(mine[3]) if memory else None
    decay = _decays(H)
    state, out = mb.decay_attention_forward(*mine[:3], decay, first, scale=scale, lengths=lengths)
    got = torch.autograd.grad((out, state.memory), mine, (go, gm))
    assert nat.device_status() == 0

    def part(x):  # the compared rows of a [T, B, ...] tensor
        return x[:, rows]

    own = None if lengths is None else lengths[rows]
    values = [part(x) for x in leaves[:3]] + [x[rows] for x in leaves[3:]]

    def plain(parts, g_out, g_mem):
        ls = [x.detach().double().requires_grad_(True) for x in parts]
        S, o = reference(*ls[:3], decay, ls[3] if memory else None, scale, own)
        return (o.detach(), S.detach(), *torch.autograd.grad((o, S), ls, (g_out, g_mem)))

    want = plain(values, part(go).double(), gm[rows].double())
    sizes = plain([x.abs() for x in values], part(go).double().abs(), gm[rows].double().abs())
    mine_rows = [part(out), state.memory[rows], *(part(x) for x in got[:3]),
                 *(x[rows] for x in got[3:])]
    names = ["out", "memory", "dq", "dk", "dv", "dmemory"]
    for name, a, w, A in zip(names, mine_rows, want, sizes):
        D = max(Dk, Dv)
        bound = memory_bound(A, dtype, T, D) if "memory" in name else out_bound(A, dtype, T, D)
        check(a.detach(), w, bound, name)
    for x in (out.detach(), *got[:3]):
        assert torch.isfinite(x).all()
        if ragged:
            assert torch.equal(x.masked_fill(_live(T, lengths), 0), torch.zeros_like(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dk, Dv", [(64, 64), (64, 128), (128, 64), (128, 128), (40, 120)])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("memory", [False, True])
def test_several_units_per_cta(Dk, Dv, dtype, ragged, memory):
    run_and_check_rows(400, 37, 9, Dk, Dv, dtype, ragged, memory, [0, 11, 36])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dk, Dv", [(64, 64), (128, 128)])
@pytest.mark.parametrize("ragged", [False, True])
def test_split_time_axis_with_several_units_per_cta(Dk, Dv, dtype, ragged):
    T, B, H = 8192, 25, 2
    need = _workspace(T, B, H, Dk, Dv, dtype)
    segments = need // (4 * B * H * Dk * Dv)
    assert segments > 1 and segments * B * H > 148
    run_and_check_rows(T, B, H, Dk, Dv, dtype, ragged, True, [3, 20])


def _workspace(T, B, H, Dk, Dv, dtype):
    x = torch.empty(16, dtype=dtype, device=DEV)
    k, v = (T, *(B * H * Dk, H * Dk, Dk)), (T, *(B * H * Dv, H * Dv, Dv))
    args = nat._ATTENTION_ARGS.pack(
        nat.dtype_code(dtype), 0, T, B, H, Dk, Dv, x.data_ptr(), *k[1:], x.data_ptr(), *k[1:],
        x.data_ptr(), *v[1:], x.data_ptr(), *v[1:], x.data_ptr(), 0, *nat._NO_MEMORY,
        *nat._NO_MEMORY, 1.0, 1.0)
    return nat.lib().mb_decay_attention_workspace_bytes(args)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T, B, H", [(200, 3, 2), (200, 80, 4), (5, 3, 2), (9000, 1, 2)])
def test_no_row_has_a_step(T, B, H, dtype):
    """Lengths that leave every row empty, NaN everywhere behind them."""

    D = 64
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    leaves = [torch.full((T, B, H, D), float("nan"), dtype=dtype, device=DEV) for _ in range(3)]
    leaves.append(_randn((B, H, D, D), 4))
    leaves = [x.requires_grad_(True) for x in leaves]
    state, out = mb.decay_attention_forward(*leaves[:3], _decays(H),
                                            mb.DecayAttentionState(leaves[3]), lengths=lengths)
    gm = _randn((B, H, D, D), 6)
    got = torch.autograd.grad((out, state.memory), leaves, (torch.full_like(out, float("nan")), gm))
    assert torch.equal(state.memory, leaves[3]) and torch.equal(got[3], gm)
    for x in (out, *got[:3]):
        assert torch.count_nonzero(x) == 0
    assert nat.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_overlapping_windows_are_read_in_place(dtype):
    """Steps that overlap in memory (a sliding window over one recording)."""

    T, B, H, D = 150, 2, 2, 64
    base = _randn((T * 16 + B * H * D,), 1, dtype)
    view = base.as_strided((T, B, H, D), (16, H * D, D, 1))
    want = mb.decay_attention_forward(*(view.contiguous(),) * 3, _decays(H), scale=0.01)
    got = mb.decay_attention_forward(view, view, view, _decays(H), scale=0.01)
    assert torch.equal(got[1], want[1]) and torch.equal(got[0].memory, want[0].memory)
