"""Argument checks of the decayed attention, without a GPU, and its compile-visible ops."""

from __future__ import annotations

import ctypes
import re

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import myelin_b200 as mb
from myelin_b200 import _native as nat


_MODE = FakeTensorMode(allow_non_fake_inputs=True)


def _fake(*shapes_dtypes):
    with _MODE:
        return [torch.empty(s, dtype=d, device="cuda") for s, d in shapes_dtypes]


def _operands(T=4, B=2, H=3, Dk=8, Dv=16, dtype=torch.bfloat16):
    return _fake(((T, B, H, Dk), dtype), ((T, B, H, Dk), dtype), ((T, B, H, Dv), dtype),
                 ((H,), torch.float32), ((B, H, Dk, Dv), torch.float32))


def test_cpu_tensors_are_refused():
    x = torch.zeros((4, 2, 3, 8))
    with pytest.raises(ValueError, match="CUDA devices only"):
        mb.decay_attention_forward(x, x, x, torch.ones(3))
    with pytest.raises(ValueError, match="CUDA devices only"):
        mb.decay_attention_step(x[0], x[0], x[0], torch.ones(3),
                                mb.DecayAttentionState(torch.zeros((2, 3, 8, 8))))


@pytest.mark.parametrize(
    "change, message",
    [
        (lambda a: a.update(q=a["q"][0]), r"queries must be shaped \[T, B, H, Dk\]"),
        (lambda a: a.update(k=a["k"][:3]), "keys must have the shape of queries"),
        (lambda a: a.update(v=a["v"][:, :1]), "values must match queries"),
        (lambda a: a.update(v=a["v"].float()), "values must have the same device and dtype"),
        (lambda a: a.update(q=a["q"].double(), k=a["k"].double(), v=a["v"].double()),
         "must be float32, bfloat16 or float16"),
        (lambda a: a.update(decay=a["decay"][:2]), r"decay must be shaped \[H\]"),
        (lambda a: a.update(decay=a["decay"].half()), "decay must be float32"),
        (lambda a: a.update(m=a["m"].half()), "state.memory must be float32"),
        (lambda a: a.update(m=a["m"].transpose(-1, -2)), "state.memory must be shaped"),
        (lambda a: a.update(lengths=a["lengths"].long()), "lengths must be int32"),
        (lambda a: a.update(lengths=a["lengths"][:1]), r"lengths must be shaped \[B\]"),
    ],
)
def test_forward_refusals(change, message):
    q, k, v, decay, m = _operands()
    (lengths,) = _fake(((2,), torch.int32))
    a = {"q": q, "k": k, "v": v, "decay": decay, "m": m, "lengths": lengths}
    with q.fake_mode:
        change(a)
    with pytest.raises(ValueError, match=message):
        mb.decay_attention_forward(a["q"], a["k"], a["v"], a["decay"],
                                   mb.DecayAttentionState(a["m"]), lengths=a["lengths"])


def test_head_sizes_and_decay_gradients_are_refused():
    q, k, v, decay, _ = _operands(Dk=257)
    with pytest.raises(ValueError, match=r"head sizes must be in \[1, 256\]"):
        mb.decay_attention_forward(q, k, v, decay)
    q, k, v, decay, _ = _operands()
    with q.fake_mode:
        decay = torch.empty((3,), device="cuda", requires_grad=True)
    with pytest.raises(NotImplementedError, match="decay is a constant"):
        mb.decay_attention_forward(q, k, v, decay)


def test_step_refusals():
    q, k, v, decay, m = _operands()
    with q.fake_mode:
        q, k, v = q[0], k[0], v[0]
        active = torch.empty((2,), dtype=torch.int32, device="cuda")
        strided = torch.empty((2, 3, 16, 8), device="cuda").transpose(-1, -2)
        leaf = torch.empty((2, 3, 8, 16), device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="active must be bool"):
        mb.decay_attention_step(q, k, v, decay, mb.DecayAttentionState(m), active=active)
    with pytest.raises(ValueError, match="contiguous state.memory"):
        mb.decay_attention_step(q, k, v, decay, mb.DecayAttentionState(strided), inplace=True)
    with pytest.raises(ValueError, match="cannot be differentiated"):
        mb.decay_attention_step(q, k, v, decay, mb.DecayAttentionState(leaf), inplace=True)


def test_traces_to_ops():
    def f(q, k, v, decay, m):
        state, out = mb.decay_attention_forward(q, k, v, decay, mb.DecayAttentionState(m))
        state, y = mb.decay_attention_step(q[0], k[0], v[0], decay, state)
        return out, y, state.memory

    args = _operands()
    gm = make_fx(f, tracing_mode="fake")(*args)
    ops = {str(n.target).split(".")[1] for n in gm.graph.nodes
           if n.op == "call_function" and str(n.target).startswith("myelin_b200.")}
    assert ops == {"decay_attention", "decay_attention_step"}
    with _MODE:
        out, y, memory = gm(*args)
    assert out.shape == (4, 2, 3, 16) and out.dtype == torch.bfloat16
    assert y.shape == (2, 3, 16) and memory.shape == (2, 3, 8, 16)


def _args(**kw):
    a = nat.DecayAttentionArgsC()
    a.dtype, a.T, a.B, a.H, a.Dk, a.Dv = nat.MB_BF16, 4, 2, 3, 8, 16
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize(
    "kw, message",
    [
        ({"dtype": nat.MB_I32}, "unsupported dtype"),
        ({"T": -1}, "negative size"),
        ({"Dk": 0}, "head sizes must be in"),
        ({"Dv": 300}, "head sizes must be in"),
        ({"B": 1 << 31}, "below 2\\^31"),
        ({}, "decay is null"),
        ({"decay": 4096}, "must not be null"),
    ],
)
def test_c_entry_reports_bad_arguments(kw, message):
    lib = nat.lib()
    args = _args(**kw)
    status = lib.mb_decay_attention(ctypes.addressof(args), None, 0, None)
    assert status != 0
    assert re.search(message, lib.mb_last_error().decode())


def test_packed_arguments_have_the_structures_layout():
    for packed, c in ((nat._ATTENTION_ARGS, nat.DecayAttentionArgsC),
                      (nat._ATTENTION_STEP_ARGS, nat.DecayAttentionStepArgsC)):
        assert packed.size == ctypes.sizeof(c)
    values = list(range(1, 36)) + [0.5, 0.25]
    a = nat.DecayAttentionArgsC.from_buffer_copy(nat._ATTENTION_ARGS.pack(*values))
    assert (a.dtype, a.reverse, a.T, a.Dv, a.q.data) == (1, 2, 3, 7, 8)
    assert (a.k.stride_t, a.o.stride_h, a.decay, a.lengths) == (13, 23, 24, 25)
    assert (a.first.data, a.last.stride_col, a.out_scale, a.kv_scale) == (26, 35, 0.5, 0.25)
    values = list(range(1, 20)) + [0.5]
    b = nat.DecayAttentionStepArgsC.from_buffer_copy(nat._ATTENTION_STEP_ARGS.pack(*values))
    assert [getattr(b, name) for name, _ in b._fields_] == values


def test_c_entry_empty_and_workspace():
    lib = nat.lib()
    assert lib.mb_decay_attention(ctypes.addressof(_args(B=0)), None, 0, None) == 0
    assert lib.mb_decay_attention(None, None, 0, None) != 0
    assert lib.mb_decay_attention_step(None, None) != 0
    one = _args(T=16384, B=1, H=1, Dk=256, Dv=256, dtype=nat.MB_F32)
    need = lib.mb_decay_attention_workspace_bytes(ctypes.addressof(one))
    assert need > 0 and need % (256 * 256 * 4) == 0  # whole memories, one per segment
    many = _args(T=16384, B=64, H=64, Dk=256, Dv=256)
    assert lib.mb_decay_attention_workspace_bytes(ctypes.addressof(many)) == 0
    # a workspace that is too small is refused before anything is launched
    one.decay = 4096
    one.q.data = one.k.data = one.v.data = one.o.data = 4096
    assert lib.mb_decay_attention(ctypes.addressof(one), None, 0, None) != 0
    assert "workspace" in lib.mb_last_error().decode()
    one.first.data = one.last.data = 8192  # the outputs read `first` after `last` is written
    assert lib.mb_decay_attention(ctypes.addressof(one), None, 0, None) != 0
    assert "must not be the buffer of first" in lib.mb_last_error().decode()
