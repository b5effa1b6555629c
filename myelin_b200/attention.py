"""Attention with a decay for each head: a leaky associative memory over time.

A head keeps a matrix memory that leaks like a membrane and stores one outer
product per time step, read by the step's query:

    S_t = decay[h] * S_{t-1} + k_t v_t^T          o_t = scale * q_t^T S_t

The layout is the scans': time-major ``[T, B, H, D]``, states ``[B, ...]``
carried between calls. ``decay_attention_forward`` runs whole sequences
(prompts, training windows) in chunks, ``decay_attention_step`` one time step
over a batch of memories. Both run hand-written CUDA kernels and need CUDA
tensors. The reference has no counterpart.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from myelin_b200 import _native as nat
from myelin_b200 import compile_ops as cops
from myelin_b200.autograd import DecayAttentionFunction, refuse_tangents, wants_grad

MAX_HEAD_SIZE = 256


@dataclass(frozen=True)
class DecayAttentionState:
    """Memories carried between calls: fp32 ``[B, H, Dk, Dv]``."""

    memory: torch.Tensor


def _validate(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
              decay: torch.Tensor, lead: str) -> None:
    """Shapes, devices and dtypes of the operands; ``lead`` names the dimensions
    in front of the head size ("T, B, H" or "B, H")."""

    # the usual call passes these few comparisons; only a refused one goes on to say why
    dtype, device, shape = queries.dtype, queries.device, queries.shape
    dims = lead.count(",") + 2
    if (
        len(shape) == dims and keys.shape == shape and values.shape[:-1] == shape[:-1]
        and 1 <= shape[-1] <= MAX_HEAD_SIZE and 1 <= values.shape[-1] <= MAX_HEAD_SIZE
        and queries.is_cuda and keys.device == device and values.device == device
        and dtype in nat.SCAN_DTYPES and keys.dtype == dtype and values.dtype == dtype
        and decay.shape == (shape[-2],) and decay.dtype == torch.float32
        and decay.device == device and not decay.requires_grad
    ):
        return
    for name, t, size in (("queries", queries, "Dk"), ("keys", keys, "Dk"),
                          ("values", values, "Dv")):
        if t.ndim != dims:
            raise ValueError(f"{name} must be shaped [{lead}, {size}]; got {tuple(t.shape)}")
    if keys.shape != queries.shape:
        raise ValueError(
            "keys must have the shape of queries; "
            f"got {tuple(keys.shape)} and {tuple(queries.shape)}"
        )
    if values.shape[:-1] != queries.shape[:-1]:
        raise ValueError(
            f"values must match queries in [{lead}]; "
            f"got {tuple(values.shape)} and {tuple(queries.shape)}"
        )
    for name, t in (("queries", queries), ("values", values)):
        if not 1 <= t.shape[-1] <= MAX_HEAD_SIZE:
            raise ValueError(
                f"head sizes must be in [1, {MAX_HEAD_SIZE}]; {name} have {t.shape[-1]}")
    nat.require_cuda(queries, "queries")
    for name, t in (("keys", keys), ("values", values)):
        if t.device != queries.device or t.dtype != queries.dtype:
            raise ValueError(f"{name} must have the same device and dtype as queries")
    if queries.dtype not in nat.SCAN_DTYPES:
        raise ValueError(
            "queries, keys and values must be float32, bfloat16 or float16; "
            f"got {queries.dtype}"
        )
    if decay.shape != (queries.shape[-2],):
        raise ValueError(f"decay must be shaped [H]; got {tuple(decay.shape)}")
    if decay.device != queries.device or decay.dtype != torch.float32:
        raise ValueError("decay must be float32 on the same device as queries")
    if decay.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(
            "decay is a constant of the operator and has no gradient; pass decay.detach()")


def _validate_memory(memory: torch.Tensor, shape: tuple[int, ...], device: torch.device) -> None:
    if tuple(memory.shape) != shape:
        raise ValueError(
            f"state.memory must be shaped [B, H, Dk, Dv] = {shape}; got {tuple(memory.shape)}")
    if memory.device != device:
        raise ValueError("state.memory must be on the same device as queries")
    if memory.dtype != torch.float32:
        raise ValueError(f"state.memory must be float32; got {memory.dtype}")


def decay_attention_forward(
    queries: torch.Tensor,
    keys: torch.Tensor,
    values: torch.Tensor,
    decay: torch.Tensor,
    initial_state: DecayAttentionState | None = None,
    *,
    scale: float = 1.0,
    lengths: torch.Tensor | None = None,
) -> tuple[DecayAttentionState, torch.Tensor]:
    """Whole sequences: queries, keys ``[T, B, H, Dk]``, values ``[T, B, H, Dv]``.

    ``decay`` is fp32 ``[H]`` on the device, each value in [0, 1] (not checked:
    that would read it back; a memory with a larger one grows, and what a
    negative one gives is not defined).
    ``initial_state`` is zero without one. ``lengths`` (int32 ``[B]`` on the
    device, clamped to [0, T]) ends each batch row early: steps past it leave
    the memory alone, give zero outputs and zero gradients, and what the inputs
    hold there (NaN included) is never used. Returns the state after each row's
    last step and the outputs ``[T, B, H, Dv]`` in the inputs' dtype; sums and
    memories are fp32. From 16 steps on, 16-bit inputs run on the tensor cores
    (heads up to 128), which round the weighed scores and the carried memory to
    the inputs' dtype where they read them: the outputs' error is then 1.4 times
    that of one rounding. A row's bits may also depend on the batch's size, which
    chooses how the time axis is split.

    Gradients flow to queries, keys, values and the initial memory, from the
    outputs and the final memory. Any strides are read in place when the head
    dimension is contiguous, so a shared head may be passed as
    ``keys.expand(...)``. A non-finite value of one step also reaches the
    outputs of up to 127 earlier steps of its row and head, which are formed
    together with it.
    """

    _validate(queries, keys, values, decay, "T, B, H")
    T, B, H, Dk = queries.shape
    memory = None
    if initial_state is not None:
        memory = initial_state.memory
        _validate_memory(memory, (B, H, Dk, values.shape[3]), queries.device)
    if lengths is not None:
        if lengths.shape != (B,):
            raise ValueError(f"lengths must be shaped [B]; got {tuple(lengths.shape)}")
        if lengths.device != queries.device or lengths.dtype != torch.int32:
            raise ValueError("lengths must be int32 on the same device as queries")
        lengths = lengths.contiguous()
    decay = decay.contiguous()
    refuse_tangents("decayed attention", queries, keys, values, memory, decay)
    if wants_grad(queries, keys, values, memory):
        out, last = DecayAttentionFunction.apply(queries, keys, values, decay, memory, lengths,
                                                 float(scale))
    else:
        out, last = cops.decay_attention(queries, keys, values, decay, memory, lengths, scale)
    return DecayAttentionState(memory=last), out


def decay_attention_step(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    decay: torch.Tensor,
    state: DecayAttentionState,
    *,
    scale: float = 1.0,
    active: torch.Tensor | None = None,
    inplace: bool = False,
) -> tuple[DecayAttentionState, torch.Tensor]:
    """One time step: query, key ``[B, H, Dk]``, value ``[B, H, Dv]``.

    Returns the new state and the outputs ``[B, H, Dv]``. ``active`` (bool
    ``[B]`` on the device) leaves the memories of rows that are False alone and
    gives them zero outputs (a padded batch). With ``inplace`` the state's own
    memory is updated, which then has to be contiguous and outside the autograd
    graph. When a gradient is asked for, the step is a sequence of length one.
    """

    _validate(query, key, value, decay, "B, H")
    B, H, Dk = query.shape
    memory = state.memory
    _validate_memory(memory, (B, H, Dk, value.shape[2]), query.device)
    if active is not None:
        if active.shape != (B,):
            raise ValueError(f"active must be shaped [B]; got {tuple(active.shape)}")
        if active.device != query.device or active.dtype != torch.bool:
            raise ValueError("active must be bool on the same device as query")
        active = active.contiguous()
    decay = decay.contiguous()
    refuse_tangents("decayed attention", query, key, value, memory, decay)
    graph = wants_grad(query, key, value, memory)
    if inplace:
        if graph:
            raise ValueError("inplace=True cannot be differentiated; use inplace=False")
        if not memory.is_contiguous():
            raise ValueError("inplace=True needs a contiguous state.memory")
        out = cops.decay_attention_step_(query, key, value, decay, memory, active, scale)
        return state, out
    if graph:
        lengths = None if active is None else active.to(torch.int32)
        last, out = decay_attention_forward(
            query.unsqueeze(0), key.unsqueeze(0), value.unsqueeze(0), decay, state, scale=scale,
            lengths=lengths)
        return last, out[0]
    out, last = cops.decay_attention_step(query, key, value, decay, memory, active, scale)
    return DecayAttentionState(memory=last), out
