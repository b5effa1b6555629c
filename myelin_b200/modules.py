"""nn.Module API of the hot path, constructor-compatible with ``myelin.modules``.

Mirrors LinearSynapse, the LIF/ALIF cells, TimeUnroll, LinearLIF,
LinearSurrogateLIF, LinearSurrogateLIFRate, RateReadoutClassifier and
LinearSurrogateLIFPacked of src/myelin/modules.py (same constructor
arguments, parameter names, shapes and default initialisation). Every
time-unrolled forward runs the CUDA scan; a single cell step is a scan of
length one.
"""

from __future__ import annotations

import math
from typing import Literal

import torch
from torch import nn

from myelin_b200.attention import (
    DecayAttentionState,
    decay_attention_forward,
    decay_attention_step,
)
from myelin_b200.checkpointing import CheckpointSize
from myelin_b200.compile_ops import i8_operand, next_seed
from myelin_b200.dropout import spike_dropout
from myelin_b200.kernels import (
    izhikevich_step,
    Backend,
    alif_forward,
    linear_surrogate_lif_forward,
    linear_surrogate_lif_packed_forward,
    linear_surrogate_lif_rate_forward,
    lif_forward,
    surrogate_alif_forward,
    surrogate_lif_forward,
)
from myelin_b200.neurons import (
    ALIFParams,
    ALIFState,
    IzhikevichParams,
    IzhikevichState,
    LIFParams,
    LIFState,
)
from myelin_b200.packing import PackedSpikes
from myelin_b200.quantized import QuantizedWeight, quantize_weight, quantized_linear
from myelin_b200.surrogates import (
    SurrogateFn,
    atan_surrogate,
    fast_sigmoid_surrogate,
    surrogate_name,
)


class LinearSynapse(nn.Module):
    """Trainable dense projection over time-major inputs (src/myelin/modules.py:112-133).

    ``weight`` is ``[in_features, out_features]`` and the projection is
    ``inputs @ weight + bias``.
    """

    def __init__(
        self,
        in_features: int,
        out_features: int,
        params: LIFParams | None = None,
        bias: bool = True,
    ) -> None:
        super().__init__()
        self.weight = nn.Parameter((torch.rand((in_features, out_features)) - 0.5) * 0.02)
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features))
        else:
            self.register_parameter("bias", None)

    def forward(self, inputs: torch.Tensor) -> torch.Tensor:
        output = torch.matmul(inputs, self.weight)
        if self.bias is not None:
            output = output + self.bias
        return output


def _keep_fp32(before: torch.Tensor, after: torch.Tensor) -> torch.Tensor:
    """A buffer after its module was moved or cast: ``after``, or where that was cast,
    ``before`` on its device."""

    return after if after.dtype == torch.float32 else before.to(after.device)


class QuantizedLinearSynapse(nn.Module):
    """A ``LinearSynapse`` for inference in 8-bit integers (``quantized_linear``).

    Holds the weight as int8 with one scale per output neuron; float inputs are
    quantised by rows on the way in, bool and int8 spikes are taken as they are.
    Spikes given as bool come out in the bias's dtype (float32 without a bias).
    """

    def __init__(self, weight: QuantizedWeight, bias: torch.Tensor | None = None) -> None:
        super().__init__()
        self.register_buffer("data", weight.data)
        self.register_buffer("scale", weight.scale)
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    @classmethod
    def from_synapse(cls, synapse: LinearSynapse) -> "QuantizedLinearSynapse":
        return cls(quantize_weight(synapse.weight.detach()), synapse.bias)

    def _apply(self, fn, recurse=True):
        # a change of dtype is for the bias; the scales stay fp32
        scale = self.scale
        super()._apply(fn, recurse)
        self.scale = _keep_fp32(scale, self.scale)
        self.data = i8_operand(self.data)  # a move to another device drops the row pitch
        return self

    def forward(self, inputs: torch.Tensor) -> torch.Tensor:
        weight = QuantizedWeight(self.data, self.scale)
        out_dtype = None
        if not inputs.dtype.is_floating_point and self.bias is not None:
            out_dtype = self.bias.dtype
        return quantized_linear(inputs, weight, self.bias, out_dtype=out_dtype)


class LIFCell(nn.Module):
    """Single-step hard-reset LIF population."""

    def __init__(self, params: LIFParams | None = None) -> None:
        super().__init__()
        self.params = params or LIFParams()

    def forward(self, state: LIFState, input_current: torch.Tensor) -> tuple[LIFState, torch.Tensor]:
        if state.membrane.shape != input_current.shape:
            raise ValueError(
                "state.membrane and input_current must have the same shape; "
                f"got {tuple(state.membrane.shape)} and {tuple(input_current.shape)}"
            )
        new_state, spikes = lif_forward(input_current.unsqueeze(0), state, self.params)
        return new_state, spikes[0]


class ALIFCell(nn.Module):
    """Single-step adaptive LIF population."""

    def __init__(self, params: ALIFParams | None = None) -> None:
        super().__init__()
        self.params = params or ALIFParams()

    def forward(
        self, state: ALIFState, input_current: torch.Tensor
    ) -> tuple[ALIFState, torch.Tensor]:
        new_state, spikes = alif_forward(input_current.unsqueeze(0), state, self.params)
        return new_state, spikes[0]


class IzhikevichCell(nn.Module):
    """Single-step Izhikevich-style population (src/myelin/modules.py:175-208)."""

    def __init__(self, params: IzhikevichParams | None = None) -> None:
        super().__init__()
        self.params = params or IzhikevichParams()

    def forward(
        self, state: IzhikevichState, input_current: torch.Tensor
    ) -> tuple[IzhikevichState, torch.Tensor]:
        return izhikevich_step(state, input_current, self.params)


class SurrogateLIFCell(nn.Module):
    """Single-step LIF with hard-forward surrogate-gradient spikes (src/myelin/modules.py:211-239)."""

    def __init__(
        self,
        params: LIFParams | None = None,
        surrogate: SurrogateFn = atan_surrogate,
        surrogate_slope: float = 10.0,
        hard_forward: bool = True,
    ) -> None:
        super().__init__()
        self.params = params or LIFParams()
        self.surrogate = surrogate
        self.surrogate_slope = surrogate_slope
        self.hard_forward = hard_forward

    def forward(self, state: LIFState, input_current: torch.Tensor) -> tuple[LIFState, torch.Tensor]:
        new_state, spikes = surrogate_lif_forward(
            input_current.unsqueeze(0),
            state,
            self.params,
            surrogate=surrogate_name(self.surrogate),
            surrogate_slope=self.surrogate_slope,
            hard_forward=self.hard_forward,
        )
        return new_state, spikes[0]


class SurrogateALIFCell(nn.Module):
    """Single-step ALIF with hard-forward surrogate-gradient spikes (src/myelin/modules.py:242-272)."""

    def __init__(
        self,
        params: ALIFParams | None = None,
        surrogate: SurrogateFn = atan_surrogate,
        surrogate_slope: float = 10.0,
        hard_forward: bool = True,
    ) -> None:
        super().__init__()
        self.params = params or ALIFParams()
        self.surrogate = surrogate
        self.surrogate_slope = surrogate_slope
        self.hard_forward = hard_forward

    def forward(
        self, state: ALIFState, input_current: torch.Tensor
    ) -> tuple[ALIFState, torch.Tensor]:
        new_state, spikes = surrogate_alif_forward(
            input_current.unsqueeze(0),
            state,
            self.params,
            surrogate=surrogate_name(self.surrogate),
            surrogate_slope=self.surrogate_slope,
            hard_forward=self.hard_forward,
        )
        return new_state, spikes[0]


class TimeUnroll(nn.Module):
    """Apply a cell across ``[T, B, N]`` inputs in one fused scan (src/myelin/modules.py:415-582)."""

    def __init__(self, cell: nn.Module, *, backend: Backend = "torch") -> None:
        super().__init__()
        self.cell = cell
        self.backend: Backend = backend

    def forward(
        self,
        inputs: torch.Tensor,
        initial_state: LIFState | ALIFState | None = None,
    ) -> tuple[LIFState | ALIFState, torch.Tensor]:
        cell = self.cell
        alif = isinstance(cell, ALIFCell | SurrogateALIFCell)
        if initial_state is None:
            zeros = torch.zeros(inputs.shape[1:], dtype=inputs.dtype, device=inputs.device)
            if alif:
                initial_state = ALIFState(membrane=zeros, adaptation=torch.zeros_like(zeros))
            else:
                initial_state = LIFState(membrane=zeros)
        if isinstance(cell, LIFCell):
            if not isinstance(initial_state, LIFState):
                raise TypeError("LIFCell requires LIFState")
            return lif_forward(inputs, initial_state, cell.params, backend=self.backend)
        if isinstance(cell, ALIFCell):
            if not isinstance(initial_state, ALIFState):
                raise TypeError("ALIFCell requires ALIFState")
            return alif_forward(inputs, initial_state, cell.params, backend=self.backend)
        if isinstance(cell, SurrogateALIFCell):
            if not isinstance(initial_state, ALIFState):
                raise TypeError("SurrogateALIFCell requires ALIFState")
            return surrogate_alif_forward(
                inputs,
                initial_state,
                cell.params,
                surrogate=surrogate_name(cell.surrogate),
                surrogate_slope=cell.surrogate_slope,
                hard_forward=cell.hard_forward,
                backend=self.backend,
            )
        if isinstance(cell, SurrogateLIFCell):
            if not isinstance(initial_state, LIFState):
                raise TypeError("SurrogateLIFCell requires LIFState")
            return surrogate_lif_forward(
                inputs,
                initial_state,
                cell.params,
                surrogate=surrogate_name(cell.surrogate),
                surrogate_slope=cell.surrogate_slope,
                hard_forward=cell.hard_forward,
                backend=self.backend,
            )
        raise TypeError(f"TimeUnroll does not support cell type {type(cell).__name__}")


class LinearLIF(nn.Module):
    """``LinearSynapse`` followed by ``TimeUnroll(LIFCell)``."""

    def __init__(self, in_features: int, out_features: int, params: LIFParams | None = None) -> None:
        super().__init__()
        self.synapse = LinearSynapse(in_features, out_features)
        self.unroll = TimeUnroll(LIFCell(params))

    def forward(self, inputs: torch.Tensor) -> tuple[LIFState, torch.Tensor]:
        return self.unroll(self.synapse(inputs))


class LinearSurrogateLIF(nn.Module):
    """Dense projection plus surrogate LIF unroll (src/myelin/modules.py:706-750)."""

    def __init__(
        self,
        in_features: int,
        out_features: int,
        params: LIFParams | None = None,
        surrogate: SurrogateFn = atan_surrogate,
        surrogate_slope: float = 10.0,
        hard_forward: bool = True,
        bias: bool = True,
        backend: Backend = "torch",
        stream_synapse: bool = False,
        checkpoint_size: CheckpointSize | None = None,
    ) -> None:
        super().__init__()
        self.synapse = LinearSynapse(in_features, out_features, bias=bias)
        self.stream_synapse = stream_synapse
        self.checkpoint_size: CheckpointSize | None = checkpoint_size
        self.unroll = TimeUnroll(
            SurrogateLIFCell(params, surrogate, surrogate_slope, hard_forward), backend=backend
        )

    def forward(self, inputs: torch.Tensor) -> torch.Tensor:
        cell = self.unroll.cell
        # (a quantised synapse has no float weight for the fused function)
        if self.stream_synapse and not isinstance(self.synapse, QuantizedLinearSynapse):
            _state, spikes = linear_surrogate_lif_forward(
                inputs,
                self.synapse.weight,
                self.synapse.bias,
                cell.params,
                surrogate=surrogate_name(cell.surrogate),
                surrogate_slope=cell.surrogate_slope,
                hard_forward=cell.hard_forward,
                backend=self.unroll.backend,
                checkpoint_size=self.checkpoint_size,
            )
            return spikes
        _state, spikes = self.unroll(self.synapse(inputs))
        return spikes


class LinearSurrogateLIFRate(nn.Module):
    """Dense projection plus surrogate LIF returning spike rates (src/myelin/modules.py:803-845)."""

    def __init__(
        self,
        in_features: int,
        out_features: int,
        params: LIFParams | None = None,
        surrogate: SurrogateFn = atan_surrogate,
        surrogate_slope: float = 10.0,
        hard_forward: bool = True,
        bias: bool = True,
        backend: Backend = "torch",
        checkpoint_size: CheckpointSize = 25,
        reduction: Literal["mean", "none"] = "none",
    ) -> None:
        super().__init__()
        self.synapse = LinearSynapse(in_features, out_features, bias=bias)
        self.cell = SurrogateLIFCell(params, surrogate, surrogate_slope, hard_forward)
        self.backend: Backend = backend
        self.checkpoint_size: CheckpointSize = checkpoint_size
        self.reduction: Literal["mean", "none"] = reduction

    def forward(self, inputs: torch.Tensor) -> torch.Tensor:
        _state, rates = linear_surrogate_lif_rate_forward(
            inputs,
            self.synapse.weight,
            self.synapse.bias,
            self.cell.params,
            surrogate=surrogate_name(self.cell.surrogate),
            surrogate_slope=self.cell.surrogate_slope,
            hard_forward=self.cell.hard_forward,
            backend=self.backend,
            checkpoint_size=self.checkpoint_size,
            reduction=self.reduction,
        )
        return rates


class SpikeDropout(nn.Module):
    """``spike_dropout`` with its own seed and a count of its calls.

    ``rng`` (int64 buffer: seed, calls so far) moves and is saved with the
    module; each call in training mode takes the next offset on the device, so a
    captured graph draws a new mask at every replay. With ``time_shared`` (the
    default) all steps of a ``[T, ...]`` input use one mask.

    A call that activation checkpointing runs again in the backward pass has to draw
    the same mask: take its seed first and pass it,
    ``checkpoint(dropout, x, dropout.next_seed())``. Without one the second run is
    refused. A copy of the module (``copy.deepcopy``) draws the same masks as the
    original, and a wrapper that broadcasts buffers from rank 0 (as
    ``DistributedDataParallel`` does) makes all ranks draw the same: where they
    should differ, give each its own first word, ``dropout.rng[0] = ...``, and keep
    the buffer out of the broadcast.
    """

    def __init__(self, p: float = 0.5, *, time_shared: bool = True,
                 seed: int | None = None) -> None:
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability must be in [0, 1]; got {p}")
        self.p = p
        self.time_shared = time_shared
        first = int(torch.randint(2**62, (), device="cpu")) if seed is None else seed
        self.register_buffer("rng", torch.tensor([first, 0], dtype=torch.int64))

    def next_seed(self) -> torch.Tensor:
        """The (seed, offset) of the next call, which is then counted as made."""

        return next_seed(self.rng)

    def forward(self, inputs: torch.Tensor, seed: torch.Tensor | None = None) -> torch.Tensor:
        """With ``seed`` (from ``next_seed``) the mask is that seed's and no call is counted."""

        if not self.training or self.p == 0.0:
            return inputs
        if seed is None:
            seed = self.next_seed()  # this call's own: its backward draws from it again
        return spike_dropout(inputs, self.p, seed, time_shared=self.time_shared)

    def extra_repr(self) -> str:
        return f"p={self.p}, time_shared={self.time_shared}"


def _drop(dropout: nn.Module, inputs: torch.Tensor, seed: torch.Tensor | None) -> torch.Tensor:
    if seed is None:
        return dropout(inputs)
    if not isinstance(dropout, SpikeDropout):
        raise ValueError(f"dropout_seed needs a SpikeDropout; got {type(dropout).__name__}")
    return dropout(inputs, seed)


class DecayAttention(nn.Module):
    """A layer of leaky associative memories: projections to queries, keys and values,
    attention with a decay for each head, dropout and an output projection.

    Each head's memory leaks with its own time constant, spaced evenly in the
    logarithm from ``tau_min`` to ``tau_max`` steps (decay ``1 - 1 / tau``, as
    ``LIFParams.decay``). ``forward`` takes ``[T, B, in_features]`` and carries the
    memories from ``initial_state`` to the state it returns; ``step`` takes one
    time step ``[B, in_features]``. Dropout (``SpikeDropout``, one mask for all
    steps) applies in training mode, in ``forward`` only; under activation
    checkpointing pass ``dropout_seed=layer.dropout.next_seed()``.
    """

    def __init__(
        self,
        in_features: int,
        heads: int,
        key_size: int,
        value_size: int | None = None,
        out_features: int | None = None,
        *,
        tau_min: float = 4.0,
        tau_max: float = 512.0,
        dropout: float = 0.0,
        bias: bool = True,
    ) -> None:
        super().__init__()
        if heads < 1 or key_size < 1:
            raise ValueError("heads and key_size must be at least 1")
        if not 1.0 <= tau_min <= tau_max:
            raise ValueError("tau_min must be at least 1 and tau_max at least tau_min")
        self.heads, self.key_size = heads, key_size
        self.value_size = key_size if value_size is None else value_size
        width = heads * self.value_size
        self.queries = LinearSynapse(in_features, heads * key_size, bias=bias)
        self.keys = LinearSynapse(in_features, heads * key_size, bias=bias)
        self.values = LinearSynapse(in_features, width, bias=bias)
        self.output = LinearSynapse(width, in_features if out_features is None else out_features,
                                    bias=bias)
        self.dropout = SpikeDropout(dropout)
        tau = torch.logspace(math.log2(tau_min), math.log2(tau_max), heads, base=2.0,
                             dtype=torch.float64)
        self.register_buffer("decay", (1.0 - 1.0 / tau).float())

    def _apply(self, fn, recurse=True):
        # a change of dtype is for the projections; decays stay fp32
        decay = self.decay
        super()._apply(fn, recurse)
        self.decay = _keep_fp32(decay, self.decay)
        return self

    def _heads(self, inputs: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        lead = inputs.shape[:-1]
        return (self.queries(inputs).view(*lead, self.heads, self.key_size),
                self.keys(inputs).view(*lead, self.heads, self.key_size),
                self.values(inputs).view(*lead, self.heads, self.value_size))

    def forward(
        self,
        inputs: torch.Tensor,
        initial_state: DecayAttentionState | None = None,
        lengths: torch.Tensor | None = None,
        dropout_seed: torch.Tensor | None = None,
    ) -> tuple[DecayAttentionState, torch.Tensor]:
        q, k, v = self._heads(inputs)
        state, out = decay_attention_forward(q, k, v, self.decay, initial_state,
                                             scale=self.key_size**-0.5, lengths=lengths)
        return state, self.output(_drop(self.dropout, out.flatten(-2), dropout_seed))

    def step(
        self,
        inputs: torch.Tensor,
        state: DecayAttentionState,
        active: torch.Tensor | None = None,
        *,
        inplace: bool = False,
    ) -> tuple[DecayAttentionState, torch.Tensor]:
        q, k, v = self._heads(inputs)
        state, out = decay_attention_step(q, k, v, self.decay, state, scale=self.key_size**-0.5,
                                          active=active, inplace=inplace)
        return state, self.output(out.flatten(-2))


class RateReadoutClassifier(nn.Module):
    """Hidden streamed LIF layer plus a rate readout (src/myelin/modules.py:848-903).

    ``time_shared_dropout`` drops hidden neurons for the whole window
    (``SpikeDropout``) instead of per step (``nn.Dropout``); under activation
    checkpointing pass ``dropout_seed=net.dropout.next_seed()`` with it.
    """

    def __init__(
        self,
        in_features: int,
        hidden_features: int,
        out_features: int,
        params: LIFParams | None = None,
        *,
        surrogate: SurrogateFn = fast_sigmoid_surrogate,
        surrogate_slope: float = 5.0,
        hard_forward: bool = True,
        bias: bool = True,
        backend: Backend = "torch",
        checkpoint_size: CheckpointSize = 25,
        dropout: float = 0.0,
        time_shared_dropout: bool = False,
    ) -> None:
        super().__init__()
        self.hidden = LinearSurrogateLIF(
            in_features,
            hidden_features,
            params,
            surrogate=surrogate,
            surrogate_slope=surrogate_slope,
            hard_forward=hard_forward,
            bias=bias,
            backend=backend,
            stream_synapse=True,
            checkpoint_size=checkpoint_size,
        )
        self.dropout = SpikeDropout(dropout) if time_shared_dropout else nn.Dropout(dropout)
        self.output = LinearSurrogateLIFRate(
            hidden_features,
            out_features,
            params,
            surrogate=surrogate,
            surrogate_slope=surrogate_slope,
            hard_forward=hard_forward,
            bias=bias,
            backend=backend,
            checkpoint_size=checkpoint_size,
            reduction="none",
        )

    def forward(
        self, inputs: torch.Tensor, dropout_seed: torch.Tensor | None = None
    ) -> torch.Tensor:
        hidden_spikes = _drop(self.dropout, self.hidden(inputs), dropout_seed)
        return self.output(hidden_spikes)


class LinearSurrogateLIFPacked(nn.Module):
    """Dense projection plus LIF returning bit-packed spikes, forward only (src/myelin/modules.py:906-943)."""

    def __init__(
        self,
        in_features: int,
        out_features: int,
        params: LIFParams | None = None,
        surrogate: SurrogateFn = atan_surrogate,
        surrogate_slope: float = 10.0,
        hard_forward: bool = True,
        bias: bool = True,
        backend: Backend = "torch",
        checkpoint_size: CheckpointSize = 25,
    ) -> None:
        super().__init__()
        self.synapse = LinearSynapse(in_features, out_features, bias=bias)
        self.cell = SurrogateLIFCell(params, surrogate, surrogate_slope, hard_forward)
        self.backend: Backend = backend
        self.checkpoint_size: CheckpointSize = checkpoint_size

    def forward(self, inputs: torch.Tensor) -> PackedSpikes:
        _state, packed = linear_surrogate_lif_packed_forward(
            inputs,
            self.synapse.weight,
            self.synapse.bias,
            self.cell.params,
            surrogate=surrogate_name(self.cell.surrogate),
            surrogate_slope=self.cell.surrogate_slope,
            hard_forward=self.cell.hard_forward,
            backend=self.backend,
            checkpoint_size=self.checkpoint_size,
        )
        return packed


def quantize_synapses(module: nn.Module) -> nn.Module:
    """Replace the synapses of every ``LinearLIF``, ``LinearSurrogateLIF`` and
    ``DecayAttention`` in ``module`` (itself included) by 8-bit ones, in place, for
    inference; returns ``module``. Rate readouts and packed layers keep theirs:
    their projection is part of a fused function that takes float weights."""

    for m in module.modules():
        if isinstance(m, LinearLIF | LinearSurrogateLIF | DecayAttention):
            for name, child in m.named_children():
                if isinstance(child, LinearSynapse):
                    setattr(m, name, QuantizedLinearSynapse.from_synapse(child))
    return module
