"""Dense projection in 8-bit integers for inference: a scale for each row and channel.

    out[m, n] = row_scale[m] * channel_scale[n] * sum_k q[m, k] w[n, k] + bias[n]

with signed 8-bit q and w, exact int32 sums, one fp32 scaling and one rounding.
Spikes are 0 or 1 and enter as they are; float inputs are quantised row by row
when they arrive. It stands beside the float projections of
``myelin_b200.projection`` (LinearSynapse, src/myelin/modules.py:112-133) and
runs hand-written CUDA kernels: tcgen05 int8 tensor-core tiles, and a
weight-streaming kernel for up to four rows. The reference has no counterpart.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from myelin_b200 import _native as nat
from myelin_b200 import compile_ops as cops
from myelin_b200.autograd import refuse_tangents, wants_grad

MAX_FEATURES = 2**17 - 1  # sums of products of bytes stay exact in int32


@dataclass(frozen=True)
class QuantizedRows:
    """int8 ``data[..., K]`` standing for ``data * scale[..., None]``."""

    data: torch.Tensor
    scale: torch.Tensor

    def dequantize(self) -> torch.Tensor:
        return self.data.to(torch.float32) * self.scale[..., None]


@dataclass(frozen=True)
class QuantizedWeight:
    """int8 ``data[N, K]`` (one row per output neuron) and fp32 ``scale[N]``.

    Rows that start on 16-byte boundaries (``quantize_weight`` makes them so) are
    read where they lie; others are copied by every product.
    """

    data: torch.Tensor
    scale: torch.Tensor

    def dequantize(self) -> torch.Tensor:
        """The float weight it stands for, ``[K, N]`` like ``LinearSynapse.weight``."""

        return (self.data.to(torch.float32) * self.scale[:, None]).t()


def _check_float(t: torch.Tensor, what: str) -> None:
    if t.dtype not in nat.SCAN_DTYPES:
        raise ValueError(f"{what} must be float32, bfloat16 or float16; got {t.dtype}")


def quantize_rows(inputs: torch.Tensor) -> QuantizedRows:
    """Symmetric 8-bit quantisation of each row of ``[..., K]``:
    ``scale = max|x| / 127``, values rounded to the nearest (ties to even).

    A row of zeros (or of magnitudes below 1e-30) has scale 0; a row that holds an
    infinity or NaN has scale NaN.
    """

    if inputs.ndim < 1 or inputs.shape[-1] < 1:
        raise ValueError(f"inputs must be shaped [..., K] with K >= 1; got {tuple(inputs.shape)}")
    nat.require_cuda(inputs)
    _check_float(inputs, "inputs")
    refuse_tangents("quantize_rows", inputs)
    K = inputs.shape[-1]
    data, scale = cops.quantize_rows(inputs.detach().reshape(-1, K))
    return QuantizedRows(data.reshape(inputs.shape), scale.reshape(inputs.shape[:-1]))


def quantize_weight(weight: torch.Tensor) -> QuantizedWeight:
    """``weight[K, N]`` (the layout of ``LinearSynapse.weight``) with one scale per
    output neuron; done once, when a model is prepared for inference."""

    if weight.ndim != 2 or weight.shape[0] < 1:
        raise ValueError(f"weight must be shaped [K, N] with K >= 1; got {tuple(weight.shape)}")
    nat.require_cuda(weight, "weight")
    _check_float(weight, "weight")
    refuse_tangents("quantize_weight", weight)
    if weight.shape[0] > MAX_FEATURES:
        raise ValueError(f"at most {MAX_FEATURES} input features; got {weight.shape[0]}")
    data, scale = cops.quantize_rows(weight.detach().t().contiguous())
    return QuantizedWeight(data, scale)


def quantized_linear(
    inputs: torch.Tensor | QuantizedRows,
    weight: QuantizedWeight,
    bias: torch.Tensor | None = None,
    *,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``inputs[..., K]`` through an 8-bit weight: ``[..., N]``.

    ``inputs`` may be float (quantised row by row, as ``quantize_rows`` does), bool
    or int8 (integers as they are: spikes), or ``QuantizedRows``. The result is in
    ``out_dtype``, which defaults to a float input's dtype and to float32 for
    integers. Forward only: inputs that require a gradient are refused while
    gradients are enabled.
    """

    scale = None
    x = inputs
    if isinstance(inputs, QuantizedRows):
        x, scale = inputs.data, inputs.scale
        if x.dtype != torch.int8:
            raise ValueError(f"QuantizedRows.data must be int8; got {x.dtype}")
    if x.ndim < 1:
        raise ValueError("inputs must be shaped [..., K]")
    if weight.data.ndim != 2:
        raise ValueError(f"weight.data must be shaped [N, K]; got {tuple(weight.data.shape)}")
    N, K = weight.data.shape
    if x.shape[-1] != K:
        raise ValueError(f"inputs.shape[-1] must match the weight's {K} features; "
                         f"got {tuple(x.shape)}")
    if not 1 <= K <= MAX_FEATURES:
        raise ValueError(f"input features must be in [1, {MAX_FEATURES}]; got {K}")
    nat.require_cuda(x)
    if x.dtype not in (torch.bool, torch.int8):
        _check_float(x, "inputs (unless bool, int8 or QuantizedRows)")
    if weight.data.dtype != torch.int8 or weight.data.device != x.device:
        raise ValueError("weight.data must be int8 on the same device as inputs")
    if weight.scale.shape != (N,) or weight.scale.dtype != torch.float32 \
            or weight.scale.device != x.device:
        raise ValueError("weight.scale must be float32 shaped [N] on the same device as inputs")
    if scale is not None and (scale.shape != x.shape[:-1] or scale.dtype != torch.float32
                              or scale.device != x.device):
        raise ValueError("QuantizedRows.scale must be float32, one per row, on the same device")
    if bias is not None:
        if bias.shape != (N,):
            raise ValueError("bias must be shaped [N]")
        if bias.device != x.device:
            raise ValueError("bias must be on the same device as inputs")
        _check_float(bias, "bias")
    if out_dtype is None:
        out_dtype = x.dtype if x.dtype.is_floating_point else torch.float32
    if out_dtype not in nat.SCAN_DTYPES:
        raise ValueError(f"out_dtype must be float32, bfloat16 or float16; got {out_dtype}")
    refuse_tangents("quantized_linear", x, scale, weight.scale, bias)
    if wants_grad(x, scale, weight.scale, bias):
        raise NotImplementedError("quantized_linear is forward only; detach its inputs or call "
                                  "it under torch.no_grad()")
    out = cops.quantized_project(
        x if x.ndim == 2 else x.reshape(-1, K), None if scale is None else scale.reshape(-1).contiguous(), weight.data,
        weight.scale.contiguous(), None if bias is None else bias.contiguous(), out_dtype)
    return out if x.ndim == 2 else out.view(*x.shape[:-1], N)
