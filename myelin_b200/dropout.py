"""Dropout from a counter-based generator: no mask is stored, none is needed.

An element's draw is a function of the seed, an offset and the element's place,
so the backward pass draws it again instead of keeping it, a run can be
repeated from its seed, and the mask does not depend on the launch. With
``time_shared`` the ``[T, ...]`` input's time steps all use one mask: a synapse
that is dropped stays dropped for the whole window, as spiking networks want it
(a fresh mask each step averages out over the membrane's time constant).
``RateReadoutClassifier``'s ``nn.Dropout`` (src/myelin/modules.py:848-903) draws
per element and stores its mask.
"""

from __future__ import annotations

import torch

from myelin_b200 import _native as nat
from myelin_b200 import compile_ops as cops
from myelin_b200.autograd import DropoutFunction, refuse_tangents, wants_grad

DRAW_RANGE = 65536  # 16 random bits per element


def spike_dropout(
    inputs: torch.Tensor,
    p: float,
    seed: torch.Tensor,
    *,
    time_shared: bool = False,
    training: bool = True,
) -> torch.Tensor:
    """Zero each element with probability ``p`` and scale the others by ``1 / (1 - p)``.

    ``seed`` is an int64 CUDA tensor (seed, offset): every pair gives another
    mask. It is read on the device when the kernel runs (a captured graph sees
    the values of each replay), and a backward pass reads it again: give each
    call its own copy if the values change before then. ``p`` in [0, 1] is
    rounded to a multiple of 2^-16, and the scale is that of the rounded value.
    A dropped element is zero whatever it held. Element ``e`` (in contiguous
    order; within one step when ``time_shared``) draws from Philox 4x32-10 at
    counter ``(e // 8, offset)``, so the mask is the same for every dtype.
    Without ``training``, or where ``p`` rounds to 0, the inputs come back as
    they are.
    """

    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be in [0, 1]; got {p}")
    if time_shared and inputs.ndim < 1:
        raise ValueError("time_shared dropout needs inputs shaped [T, ...]")
    threshold = round(p * DRAW_RANGE)
    if not training or threshold == 0:
        return inputs
    nat.require_cuda(inputs)
    if inputs.dtype not in nat.SCAN_DTYPES:
        raise ValueError(f"inputs must be float32, bfloat16 or float16; got {inputs.dtype}")
    if seed.shape != (2,) or seed.dtype != torch.int64:
        raise ValueError(
            f"seed must be int64 shaped [2]; got {seed.dtype} shaped {tuple(seed.shape)}")
    if seed.device != inputs.device:
        raise ValueError("seed must be on the same device as inputs")
    seed = seed.contiguous()
    refuse_tangents("dropout", inputs)
    if wants_grad(inputs):
        return DropoutFunction.apply(inputs, seed, threshold, bool(time_shared))
    return cops.dropout(inputs, seed, threshold, time_shared)
