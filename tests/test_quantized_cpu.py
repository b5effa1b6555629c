"""Argument checks of the 8-bit projection, without a GPU."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import myelin_b200 as mb
from myelin_b200 import _native as nat

MODE = FakeTensorMode(allow_non_fake_inputs=True)


def _cuda(shape, dtype=torch.float32, **kw):
    with MODE:
        return torch.empty(shape, dtype=dtype, device="cuda", **kw)


def _weight(N=6, K=8):
    return mb.QuantizedWeight(_cuda((N, K), torch.int8), _cuda((N,)))


def test_cpu_tensors_are_refused():
    w = mb.QuantizedWeight(torch.zeros((6, 8), dtype=torch.int8), torch.zeros(6))
    with pytest.raises(ValueError, match="CUDA devices only"):
        mb.quantized_linear(torch.zeros((2, 8)), w)
    with pytest.raises(ValueError, match="CUDA devices only"):
        mb.quantize_rows(torch.zeros((2, 8)))
    with pytest.raises(ValueError, match="CUDA devices only"):
        mb.quantize_weight(torch.zeros((2, 8)))


@pytest.mark.parametrize("call, message", [
    (lambda: mb.quantized_linear(_cuda((2, 9)), _weight()), "must match the weight's 8"),
    (lambda: mb.quantized_linear(_cuda((2, 8), torch.int32), _weight()), "must be float32"),
    (lambda: mb.quantized_linear(_cuda((2, 8)), _weight(), _cuda((5,))), r"shaped \[N\]"),
    (lambda: mb.quantized_linear(_cuda((2, 8)), _weight(), out_dtype=torch.int8), "out_dtype"),
    (lambda: mb.quantized_linear(
        _cuda((2, 8)), mb.QuantizedWeight(_cuda((6, 8)), _cuda((6,)))), "weight.data must be int8"),
    (lambda: mb.quantized_linear(
        _cuda((2, 8)), mb.QuantizedWeight(_cuda((6, 8), torch.int8), _cuda((5,)))),
     "weight.scale must be float32"),
    (lambda: mb.quantized_linear(
        mb.QuantizedRows(_cuda((2, 8), torch.int8), _cuda((3,))), _weight()), "one per row"),
    (lambda: mb.quantized_linear(mb.QuantizedRows(_cuda((2, 8)), _cuda((2,))), _weight()),
     "must be int8"),
    (lambda: mb.quantized_linear(_cuda((2, 2**17)), _weight(2, 2**17)), "input features must be"),
    (lambda: mb.quantize_rows(_cuda((2, 0))), "K >= 1"),
    (lambda: mb.quantize_rows(_cuda((2, 4), torch.float64)), "must be float32"),
    (lambda: mb.quantize_weight(_cuda((4,))), r"shaped \[K, N\]"),
])
def test_refusals(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def test_gradients_are_refused():
    x = _cuda((2, 8), requires_grad=True)
    with pytest.raises(NotImplementedError, match="forward only"):
        mb.quantized_linear(x, _weight())
    with torch.no_grad():
        assert mb.quantized_linear.__name__  # the same call is allowed there (traced below)


def test_traces_to_ops():
    def f(x, data, scale):
        rows = mb.quantize_rows(x)
        w = mb.QuantizedWeight(data, scale)
        return mb.quantized_linear(x, w), mb.quantized_linear(rows, w, out_dtype=torch.float16)

    args = (_cuda((3, 2, 8), torch.bfloat16), _cuda((6, 8), torch.int8), _cuda((6,)))
    gm = make_fx(f, tracing_mode="fake")(*args)
    ops = {str(n.target).split(".")[1] for n in gm.graph.nodes
           if n.op == "call_function" and str(n.target).startswith("myelin_b200.")}
    assert ops == {"quantize_rows", "quantized_project"}
    with MODE:
        a, b = gm(*args)
    assert a.shape == b.shape == (3, 2, 6)
    assert a.dtype == torch.bfloat16 and b.dtype == torch.float16


def test_c_entries():
    lib = nat.lib()
    assert lib.mb_quantize_rows(0, None, 0, 8, 8, None, 8, None, None) == 0
    assert lib.mb_gemm_i8(None, 16, None, None, 16, None, None, 0, 0, None, 4, 0, 4, 8, None) == 0
    for M, K, want in ((1, 32768, 1), (1, 32769, 0), (4, 8192, 1), (5, 16, 0), (0, 8, 0)):
        assert lib.mb_linear_i8_rows_supported(M, K) == want
        assert want == (1 <= M <= nat.I8_ROWS and M * ((K + 15) // 16 * 16) <= nat.I8_ROWS_BYTES)
    bad = [
        (lib.mb_quantize_rows(2, None, 4, 0, 8, None, 8, None, None), "cols >= 1"),
        (lib.mb_quantize_rows(7, None, 4, 8, 8, None, 8, None, None), "unsupported dtype"),
        (lib.mb_quantize_rows(0, None, 4, 8, 8, None, 8, None, None), "null tensor"),
    ]
    assert all(status != 0 for status, _ in bad)
    p = 4096  # an aligned address that is never read: every call is refused first
    for args, message in [
        ((p, 16, None, p, 16, p, None, 0, 0, p, 4, 2, 4, 0, None), "K must be in"),
        ((p, 16, None, p, 16, p, None, 0, 0, p, 4, 2, 4, 1 << 17, None), "K must be in"),
        ((p, 16, None, p, 8, p, None, 0, 0, p, 4, 2, 4, 8, None), "16-byte boundaries"),
        ((p, 16, None, p + 8, 16, p, None, 0, 0, p, 4, 2, 4, 8, None), "16-byte boundaries"),
        ((p, 24, None, p, 16, p, None, 0, 0, p, 4, 2, 4, 8, None), "input rows must start"),
        ((p, 16, None, p, 16, p, None, 0, 6, p, 4, 2, 4, 8, None), "output dtype"),
        ((p, 16, None, p, 16, p, p, 7, 0, p, 4, 2, 4, 8, None), "bias dtype"),
        ((p, 16, None, p, 16, p, None, 0, 0, p, 3, 2, 4, 8, None), "ldc"),
        ((p, 16, None, p, 16, None, None, 0, 0, p, 4, 2, 4, 8, None), "null tensor"),
    ]:
        assert lib.mb_gemm_i8(*args) != 0 and message in lib.mb_last_error().decode()
    assert lib.mb_linear_i8_rows(0, p, 8, None, p, 16, p, None, 0, 0, p, 4, 5, 4, 8, None) != 0
    assert "at most" in lib.mb_last_error().decode()


def test_synapse_keeps_its_row_pitch_across_devices():
    data = torch.zeros((6, 32), dtype=torch.int8)[:, :20]
    synapse = mb.QuantizedLinearSynapse(mb.QuantizedWeight(data, torch.ones(6)))
    synapse.data = data.contiguous()  # as a copy to another device leaves it
    synapse.half()
    assert synapse.data.stride(0) % 16 == 0 and synapse.data.shape == (6, 20)
    assert synapse.scale.dtype == torch.float32
