"""Projection in 8-bit integers against 64-bit arithmetic on the same integers.

Quantised values have to be exact: the definition's fp32 operations (a division,
a product, a rounding to the nearest) are repeated here by torch on the CPU. The
sums are exact, so an output is off by the rounding of the int32 sum to fp32, of
the scales' product, of the scaling with its bias and of the result:
(3 2^-24 |scaled sum|) + (eps / 2 + 2^-24) |out|.
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


def _randn(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV).to(dtype)


def reference_rows(x):
    """(q, scale) by the definition, in fp32 on the CPU."""

    x = x.detach().float().cpu()
    top = x.abs().amax(dim=-1, keepdim=True)
    some = top >= 1e-30
    # tensor by tensor is one division; torch takes 127.0 / tensor as reciprocal * 127.0
    levels = torch.full_like(top, 127.0)
    inv = torch.where(some, levels / torch.where(some, top, 1.0), 0.0)
    scale = torch.where(some, top / levels, 0.0)
    return torch.round(x * inv).to(torch.int8), scale[..., 0]


def weights(N, K, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    w = torch.randint(-127, 128, (N, K), generator=g, device=DEV).to(torch.int8)
    return mb.QuantizedWeight(w, torch.rand((N,), generator=g, device=DEV) + 0.01)


def check_product(out, q, scale, weight, bias):
    acc = q.double().cpu() @ weight.data.double().cpu().t()
    sum_ = acc * weight.scale.double().cpu()
    if scale is not None:
        sum_ = sum_ * scale.double().cpu()[:, None]
    want = sum_ if bias is None else sum_ + bias.double().cpu()
    got = out.double().cpu()
    eps = torch.finfo(out.dtype).eps
    tol = 3 * 2.0**-24 * sum_.abs() + (eps / 2 + 2.0**-24) * want.abs()
    if out.dtype == torch.float16:
        tol = tol + 2.0**-25
    assert got.shape == want.shape
    # past the type's range (fp16: 65520 and up rounds to infinity) the result is infinite
    largest = torch.finfo(out.dtype).max
    past = want.abs() > largest * (1 + eps)
    assert torch.equal(got[past], torch.copysign(torch.tensor(float("inf")).double(), want[past]))
    inside = want.abs() < largest
    assert ((got - want).abs() <= tol)[inside].all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 7), (9, 8), (33, 1000), (5, 1024), (70, 1032),
                                        (2, 8192), (3, 9000), (4, 20001)])
def test_rows_are_quantised_by_the_definition(rows, cols, dtype):
    x = _randn((rows, cols), 1, dtype) * torch.logspace(-3, 3, rows, device=DEV)[:, None].to(dtype)
    x[rows // 2] = 0
    got = mb.quantize_rows(x)
    q, scale = reference_rows(x)
    assert torch.equal(got.data.cpu(), q) and torch.equal(got.scale.cpu(), scale)
    # every value within half a step, and a little for the two fp32 roundings
    step = got.scale.double().cpu()[:, None]
    back = got.data.double().cpu() * step
    assert ((back - x.double().cpu()).abs() <= step * (0.5 + 127 * 3 * 2.0**-24)).all()


def test_rows_that_are_not_finite_or_tiny():
    x = _randn((6, 300), 1)
    x[1, 5], x[2, 7], x[3, 299] = float("inf"), float("nan"), -float("inf")
    x[4] *= 1e-34
    got = mb.quantize_rows(x)
    assert torch.isnan(got.scale[1:4]).all() and torch.isfinite(got.scale[[0, 5]]).all()
    assert got.scale[4] == 0 and torch.count_nonzero(got.data[1:5]) == 0
    w = weights(40, 300, 2)
    for rows in (x, x[:4], x.repeat(30, 1)):  # both kernels
        out = mb.quantized_linear(rows, w)
        assert torch.isnan(out[1:4]).all() and torch.isfinite(out[0]).all()
        assert torch.equal(out[0], mb.quantized_linear(x[:1], w)[0])


SIZES = [(1, 1, 1), (1, 33, 16), (2, 5, 100), (3, 70, 1000), (4, 257, 4096), (4, 9, 8192),
         (5, 64, 128), (9, 40, 3), (200, 1, 64), (17, 1001, 784), (128, 32, 64), (129, 130, 129), (200, 200, 4112),
         (300, 1000, 333), (2000, 2304, 640), (2600, 2561, 200)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M, N, K", SIZES)
def test_float_inputs(M, N, K, dtype):
    x = _randn((M, K), 1, dtype)
    w = weights(N, K, 2)
    bias = _randn((N,), 3, dtype) if N % 2 else None
    out = mb.quantized_linear(x, w, bias)
    q, scale = reference_rows(x)
    assert out.dtype == dtype
    check_product(out, q, scale, w, bias)


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("M, N, K", [(1, 40, 70), (4, 100, 784), (6, 31, 17), (150, 1001, 784),
                                     (260, 300, 1024)])
@pytest.mark.parametrize("kind", ["spikes", "int8", "rows"])
def test_integer_inputs(M, N, K, out_dtype, kind):
    g = torch.Generator(DEV).manual_seed(5)
    w = weights(N, K, 2)
    bias = _randn((N,), 3, torch.bfloat16)
    scale = None
    if kind == "spikes":
        x = given = torch.rand((M, K), generator=g, device=DEV) < 0.3
    else:
        x = given = torch.randint(-128, 128, (M, K), generator=g, device=DEV).to(torch.int8)
        if kind == "rows":
            scale = torch.rand((M,), generator=g, device=DEV)
            given = mb.QuantizedRows(x, scale)
    out = mb.quantized_linear(given, w, bias, out_dtype=out_dtype)
    assert out.dtype == out_dtype
    check_product(out, x.to(torch.int8), scale, w, bias)


def test_largest_sums_stay_exact():
    K = 2**17 - 1
    w = mb.QuantizedWeight(torch.full((40, K), -128, dtype=torch.int8, device=DEV),
                           torch.ones(40, device=DEV))
    x = torch.full((130, K), -128, dtype=torch.int8, device=DEV)
    x[:, 0] = 1
    out = mb.quantized_linear(x, w)
    want = torch.tensor((K - 1) * 128 * 128 - 128, dtype=torch.int64).float()
    assert torch.equal(out.cpu(), want.expand(130, 40))


def test_layouts():
    """Leading dimensions, pitched rows, odd bases and transposed views."""

    T, B, K, N = 6, 25, 100, 72
    w = weights(N, K, 2)
    x = _randn((T, B, K), 1, torch.bfloat16)
    base = mb.quantized_linear(x, w)
    assert base.shape == (T, B, N)
    wide = torch.zeros((T, B, K + 5), dtype=torch.bfloat16, device=DEV)
    wide[..., 3:K + 3] = x
    assert torch.equal(mb.quantized_linear(wide[..., 3:K + 3], w), base)
    turned = x.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(mb.quantized_linear(turned, w), base)
    padded = torch.full((N, 112), 77, dtype=torch.int8, device=DEV)
    padded[:, :K] = w.data
    odd = torch.full((N * 101 + 1,), 55, dtype=torch.int8, device=DEV)[1:].view(N, 101)
    odd[:, :K] = w.data
    for data in (padded[:, :K], odd[:, :K], w.data.t().contiguous().t()):
        again = mb.QuantizedWeight(data, w.scale)
        assert torch.equal(mb.quantized_linear(x, again), base)
        # the kernel for few rows reads nothing past K either
        assert torch.equal(mb.quantized_linear(x[0, :2], again), base[0, :2])
    assert mb.quantized_linear(x[:0], w).shape == (0, B, N)


def test_rows_do_not_depend_on_their_batch():
    w, x = weights(300, 512, 2), _randn((700, 512), 1, torch.bfloat16)
    whole = mb.quantized_linear(x, w)
    for m in (1, 3, 4, 5, 130):
        assert torch.equal(mb.quantized_linear(x[:m], w), whole[:m])


def test_weight_quantisation_and_error_of_a_layer():
    weight = _randn((640, 96), 1) * 0.02
    qw = mb.quantize_weight(weight)
    q, scale = reference_rows(weight.t().contiguous())
    assert torch.equal(qw.data.cpu(), q) and torch.equal(qw.scale.cpu(), scale)
    x = _randn((50, 640), 2)
    out = mb.quantized_linear(x, qw)
    want = x.double() @ weight.double()
    # half a step of either operand against each term of the sums
    sx, sw = mb.quantize_rows(x).scale.double()[:, None], qw.scale.double()[None]
    bound = 0.5 * (sx * weight.double().abs().sum(0) + sw * x.double().abs().sum(1, keepdim=True)
                   ) + 0.25 * 640 * sx * sw
    assert ((out.double() - want).abs() <= 1.001 * bound).all()


def test_network_with_quantised_synapses():
    torch.manual_seed(0)
    net = mb.LinearSurrogateLIF(200, 64, stream_synapse=True).to(DEV)
    with torch.no_grad():
        net.synapse.weight.mul_(40)
        net.synapse.bias.normal_()
    x = torch.randn((20, 8, 200), device=DEV)
    with torch.no_grad():
        currents = mb.QuantizedLinearSynapse.from_synapse(net.synapse)(x)
        _, want = net.unroll(currents)
        mb.quantize_synapses(net)
        assert isinstance(net.synapse, mb.QuantizedLinearSynapse)
        assert torch.equal(net(x), want)
        spikes = torch.rand((20, 8, 200), device=DEV) < 0.2
        assert torch.equal(net.synapse(spikes),
                           mb.quantized_linear(spikes, mb.QuantizedWeight(net.synapse.data,
                                                                          net.synapse.scale),
                                               net.synapse.bias))
        net.to(torch.bfloat16)
        assert net.synapse.scale.dtype == torch.float32
        assert net.synapse(x.to(torch.bfloat16)).dtype == torch.bfloat16
        state = net.state_dict()
        assert state["synapse.data"].dtype == torch.int8


def test_graph_replay_and_opcheck():
    w, x = weights(70, 96, 2), _randn((40, 96), 1, torch.bfloat16)
    one = x[:1].clone()
    mb.quantized_linear(x, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = mb.quantized_linear(x, w), mb.quantized_linear(one, w)
    x.copy_(_randn((40, 96), 9, torch.bfloat16))
    one.copy_(x[:1])
    graph.replay()
    assert torch.equal(a, mb.quantized_linear(x, w)) and torch.equal(b, a[:1])
    torch.library.opcheck(cops.quantize_rows_op, (x,))
    torch.library.opcheck(cops.quantized_project_op,
                          (x, None, w.data, w.scale, None, torch.float32))


def test_wait_timeout_is_reported():
    nat.device_status()
    nat.debug_wait_timeout(nat.MB_UNIT_GEMM_I8)
    torch.cuda.synchronize()
    assert nat.device_status() == 1 and nat.device_status() == 0
