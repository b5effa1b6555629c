"""First calls of a thread that has made no CUDA call yet, as the first backward
pass of a process is in the autograd engine's thread: the tensor maps of the
tensor-core kernels are made by the driver, which needs the thread's context."""

from __future__ import annotations

import threading

import pytest
import torch

from myelin_b200 import _native as nat

pytestmark = pytest.mark.gpu
DEV = "cuda"


def in_a_fresh_thread(call):
    failure = []

    def run():
        try:
            call()
        except Exception as error:  # noqa: BLE001  (reported by the caller)
            failure.append(error)

    thread = threading.Thread(target=run)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    if failure:
        raise failure[0]


def _randn(*shape, dtype=torch.bfloat16):
    return torch.randn(shape, device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decayed_attention(dtype):
    q, k, v = (_randn(130, 2, 2, 64, dtype=dtype) for _ in range(3))
    decay = torch.tensor([0.5, 0.9], device=DEV)
    outs = [torch.zeros_like(q) for _ in range(2)]

    def call(out):
        nat.decay_attention(q, k, v, out, decay, None, None, None, reverse=False, out_scale=1.0,
                            kv_scale=1.0)

    torch.cuda.synchronize()
    in_a_fresh_thread(lambda: call(outs[0]))
    call(outs[1])
    assert torch.equal(*outs) and torch.count_nonzero(outs[0])


def test_integer_product():
    a = torch.ones((40, 64), dtype=torch.int8, device=DEV)
    out = torch.zeros((40, 40), device=DEV)
    scale = torch.ones((40,), device=DEV)
    torch.cuda.synchronize()
    in_a_fresh_thread(lambda: nat.gemm_i8(a, None, a, scale, None, out))
    assert torch.equal(out, torch.full_like(out, 64.0))


def test_projection():
    a, out = torch.ones((128, 64), dtype=torch.bfloat16, device=DEV), _randn(128, 128)
    torch.cuda.synchronize()
    in_a_fresh_thread(lambda: nat.gemm_tn(a, a, None, out))
    assert torch.equal(out, torch.full_like(out, 64.0))
