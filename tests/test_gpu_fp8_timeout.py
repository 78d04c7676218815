"""The bounded-wait path of the 8-bit products, made to run out on purpose.

A diagnostic hold (mtc_debug_withhold_bytes) makes the first stage of every
CTA (of a cluster's first CTA where the inputs are split) expect 16 bytes that
no copy delivers: the wait for it gives up at the (shortened) limit, whichever
warp waits.  The call reports MTC_STATUS_TIMEOUT, writes nothing and returns;
the next call is correct.  Every wait is bounded: nothing here hangs.
"""

import contextlib

import pytest
import torch

from test_gpu_experts import stack
from test_gpu_fp8 import TYPES, dev, normal, weights  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def held_first_stage():
    from tensorpack_b200 import _lib

    lib = _lib.load()
    try:
        assert lib.mtc_set_wait_limit_ns(1_000_000) == 0  # 1 ms
        assert lib.mtc_debug_withhold_bytes(16) == 0
        yield
    finally:
        lib.mtc_debug_withhold_bytes(0)
        lib.mtc_set_wait_limit_ns(0)


def timed_out(m):
    with pytest.raises(RuntimeError, match="timed out"):
        m.check_status()
    m.check_status()  # raised once, then clear


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("M,K,N", [
    (3, 256, 300), (3, 4096, 40000),          # activations quantized inside: fewer blocks than stages, many items
    (4, 4864, 256), (1, 14336, 2048),         # inputs split over a cluster
    (16, 300, 200), (60, 1500, 40000),        # codes
    (16, 4864, 512), (40, 4864, 512), (100, 4000, 300),
    (1300, 100, 4000), (1300, 300, 4000), (2100, 2000, 4864),  # the kernel for many rows
])
def test_a_product_whose_wait_runs_out(dev, M, K, N, dtype):
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    x, m = normal((M, K), M, dev, TYPES[dtype]), weights(K, N, N, dev)
    want = fp8_gemm(x, m)
    y = torch.full((M, N), float("nan"), device=dev)
    torch.cuda.synchronize()
    m.check_status()
    with held_first_stage():
        fp8_gemm(x, m, Y=y)
        torch.cuda.synchronize()  # the kernel ended: no wait outlived its limit
    timed_out(m)
    assert torch.isnan(y).all(), "a CTA that gave up, or whose cluster did, must not write its output"
    fp8_gemm(x, m, Y=y)
    torch.cuda.synchronize()
    m.check_status()
    assert torch.equal(y, want)


@pytest.mark.parametrize("T,E,k,D,I", [
    (1, 16, 4, 1200, 130), (6, 16, 4, 300, 260),   # activations quantized inside, without and with a plan
    (20, 4, 2, 2048, 128),                         # split
    (120, 16, 2, 260, 200),                        # a few rows more than those take
    (700, 4, 2, 200, 150), (1000, 8, 2, 1100, 300),  # the kernel for many rows
])
def test_experts_whose_wait_runs_out(dev, T, E, k, D, I):
    from tensorpack_b200.kernels.experts import experts_forward

    mats = stack(E, D, I, 1, dev), stack(E, D, I, 2, dev), stack(E, I, D, 3, dev)
    x = normal((T, D), 4, dev, torch.bfloat16)
    ids = normal((T, E), 5, dev).topk(k, 1).indices.to(torch.int32)
    w = torch.softmax(normal((T, k), 6, dev), 1)
    want = experts_forward(x, ids, w, *mats)
    torch.cuda.synchronize()
    mats[0].check_status()
    with held_first_stage():  # of gate and up; what follows reads what they left
        experts_forward(x, ids, w, *mats)
        torch.cuda.synchronize()
    timed_out(mats[0])
    y = experts_forward(x, ids, w, *mats)
    torch.cuda.synchronize()
    mats[0].check_status()
    assert torch.equal(y, want)
