"""Operands with more than 2^31 elements: rows far into them agree with the
same rows in a call of their own."""

import pytest
import torch

from test_gpu_experts import stack
from test_gpu_fp8 import dev, normal, weights  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def many_rows(T, D, dev):
    """T rows of D values, each from a few hundred, so that it is quick to make."""
    base = normal((257, D), 1, dev, torch.bfloat16)
    return base.repeat(-(-T // 257), 1)[:T]


def test_activations_past_2_31_elements(dev):
    from tensorpack_b200.kernels.fp8 import fp8_gemm, fp8_quantize

    M, K, N = 270001, 8200, 200
    x, m = many_rows(M, K, dev), weights(K, N, 2, dev)
    codes, scales = fp8_quantize(x)
    few, fs = fp8_quantize(x[:257])
    for at in (0, 257 * 1000, 257 * 1050):
        rows = min(257, M - at)
        assert torch.equal(codes[at:at + rows].view(torch.uint8), few[:rows].view(torch.uint8))
        assert torch.equal(scales[at:at + rows], fs[:rows])
    del codes, scales
    y = fp8_gemm(x, m)
    assert torch.equal(y[:257], y[257 * 1049:257 * 1050]) and torch.equal(y[:M - 257 * 1050], y[257 * 1050:])
    ref = fp8_gemm(x[:257].float(), m)
    assert (y[:257] - ref).norm() <= 1e-5 * ref.norm()  # (another order of sums)


def test_outputs_past_2_31_elements(dev):
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    M, K, N = 75000, 130, 30000
    x, m = many_rows(M, K, dev), weights(K, N, 2, dev)
    y = fp8_gemm(x, m, out_dtype=torch.bfloat16)
    assert torch.equal(y[257 * 290:257 * 291], y[:257]) and torch.equal(y[257 * 291:], y[:M - 257 * 291])
    m.check_status()


@pytest.mark.parametrize("T,E,k,D,I", [(150001, 8, 8, 2048, 64), (50001, 4, 1, 64, 45000)])
def test_experts_past_2_31_elements(dev, T, E, k, D, I):
    """Experts' outputs (T * k rows of D), then gated values (rows of I), past 2^31."""
    from tensorpack_b200.kernels.experts import experts_forward

    mats = stack(E, D, I, 1, dev), stack(E, D, I, 2, dev), stack(E, I, D, 3, dev)
    x = many_rows(T, D, dev)
    ids = normal((257, E), 5, dev).topk(k, 1).indices.to(torch.int32).repeat(-(-T // 257), 1)[:T]
    w = torch.softmax(normal((257, k), 6, dev), 1).repeat(-(-T // 257), 1)[:T]
    y = experts_forward(x, ids, w, *mats, out_dtype=torch.bfloat16)
    mats[0].check_status()
    last = T // 257
    for n in (1, last // 2, last - 1):
        assert torch.equal(y[257 * n:257 * (n + 1)], y[:257])
    assert torch.equal(y[257 * last:], y[:T - 257 * last])
    ref = experts_forward(x[:257], ids[:257], w[:257], *mats)
    assert (y[:257].float() - ref).norm() <= 6e-3 * ref.norm()  # half a step of bf16, codes next to a border
