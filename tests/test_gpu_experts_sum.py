"""The experts' weighted sum keeps its terms in fp32.

A result of 16 bits is the fp32 result rounded once, bit for bit: nothing
before the last rounding depends on the result's type.
"""

import pytest
import torch

from test_gpu_experts import stack
from test_gpu_fp8 import dev, normal  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,D,I", [(1, 64, 8, 256, 130), (7, 8, 5, 300, 60), (48, 64, 8, 512, 200),
                                       (120, 16, 2, 260, 200), (300, 96, 6, 144, 96), (700, 4, 2, 200, 150),
                                       (1000, 8, 8, 384, 300)])
def test_a_16_bit_result_is_rounded_once(dev, T, E, k, D, I, dtype):
    from tensorpack_b200.kernels.experts import experts_forward

    mats = stack(E, D, I, 1, dev), stack(E, D, I, 2, dev), stack(E, I, D, 3, dev)
    x = normal((T, D), 4, dev, torch.bfloat16)
    ids = normal((T, E), 5, dev).topk(k, 1).indices.to(torch.int32)
    w = torch.softmax(normal((T, k), 6, dev), 1)
    full = experts_forward(x, ids, w, *mats)
    assert torch.equal(experts_forward(x, ids, w, *mats, out_dtype=dtype), full.to(dtype))
