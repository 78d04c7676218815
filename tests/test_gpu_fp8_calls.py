"""Ways to make and call 8-bit matrices that a program may use."""

import pytest
import torch

from test_gpu_fp8 import dev, normal, weights  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def test_a_matrix_from_the_codes_and_scales_of_another(dev):
    from tensorpack_b200.kernels.fp8 import FP8Experts, FP8Matrix

    for K, N in ((300, 200), (128, 130)):
        m = weights(K, N, 1, dev)
        assert m.codes.shape == (N, K) and m.scales.shape == (1, -(-N // 128), -(-K // 128))
        for scales in (m.scales, m.scales[0]):
            again = FP8Matrix.from_codes(m.codes, scales)
            assert again.shape == m.shape and torch.equal(again.to_tensor(), m.to_tensor())
        stack = FP8Experts.from_tensor(normal((2, K, N), 2, dev))
        assert torch.equal(FP8Experts.from_codes(stack.codes, stack.scales).to_tensor(), stack.to_tensor())
        with pytest.raises(ValueError):
            FP8Matrix.from_codes(m.codes, m.scales.expand(2, -1, -1))
        with pytest.raises(ValueError):
            FP8Matrix.from_codes(m.codes, m.scales[0, 0])
