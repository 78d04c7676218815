"""The many-row product where its tile changes with every block of inputs.

With 128 inputs at most a tile is a single block, so the tile that the scaling
warps are told about (first row, end, features) is another one in every slot
of their ring, and a CTA goes through the ring several times.  A row stored by
the wrong tile would miss its place: every row is compared with the same row
of a product of few rows, which knows no tiles, and the rows behind the last
one stay as they were.
"""

import pytest
import torch

import fp8_ref as R
from test_gpu_experts import near, pairs, stack
from test_gpu_fp8 import close, dev, normal, weights  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,K,N", [(5000, 128, 12000), (3333, 100, 20001), (20000, 17, 3000)])
def test_a_tile_per_block(dev, M, K, N):
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    x, m = normal((M, K), M, dev), weights(K, N, N, dev)
    hold = torch.full((M + 3, N), 7.0, device=dev)
    y = fp8_gemm(x, m, Y=hold[:M])
    torch.cuda.synchronize()
    m.check_status()
    assert (hold[M:] == 7).all()
    for at in range(0, M, 997):
        rows = x[at:at + 8]
        # one block of inputs: the same sums and scales in both kernels
        assert torch.equal(y[at:at + 8], fp8_gemm(rows, m))
    ref, mag = R.gemm(x, m.codes, m.scales[0])
    close(y, ref, mag, K, torch.float32)


@pytest.mark.parametrize("T,E,k,D,I", [(3000, 48, 4, 128, 128), (2000, 24, 3, 100, 90), (9000, 60, 2, 128, 260)])
def test_experts_with_a_tile_per_block(dev, T, E, k, D, I):
    from tensorpack_b200.kernels.experts import experts_forward

    mats = stack(E, D, I, 1, dev), stack(E, D, I, 2, dev), stack(E, I, D, 3, dev)
    x = normal((T, D), 4, dev)
    # unequal experts: tiles that end anywhere
    ids = (normal((T, E), 5, dev) + normal((E,), 6, dev)).topk(k, 1).indices.to(torch.int32)
    w = torch.softmax(normal((T, k), 7, dev), 1)
    y = experts_forward(x, ids, w, *mats)
    torch.cuda.synchronize()
    mats[0].check_status()
    ref, _ = R.experts(x, ids, w, *pairs(*mats))
    near(y, ref, torch.float32)
    for _ in range(20):
        assert torch.equal(experts_forward(x, ids, w, *mats), y)
