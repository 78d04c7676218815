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


@pytest.mark.parametrize("M", [3, 20, 100, 1300])
def test_a_descriptor_that_was_not_initialised(dev, M):
    """map_ready = 0: every product encodes the TMA descriptor itself."""
    import ctypes

    from tensorpack_b200 import _lib
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    K, N = 300, 4000
    m, x = weights(K, N, 1, dev), normal((M, K), 2, dev)
    lib, d = _lib.load(), m.desc
    bare = _lib.FP8Desc(codes=d.codes, scales=d.scales, ldk=d.ldk, E=1, K=K, N=N)
    need = lib.mtc_fp8_gemm_workspace_bytes(ctypes.byref(bare), M)
    ws, y = torch.empty(need + 1, dtype=torch.uint8, device=dev), torch.full((M, N), 7.0, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    rc = lib.mtc_fp8_gemm(ctypes.byref(bare), x.data_ptr(), _lib.F32, M, K, y.data_ptr(), _lib.F32, N, ws.data_ptr(), need,
                          status.data_ptr(), None, torch.cuda.current_stream(dev).cuda_stream)
    assert rc == 0, lib.mtc_last_error()
    assert torch.equal(y, fp8_gemm(x, m)) and int(status) == 0 and bare.map_ready == 0


def test_calls_of_several_host_threads(dev):
    """Threads that call on streams of their own with the same matrices, and
    whose refused calls keep their own error texts."""
    import threading

    from tensorpack_b200.kernels.experts import experts_forward, route_experts
    from tensorpack_b200.kernels.fp8 import FP8Experts, fp8_gemm, fp8_quantize

    m = weights(512, 4000, 1, dev)
    mats = [FP8Experts.from_tensor(normal(shape, 2, dev, scale=0.05)) for shape in ((8, 512, 200), (8, 512, 200), (8, 200, 512))]
    xs = [normal((M, 512), M, dev, torch.bfloat16) for M in (1, 7, 40, 129, 600, 1300)]

    def calls(x):
        ids, w = route_experts(x[:, :8].float(), 2, n_groups=2, top_groups=1)
        codes, scales = fp8_quantize(x)
        return [fp8_gemm(x, m, activation="silu"), experts_forward(x, ids, w, *mats), ids, w, codes.view(torch.uint8), scales]

    want = [calls(x) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            s = torch.cuda.Stream(dev)
            with torch.cuda.stream(s):
                for _ in range(15):
                    got = calls(xs[i])
                    with pytest.raises(ValueError, match=f"{i + 3} experts in 2 groups|top_k={i + 20}"):
                        route_experts(xs[0][:, :i + 3], i + 20, n_groups=2)
                    s.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
        except BaseException as e:  # noqa: BLE001  (told by the main thread)
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    m.check_status()
