"""8-bit matrices on the GPU against the plain restatement (fp8_ref).

Codes and scales are compared bit for bit.  A product's fp32 value is off by
at most c * sum|products|: 128 additions of a block on the tensor cores (taken
as truncating, 2^-23 each), K/128 fused multiply-adds, the product of the two
scales, the bias; the activations add a Lipschitz factor of at most 1.13 and a
few ulp of their own (2^-21 of the magnitude covers expf and tanhf).  An
output type with fewer bits adds half a step.
"""

import numpy as np
import pytest
import torch

import fp8_ref as R

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    from tensorpack_b200 import build

    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    build.build()
    return torch.device("cuda", 0)


def normal(shape, seed, dev, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (scale * torch.randn(shape, device=dev, generator=g)).to(dtype)


def weights(K, N, seed, dev):
    from tensorpack_b200.kernels.fp8 import FP8Matrix

    return FP8Matrix.from_tensor(normal((K, N), seed, dev, scale=0.05))


def close(y, ref, mag, K, dtype):
    blocks = -(-K // 128)
    c = (128 * 2.0 + blocks + 4) * 2 ** -24
    tol = (1.13 * c + 2 ** -21) * mag + 2.0 ** -30
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (ref.abs() + tol) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    bad = (y.double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {((y.double() - ref).abs() / tol).max()}"


# ------------------------------------------------------------------------------------------ formats
@pytest.mark.parametrize("K,N", [(1, 1), (17, 300), (128, 128), (130, 257), (896, 128)])
def test_pack_and_unpack_match_the_format(dev, K, N):
    from tensorpack_b200.kernels.fp8 import FP8Matrix

    W = normal((K, N), K + N, dev)
    m = FP8Matrix.from_tensor(W)
    codes, scales = R.pack(W)
    assert m.shape == (K, N) and torch.equal(m.codes.double(), codes) and torch.equal(m.scales[0].double(), scales)
    full = m.to_tensor()
    assert torch.equal(full, R.spread(codes, scales, 128).T.float())
    assert np.array_equal(m.to_array(), full.cpu().numpy())
    again = FP8Matrix.from_codes(m.codes, m.scales[0])
    assert torch.equal(again.to_tensor(), full)
    assert m.weight_bytes == K * N + 4 * scales.numel()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K", [(1, 1), (3, 100), (5, 129), (16, 4096), (257, 130), (1000, 264)])
def test_quantize_is_bit_exact(dev, M, K, dtype):
    from tensorpack_b200.kernels.fp8 import fp8_quantize

    x = normal((M, K), M * K, dev, TYPES[dtype]) * torch.logspace(-3, 2, K, device=dev).to(TYPES[dtype])
    codes, scales = fp8_quantize(x)
    rc, rs = R.quantize(x)
    assert codes.shape == (M, K) and scales.shape == rs.shape
    assert torch.equal(codes.double(), rc) and torch.equal(scales.double(), rs)


def test_quantize_views_zeros_and_tiny_values(dev):
    from tensorpack_b200.kernels.fp8 import fp8_quantize

    big = normal((40, 700), 3, dev)
    for x in (big[::3, :300], big[:, 5:205], big.T, big[7:8, 1:].expand(4, -1), torch.zeros(3, 200, device=dev),
              torch.full((2, 130), 1e-40, device=dev), torch.full((2, 130), -3e38, device=dev), big[:0], big.double()):
        codes, scales = fp8_quantize(x)
        rc, rs = R.quantize(x)
        assert torch.equal(codes.double(), rc) and torch.equal(scales.double(), rs)


def test_groups_that_are_not_finite(dev):
    from tensorpack_b200.kernels.fp8 import fp8_gemm, fp8_quantize

    x = normal((40, 300), 4, dev)
    x[1, 5], x[2, 299], x[39, 130] = float("nan"), float("inf"), -float("inf")
    codes, scales = fp8_quantize(x)
    rc, rs = R.quantize(x)
    assert torch.equal(codes.double(), rc)
    assert torch.equal(torch.isnan(scales), torch.isnan(rs)) and torch.equal(scales.nan_to_num(-1).double(),
                                                                            rs.nan_to_num(-1))
    m = weights(300, 200, 5, dev)
    clean = x.clone()
    clean[[1, 2, 39]] = 0
    for rows in (slice(0, 16), slice(0, 40)):
        y, ref = fp8_gemm(x[rows], m), fp8_gemm(clean[rows], m)
        hit = torch.tensor([i in (1, 2, 39) for i in range(40)], device=dev)[rows]
        assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], ref[~hit])


# ------------------------------------------------------------------------------------------ products
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 32, 33, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("K,N", [(1, 1), (100, 60), (128, 128), (896, 130), (1300, 514)])
def test_gemm_matches_the_restatement(dev, M, K, N):
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    x, m = normal((M, K), M + K, dev), weights(K, N, N, dev)
    y = fp8_gemm(x, m)
    torch.cuda.synchronize()
    m.check_status()
    ref, mag = R.gemm(x, m.codes, m.scales[0])
    assert y.dtype == torch.float32 and y.shape == (M, N)
    close(y, ref, mag, K, torch.float32)
    assert torch.equal(y, fp8_gemm(x, m))  # the same bits every time


@pytest.mark.parametrize("M,K,N", [(1, 4096, 1024), (16, 14336, 512), (4, 4864, 896), (2100, 300, 4864), (1500, 1000, 3333),
                                   (9, 1100, 40000), (40, 300, 40000), (100, 700, 40000)])
def test_gemm_long_and_large(dev, M, K, N):
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    x, m = normal((M, K), M + K, dev, torch.bfloat16), weights(K, N, N, dev)
    y = fp8_gemm(x, m)
    torch.cuda.synchronize()
    m.check_status()
    ref, mag = R.gemm(x, m.codes, m.scales[0])
    close(y, ref, mag, K, torch.float32)


@pytest.mark.parametrize("M,K,N", [(7, 1300, 900), (8, 1300, 900), (9, 1300, 900), (10, 300, 40000), (64, 300, 20000),
                                   (65, 700, 9700), (65, 700, 9400), (128, 300, 9500), (129, 264, 4700), (129, 264, 4900),
                                   (200, 1000, 4900), (257, 129, 6400)])
def test_gemm_on_both_sides_of_its_variants(dev, M, K, N):
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    m, b = weights(K, N, N, dev), normal((N,), 9, dev)
    for t in (torch.float32, torch.float16):
        x = normal((M, K), M + K, dev, t)
        y = fp8_gemm(x, m, b, "silu")
        torch.cuda.synchronize()
        m.check_status()
        ref, mag = R.gemm(x, m.codes, m.scales[0], b, "silu")
        close(y, ref, mag, K, torch.float32)


@pytest.mark.parametrize("M", [1, 12, 40, 70])
@pytest.mark.parametrize("K,N", [(5000, 2000), (5000, 2100), (3600, 2500), (3600, 2800), (3600, 3600), (3600, 4200),
                                 (3600, 4500), (3600, 5800), (1000, 6100)])
def test_gemm_split_over_clusters_of_any_size(dev, M, K, N):
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    x, m, b = normal((M, K), M + K, dev), weights(K, N, N, dev), normal((N,), 9, dev)
    y = fp8_gemm(x, m, b, "relu")
    torch.cuda.synchronize()
    m.check_status()
    ref, mag = R.gemm(x, m.codes, m.scales[0], b, "relu")
    close(y, ref, mag, K, torch.float32)
    assert torch.equal(y, fp8_gemm(x, m, b, "relu"))


@pytest.mark.parametrize("xt", list(TYPES))
@pytest.mark.parametrize("yt", list(TYPES))
@pytest.mark.parametrize("M,N", [(3, 200), (50, 200), (1300, 4000)])
def test_types_bias_and_activations(dev, xt, yt, M, N):
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    K = 264
    x, m, b = normal((M, K), 7, dev, TYPES[xt]), weights(K, N, 8, dev), normal((N,), 9, dev)
    for bias, act in ((b, None), (None, "relu"), (b, "silu"), (b, "gelu_tanh")):
        y = fp8_gemm(x, m, bias, act, out_dtype=TYPES[yt])
        ref, mag = R.gemm(x, m.codes, m.scales[0], bias, act)
        assert y.dtype == TYPES[yt]
        close(y, ref, mag, K, TYPES[yt])


@pytest.mark.parametrize("yt", list(TYPES))
@pytest.mark.parametrize("N", [4872, 4881, 4865, 4991])
def test_aligned_rows_with_a_ragged_end(dev, yt, N):
    """Rows that start on 32 bytes and end inside a vector: what lies behind
    them in the larger tensor stays."""
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    M, K, t = 300, 260, TYPES[yt]
    x, m, b = normal((M, K), 3, dev), weights(K, N, 4, dev), normal((N,), 5, dev)
    hold = torch.full((M + 1, 5008), 7.0, device=dev, dtype=t)
    for bias, act in ((None, None), (b, "gelu_tanh")):
        y = fp8_gemm(x, m, bias, act, Y=hold[:M, :N])
        ref, mag = R.gemm(x, m.codes, m.scales[0], bias, act)
        close(y, ref, mag, K, t)
        assert (hold[M] == 7).all() and (hold[:, N:] == 7).all()


@pytest.mark.parametrize("M", [2, 40, 1300])
def test_operands_that_are_views(dev, M):
    """Rows with a stride, rows that start off 16 bytes, an output inside a
    larger tensor whose other values stay."""
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    K, N = 301, 4001
    wide = normal((M, 700), 11, dev, torch.float16)
    m = weights(K, N, 12, dev)
    for x in (wide[:, :K], wide[:, 3:3 + K], wide.T[:K].T):
        ref, mag = R.gemm(x, m.codes, m.scales[0])
        hold = torch.full((M + 2, N + 6), 7.0, device=dev)
        y = hold[1:M + 1, 3:N + 3]
        assert fp8_gemm(x, m, Y=y) is y
        close(y, ref, mag, K, torch.float32)
        edge = torch.ones_like(hold, dtype=torch.bool)
        edge[1:M + 1, 3:N + 3] = False
        assert (hold[edge] == 7).all()
        # the copy of a view gives the same bits
        assert torch.equal(y, fp8_gemm(x.contiguous(), m))


def test_numpy_and_empty_batches(dev):
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    m = weights(200, 150, 1, dev)
    x = normal((9, 200), 2, dev)
    y = fp8_gemm(x.cpu().numpy(), m)
    assert isinstance(y, np.ndarray) and np.array_equal(y, fp8_gemm(x, m).cpu().numpy())
    assert fp8_gemm(x[:0], m).shape == (0, 150)


def test_a_nan_code_stays_in_its_column(dev):
    from tensorpack_b200.kernels.fp8 import FP8Matrix, fp8_gemm

    m = weights(200, 300, 1, dev)
    codes = m.codes.view(torch.uint8).clone()
    codes[17, 3] = 0x7F
    bad = FP8Matrix.from_codes(codes, m.scales[0])
    for M in (3, 40):
        x = normal((M, 200), 2, dev)
        y, ref = fp8_gemm(x, bad), fp8_gemm(x, m)
        col = torch.arange(300, device=dev) == 17
        assert torch.isnan(y[:, col]).all() and torch.equal(y[:, ~col], ref[:, ~col])


def test_from_mtc_and_the_layer(dev):
    import inputs
    from oracle import mtc_oracle as O
    from tensorpack_b200.kernels.fp8 import FP8Matrix, fp8_gemm
    from tensorpack_b200.kernels.gemm import MTCMatrix
    from tensorpack_b200.nn import LinearFP8, LinearMTCAdaptive

    W, sizes, leaf, modes, scales = inputs.forced_mode_allocation(128, 256, seed=7, p_split=0.5)
    mat = MTCMatrix.from_qt_allocation(W, O.QuadtreeAllocation(sizes, leaf, modes, scales, None, 0))
    bias = np.arange(256, dtype=np.float32) / 100
    packed = LinearMTCAdaptive.from_mtc(mat, bias, activation="silu")
    layer = LinearFP8.from_mtc(packed, dev)
    m = FP8Matrix.from_tensor(mat.to_tensor(dev))
    assert torch.equal(layer.W_fp8.codes.view(torch.uint8), m.codes.view(torch.uint8))
    x = normal((20, 128), 3, dev)
    y = layer(x)
    assert torch.equal(y, fp8_gemm(x, m, torch.from_numpy(bias).to(dev), "silu"))
    assert np.array_equal(layer(x.cpu().numpy()), y.cpu().numpy())
    assert layer.weight_bytes == m.weight_bytes + bias.nbytes
    half = LinearFP8(m, out_dtype=torch.bfloat16)
    assert half(x).dtype == torch.bfloat16


# ------------------------------------------------------------------------------------------ streams, graphs
@pytest.mark.parametrize("M", [1, 40, 1300])
def test_other_streams_and_captured_graphs(dev, M):
    from tensorpack_b200.kernels.fp8 import fp8_gemm

    ms = [weights(512, 4000, s, dev) for s in (1, 2)]
    xs = [normal((M, 512), s, dev) for s in (3, 4)]
    want = [fp8_gemm(x, m) for x, m in zip(xs, ms)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = fp8_gemm(xs[i], ms[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    held = [x.clone() for x in xs]
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(fp8_gemm(held[i], ms[i]))
        graphs.append(g)
    for a, b in ((0, 1), (1, 0)):
        for i in range(2):
            held[i].copy_(xs[i] if (a, b) == (0, 1) else 2 * xs[i])
        for i, s in zip((a, b), streams):
            s.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(s):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], fp8_gemm(held[i], ms[i]))


def test_refusals(dev):
    from tensorpack_b200.kernels.fp8 import FP8Experts, FP8Matrix, fp8_gemm, fp8_quantize

    m = weights(64, 32, 1, dev)
    x = normal((4, 64), 2, dev)
    with pytest.raises(AssertionError, match="Shape mismatch"):
        fp8_gemm(x[:, :63], m)
    with pytest.raises(ValueError, match="CUDA"):
        fp8_gemm(x.cpu(), m)
    with pytest.raises(ValueError, match="matrix"):
        fp8_gemm(x[0], m)
    with pytest.raises(ValueError, match="bias"):
        fp8_gemm(x, m, torch.zeros(31, device=dev))
    with pytest.raises(ValueError, match="activation"):
        fp8_gemm(x, m, activation="tanh")
    with pytest.raises(ValueError, match="type"):
        fp8_gemm(x, m, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="Y must"):
        fp8_gemm(x, m, Y=torch.empty(4, 31, device=dev))
    with pytest.raises(ValueError, match="contiguous"):
        fp8_gemm(x, m, Y=torch.empty(32, 4, device=dev).T)
    with pytest.raises(ValueError, match="overlaps"):
        fp8_gemm(x, m, Y=x[:, :32])
    with pytest.raises(ValueError):
        fp8_quantize(x[:, :0])
    codes = torch.zeros(32, 64, dtype=torch.float8_e4m3fn, device=dev)
    for c, s in ((codes, torch.zeros(1, 2, device=dev)), (codes, torch.zeros(1, 1, device=dev).double()),
                 (codes.float(), torch.zeros(1, 1, device=dev)), (codes[0], torch.zeros(1, 1, device=dev)),
                 (codes, torch.zeros(1, 1))):
        with pytest.raises(ValueError):
            FP8Matrix.from_codes(c, s)
    with pytest.raises(ValueError):
        FP8Experts.from_codes(codes, torch.zeros(1, 1, device=dev))
    with pytest.raises(ValueError):
        FP8Matrix.from_tensor(torch.zeros(3, device=dev))
