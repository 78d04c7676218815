"""8-bit and expert operators without a GPU: argument checks of the C entry
points (they come before any CUDA call), the Python refusals that need no
device, and the plain restatement the GPU tests compare with."""

import ctypes
import math

import numpy as np
import pytest
import torch

import fp8_ref as R
from tensorpack_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def matrix(E=1, K=256, N=128, ldk=256, codes=4096, scales=4096):
    return _lib.FP8Desc(codes=codes, scales=scales, ldk=ldk, E=E, K=K, N=N)


P = 4096  # a non-null, aligned address that is never read: the checks come first


def gemm(lib, w, x_type=0, M=1, ldx=256, y_type=0, ldy=128, X=P, Y=P, ep=None):
    return lib.mtc_fp8_gemm(ctypes.byref(w), X, x_type, M, ldx, Y, y_type, ldy, None, 0, None, ep, None)


@pytest.mark.parametrize("kw,text", [
    (dict(codes=None), b"null"), (dict(scales=None), b"null"), (dict(K=0), b"shape"), (dict(N=-1), b"shape"),
    (dict(E=0), b"shape"), (dict(ldk=250), b"stride"), (dict(ldk=240), b"stride"), (dict(codes=4104), b"aligned"),
    (dict(E=1 << 20, N=1 << 20), b"2^31"), (dict(K=2 ** 31 - 1, ldk=2 ** 31), b"2^31"),
])
def test_bad_matrices_are_refused(lib, kw, text):
    assert gemm(lib, matrix(**kw)) == _lib.MTC_ERR_INVALID
    assert text in lib.mtc_last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(X=None), b"null"), (dict(Y=None), b"null"), (dict(x_type=3), b"type"), (dict(y_type=-1), b"type"),
    (dict(M=0), b"shape"), (dict(M=2 ** 31 - 1), b"shape"), (dict(ldx=255), b"shape"), (dict(ldy=127), b"shape"),
])
def test_bad_products_are_refused(lib, kw, text):
    assert gemm(lib, matrix(), **kw) == _lib.MTC_ERR_INVALID
    assert text in lib.mtc_last_error()


def test_dense_product_takes_one_matrix_and_a_known_activation(lib):
    assert gemm(lib, matrix(E=2)) == _lib.MTC_ERR_INVALID
    assert gemm(lib, matrix(), ep=ctypes.byref(_lib.Epilogue(bias=None, act=9))) == _lib.MTC_ERR_INVALID
    assert b"activation" in lib.mtc_last_error()
    assert lib.mtc_fp8_gemm(None, P, 0, 1, 256, P, 0, 128, None, 0, None, None, None) == _lib.MTC_ERR_INVALID


def test_bad_quantize_arguments_are_refused(lib):
    ok = dict(X=P, t=0, M=2, K=100, ldx=100, q=P, ldq=112, s=P, lds=2)
    for bad in (dict(X=None), dict(t=5), dict(K=0), dict(ldx=99), dict(q=None), dict(ldq=100), dict(ldq=96),
                dict(q=P + 8), dict(s=None), dict(lds=1), dict(M=-1), dict(M=2 ** 31 - 1, lds=2 ** 31),
                dict(K=2 ** 31 - 1, ldx=2 ** 31, ldq=2 ** 31)):
        a = {**ok, **bad}
        assert lib.mtc_fp8_quantize(a["X"], a["t"], a["M"], a["K"], a["ldx"], a["q"], a["ldq"], a["s"], a["lds"],
                                    None) == _lib.MTC_ERR_INVALID, bad
    assert lib.mtc_fp8_pack(P, 0, 4, 4, P, 16, P, None) == _lib.MTC_ERR_INVALID
    assert lib.mtc_fp8_unpack(ctypes.byref(matrix()), 1, P, 128, None) == _lib.MTC_ERR_INVALID


@pytest.mark.parametrize("kw", [
    dict(logits=None), dict(t=4), dict(E=0), dict(E=1025), dict(ld=7), dict(k=0), dict(k=9), dict(score=2),
    dict(groups=3), dict(groups=4, top=0), dict(groups=4, top=5), dict(groups=4, top=1, k=3), dict(E=64, ld=64, k=33),
    dict(E=66, ld=66, groups=33, top=1, k=1), dict(ids=None), dict(T=-1), dict(T=2 ** 31 - 1),
])
def test_bad_routing_is_refused(lib, kw):
    a = {**dict(logits=P, t=0, T=2, E=8, ld=8, k=2, score=0, groups=1, top=1, ids=P), **kw}
    assert lib.mtc_route_experts(a["logits"], a["t"], a["T"], a["E"], a["ld"], a["k"], a["score"], None, a["groups"],
                                 a["top"], 1, 1.0, a["ids"], P, None) == _lib.MTC_ERR_INVALID


def test_bad_expert_products_are_refused(lib):
    gate, down = matrix(E=4, K=256, N=128), matrix(E=4, K=128, N=256, ldk=128)

    def call(g=gate, u=gate, d=down, X=P, xt=0, T=2, ldx=256, ids=P, k=2, act=2, yt=0, ldy=256):
        return lib.mtc_experts_forward(ctypes.byref(g), ctypes.byref(u), ctypes.byref(d), X, xt, T, ldx, ids, P, k,
                                       act, P, yt, ldy, None, 0, None, None)

    assert call() == _lib.MTC_ERR_WORKSPACE
    for kw in (dict(u=matrix(E=4, K=256, N=127)), dict(d=matrix(E=4, K=128, N=255, ldk=128)),
               dict(d=matrix(E=3, K=128, N=256, ldk=128)), dict(X=None), dict(xt=3), dict(yt=9), dict(T=0),
               dict(ldx=255), dict(ldy=255), dict(ids=None), dict(k=0), dict(k=33), dict(act=4),
               dict(g=matrix(E=1025), u=matrix(E=1025), d=matrix(E=1025, K=128, N=256, ldk=128)),
               dict(T=1 << 30, k=32)):
        assert call(**kw) == _lib.MTC_ERR_INVALID, kw
    assert lib.mtc_experts_workspace_bytes(ctypes.byref(gate), 1 << 30, 32, 0) == 0
    wide = matrix(E=1, K=1 << 20, N=128, ldk=1 << 20)  # 512 parts of 2048 columns per token
    assert lib.mtc_experts_workspace_bytes(ctypes.byref(wide), 1 << 22, 1, 0) == 0
    assert lib.mtc_experts_workspace_bytes(None, 1, 1, 0) == 0


def test_host_tensors_are_refused():
    from tensorpack_b200.kernels import experts, fp8

    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        fp8.fp8_quantize(x)
    with pytest.raises(ValueError, match="CUDA"):
        experts.route_experts(x, 2)
    with pytest.raises(TypeError):
        fp8.fp8_gemm(x, "W")
    with pytest.raises(TypeError):
        fp8.fp8_quantize(np.zeros((2, 8), np.float32))
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="CUDA"):
            fp8.FP8Matrix.from_tensor(np.zeros((8, 8), np.float32))


def test_restatement_quantizes_to_the_nearest_code():
    """Every value is within half a step of e4m3: 2^-4 of itself, or half the
    smallest subnormal (2^-10 scales)."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(7, 300, generator=g) * torch.logspace(-6, 3, 300)
    codes, scales = R.quantize(x)
    v = R.spread(codes, scales)
    s = scales.repeat_interleave(128, 1)[:, :300]
    assert ((v - x.double()).abs() <= torch.maximum(x.double().abs() * 2 ** -4, s * 2 ** -10) * (1 + 1e-5)).all()
    assert codes.abs().max() == 448


def test_restatement_routes_ties_and_masks():
    inf = math.inf
    z = torch.tensor([[1.0, 3.0, 3.0, 2.0], [-inf, -inf, 0.0, -inf], [-inf] * 4, [math.nan, 5.0, inf, 5.0]])
    ids, w = R.route(z, 3)
    assert ids.tolist() == [[1, 2, 3], [2, 0, 1], [0, 1, 2], [2, 1, 3]]
    assert w[1].tolist() == [1.0, 0.0, 0.0] and w[2].tolist() == [0.0, 0.0, 0.0]
    # a bias cannot bring a masked expert in front of a free one
    assert R.route(z[1:2], 2, bias=torch.tensor([9.0, 0.0, 0.0, 0.0]))[0].tolist() == [[2, 0]]
