"""Linear layers in 8-bit floating point (e4m3), scaled by blocks of 128.

``FP8Matrix`` is the 8-bit counterpart of ``MTCMatrix``: a K x N weight kept
as e4m3 codes with one fp32 scale per 128 x 128 block.  ``fp8_gemm(X, W)`` is
the counterpart of ``gemm_fused``: it quantizes the activations (one fp32
scale per row and 128 inputs, ``fp8_quantize``), multiplies the codes on the
tensor cores and adds the scaled sums of the blocks in fp32.  ``FP8Experts``
stacks the matrices of several experts for ``kernels.experts``.

A group (a block of weights, or 128 inputs of an activation row) is quantized
as amax = max(max|x|, 2^-100), scale = amax / 448, code = e4m3(x * (448 /
amax)), every step rounded to nearest even in fp32.  A group that holds an
infinity or a NaN gets a NaN scale, so what is computed from it is NaN.

There is no CPU fallback: without CUDA these raise.  Inference only: results
carry no gradient.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import numpy as np
import torch

from .. import _lib
from .device import _ep, epilogue

BLOCK = 128            # inputs (and outputs) that share a scale
RAW_MAX_M = 8          # largest M whose activations the product quantizes itself (no workspace)
_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_CODES = torch.float8_e4m3fn


# torch.cuda.current_stream builds a Stream object (2 us, as long as a launch);
# torch's own code generator asks for the bare handle like this.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = torch.cuda.current_device
# (the cheapest of torch's allocations: 1.5 us against 2 to 2.4 for empty and new_empty)
_empty = torch.empty_strided


def _cuda_device(device=None) -> torch.device:
    if not torch.cuda.is_available():
        raise RuntimeError("the 8-bit kernels need a CUDA device (B200, sm_100a); none is available")
    dev = torch.device(device if device is not None else "cuda")
    if dev.type != "cuda":
        raise ValueError(f"the 8-bit kernels need a CUDA device, got {dev}")
    return torch.device("cuda", torch.cuda.current_device()) if dev.index is None else dev


def _stream(dev: torch.device) -> int:
    return _raw_stream(dev.index)


def _rows(X: torch.Tensor, what: str) -> torch.Tensor:
    """X as a CUDA matrix of a supported type whose rows are contiguous and
    do not overlap."""
    if not isinstance(X, torch.Tensor):
        raise TypeError(f"{what}: unsupported operand type {type(X).__name__}")
    if not X.is_cuda:
        raise ValueError(f"{what}: activations must be a CUDA tensor (no CPU path)")
    if X.dim() != 2:
        raise ValueError(f"{what}: activations must be a matrix, got shape {tuple(X.shape)}")
    if X.dtype not in _TYPES:
        X = X.float()
    if X.is_contiguous():
        return X
    if (X.shape[1] > 1 and X.stride(1) != 1) or (X.shape[0] > 1 and X.stride(0) < X.shape[1]):
        X = X.contiguous()
    return X


def _span(t: torch.Tensor):
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _check_output(Y, shape, out_dtype, dev, inputs, what: str) -> None:
    """The caller's output tensor: shape, type, rows, no overlap with an input."""
    if out_dtype is not None and Y.dtype != out_dtype or Y.dtype not in _TYPES:
        raise ValueError(f"{what}: Y must be a {out_dtype or 'float32, bfloat16 or float16'} tensor, got {Y.dtype}")
    if tuple(Y.shape) != tuple(shape) or Y.device != dev:
        raise ValueError(f"{what}: Y must be a {tuple(shape)} tensor on {dev}")
    if (shape[1] > 1 and Y.stride(1) != 1) or (shape[0] > 1 and Y.stride(0) < shape[1]):
        raise ValueError(f"{what}: Y's rows must be contiguous and must not overlap")
    lo, hi = _span(Y)
    for t in inputs:
        a, b = _span(t)
        if a < hi and lo < b:
            raise ValueError(f"{what}: Y overlaps an input")


class FP8Experts:
    """E stacked K x N weights in e4m3 (``shape`` = (E, K, N)).

    ``codes`` is (E, N, K) with one row of K codes per output feature,
    ``scales`` (E, ceil(N/128), ceil(K/128)) fp32:
    W[e, k, n] = codes[e, n, k] * scales[e, n // 128, k // 128]."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        what = type(self).__name__
        if codes.dtype == torch.uint8:
            codes = codes.view(_CODES)
        if codes.dtype != _CODES or codes.dim() != 3 or scales.dim() != 3:
            raise ValueError(f"{what}: codes must be float8_e4m3fn with a row of K codes per output feature")
        E, N, K = codes.shape
        nb, kb = -(-N // BLOCK), -(-K // BLOCK)
        if min(E, N, K) < 1 or tuple(scales.shape) != (E, nb, kb) or scales.dtype != torch.float32:
            raise ValueError(f"{what}: codes {tuple(codes.shape)} need float32 scales {(E, nb, kb)}, "
                             f"got {scales.dtype} {tuple(scales.shape)}")
        if E * N > 0x7fffff00:
            raise ValueError(f"{what}: more than 2^31 weight rows")
        self.device = _cuda_device(codes.device)
        if scales.device != self.device:
            raise ValueError(f"{what}: codes on {self.device}, scales on {scales.device}")
        ld = -(-K // 16) * 16
        store = codes.view(torch.uint8)
        if ld != K or not store.is_contiguous() or store.data_ptr() % 16:
            # the kernels read rows that start on 16-byte boundaries
            store = torch.zeros(E, N, ld, dtype=torch.uint8, device=self.device)
            store[:, :, :K] = codes.view(torch.uint8)
        self._store, self.scales = store, scales.contiguous()
        self.shape = (E, K, N)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.desc = _lib.FP8Desc(codes=store.data_ptr(), scales=self.scales.data_ptr(), ldk=ld, E=E, K=K, N=N)
        self._ref = ctypes.byref(self.desc)
        _lib.check(_lib.load().mtc_fp8_matrix_init(self._ref), what)
        self._status_ptr = self.status.data_ptr()

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor) -> "FP8Experts":
        """Wrap codes (E, N, K) and scales on the GPU.  Shared, not copied, when
        K is a multiple of 16 and the codes are contiguous."""
        return cls(codes, scales)

    @classmethod
    def from_tensor(cls, W, device=None) -> "FP8Experts":
        """Quantize fp32 weights (E, K, N) (numpy or torch) on the GPU."""
        dev = _cuda_device(device if device is not None or not isinstance(W, torch.Tensor) or not W.is_cuda
                           else W.device)
        Wd = torch.as_tensor(W, dtype=torch.float32, device=dev)
        if Wd.dim() != 3 or 0 in Wd.shape:
            raise ValueError(f"{cls.__name__}: weights must be (experts, inputs, outputs), got {tuple(Wd.shape)}")
        E, K, N = Wd.shape
        ld = -(-K // 16) * 16
        codes = torch.zeros(E, N, ld, dtype=torch.uint8, device=dev)
        scales = torch.empty(E, -(-N // BLOCK), -(-K // BLOCK), dtype=torch.float32, device=dev)
        lib = _lib.load()
        with torch.cuda.device(dev):
            for e in range(E):
                We = Wd[e] if Wd[e].stride(1) == 1 and Wd[e].stride(0) >= N else Wd[e].contiguous()
                _lib.check(lib.mtc_fp8_pack(We.data_ptr(), K, N, max(We.stride(0), N), codes[e].data_ptr(), ld,
                                            scales[e].data_ptr(), _stream(dev)), "fp8 pack")
        return cls(codes[:, :, :K].view(_CODES) if ld == K else codes.view(_CODES)[:, :, :K], scales)

    @property
    def codes(self) -> torch.Tensor:
        """The e4m3 codes, (E, N, K)."""
        return self._store.view(_CODES)[:, :, :self.shape[1]]

    @property
    def weight_bytes(self) -> int:
        E, K, N = self.shape
        return E * K * N + 4 * self.scales.numel()

    @property
    def average_bits_per_element(self) -> float:
        E, K, N = self.shape
        return 8.0 * self.weight_bytes / (E * K * N)

    def to_tensor(self) -> torch.Tensor:
        """The weights as fp32 (E, K, N): code times scale."""
        E, K, N = self.shape
        out = torch.empty(E, K, N, dtype=torch.float32, device=self.device)
        lib = _lib.load()
        with torch.cuda.device(self.device):
            for e in range(E):
                _lib.check(lib.mtc_fp8_unpack(self._ref, e, out[e].data_ptr(), N, _stream(self.device)), "fp8 unpack")
        return out

    def to_array(self) -> np.ndarray:
        return self.to_tensor().cpu().numpy()

    def check_status(self):
        """Raise if a kernel reported a runtime problem (synchronises)."""
        v = int(self.status.item())
        if v:
            self.status.zero_()
            raise RuntimeError("MTC kernel status: " + ("pipeline wait timed out" if v & _lib.STATUS_TIMEOUT
                                                        else f"bits {v:#x}"))


class FP8Matrix(FP8Experts):
    """One K x N weight in e4m3 (``shape`` = (K, N)): codes (N, K), scales
    (ceil(N/128), ceil(K/128)).

    The ``scales`` attribute keeps the stack's leading axis,
    (1, ceil(N/128), ceil(K/128)); ``from_codes`` takes either form."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dim() != 2 or scales.dim() not in (2, 3):
            raise ValueError("FP8Matrix: codes and scales must be matrices")
        super().__init__(codes[None], scales if scales.dim() == 3 else scales[None])
        self.shape = self.shape[1:]

    @classmethod
    def from_tensor(cls, W, device=None) -> "FP8Matrix":
        """Quantize fp32 weights (K, N) (numpy or torch) on the GPU."""
        if len(W.shape) != 2:
            raise ValueError(f"FP8Matrix: weights must be a matrix, got {tuple(W.shape)}")
        stack = FP8Experts.from_tensor(W[None], device)
        return cls(stack.codes[0], stack.scales[0])

    @classmethod
    def from_mtc(cls, mat, device=None) -> "FP8Matrix":
        """The 8-bit form of a packed ``MTCMatrix`` (its exact dequantisation, requantized)."""
        return cls.from_tensor(mat.to_tensor(_cuda_device(device)))

    @property
    def codes(self) -> torch.Tensor:
        """The e4m3 codes, (N, K)."""
        return self._store.view(_CODES)[0, :, :self.shape[0]]

    @property
    def weight_bytes(self) -> int:
        return self.shape[0] * self.shape[1] + 4 * self.scales.numel()

    @property
    def average_bits_per_element(self) -> float:
        return 8.0 * self.weight_bytes / (self.shape[0] * self.shape[1])

    def to_tensor(self) -> torch.Tensor:
        """The weights as fp32 (K, N): code times scale."""
        K, N = self.shape
        out = torch.empty(K, N, dtype=torch.float32, device=self.device)
        with torch.cuda.device(self.device):
            _lib.check(_lib.load().mtc_fp8_unpack(self._ref, 0, out.data_ptr(), N, _stream(self.device)), "fp8 unpack")
        return out


def fp8_quantize(X: torch.Tensor):
    """Activations (M, K) to (codes (M, K) float8_e4m3fn, scales (M, ceil(K/128)) float32).

    The tensors are views: rows of codes are padded to a multiple of 16
    bytes, the scales are stored by group (their column stride is M)."""
    X = _rows(X, "fp8_quantize")
    dev = X.device
    if _current_device() != dev.index:
        with torch.cuda.device(dev):
            return fp8_quantize(X)
    M, K = X.shape
    if K < 1:
        raise ValueError("fp8_quantize: rows without values")
    ld, kb = -(-K // 16) * 16, -(-K // BLOCK)
    codes = _empty((M, K), (ld, 1), dtype=_CODES, device=dev)
    scales = _empty((M, kb), (1, M), dtype=torch.float32, device=dev)
    if M:
        rc = _lib.load().mtc_fp8_quantize(X.data_ptr(), _TYPES[X.dtype], M, K, X.stride(0) if M > 1 else K,
                                          codes.data_ptr(), ld, scales.data_ptr(), M, _raw_stream(dev.index))
        if rc:
            _lib.check(rc, "fp8 quantize")
    return codes, scales


def fp8_gemm(X, W: FP8Matrix, bias=None, activation: Optional[str] = None, Y=None, *, out_dtype=None):
    """Y = act(quantized(X) @ W + bias).

    X: (M, K) CUDA tensor (fp32, bf16 or fp16; other types become fp32), or a
    numpy array, for which numpy is returned.  bias: None or N floats.
    activation: None, "relu", "silu" or "gelu_tanh".  The result is fp32, or
    ``out_dtype`` (float32, bfloat16, float16), rounded once; ``Y`` takes it
    if given (it must not overlap X)."""
    if not isinstance(W, FP8Matrix):
        raise TypeError("fp8_gemm: the right operand must be an FP8Matrix")
    dev = W.device
    if isinstance(X, np.ndarray):
        Xd = torch.from_numpy(np.ascontiguousarray(X, dtype=np.float32)).to(dev)
        y = fp8_gemm(Xd, W, bias, activation, Y, out_dtype=out_dtype)
        W.check_status()
        return y.float().cpu().numpy()
    X = _rows(X, "fp8_gemm")
    if X.device != dev:
        raise ValueError(f"fp8_gemm: activations on {X.device}, weights on {dev}")
    index = dev.index
    if _current_device() != index:
        with torch.cuda.device(dev):
            return fp8_gemm(X, W, bias, activation, Y, out_dtype=out_dtype)
    M, K = X.shape
    K2, N = W.shape
    assert K == K2, f"Shape mismatch: {tuple(X.shape)} vs {W.shape}"
    ep = None
    if bias is not None:
        if not (isinstance(bias, torch.Tensor) and bias.dtype == torch.float32 and bias.device == dev
                and bias.dim() == 1 and bias.is_contiguous()):
            bias = torch.as_tensor(bias, dtype=torch.float32, device=dev).reshape(-1).contiguous()
        if bias.shape[0] != N:
            raise ValueError(f"bias has {bias.shape[0]} values, the output {N} columns")
        ep = _ep(epilogue(bias, activation))
    elif activation is not None:
        ep = _ep(epilogue(None, activation))
    if Y is None:
        y_type = _TYPES.get(out_dtype)
        if y_type is None:
            if out_dtype is not None:
                raise ValueError(f"fp8_gemm: output type {out_dtype} (one of float32, bfloat16, float16)")
            out_dtype, y_type = torch.float32, _lib.F32
        Y, ldy = _empty((M, N), (N, 1), dtype=out_dtype, device=dev), N
    else:
        _check_output(Y, (M, N), out_dtype, dev, (X, W._store, W.scales) if bias is None else
                      (X, W._store, W.scales, bias), "fp8_gemm")
        y_type, ldy = _TYPES[Y.dtype], Y.stride(0) if M > 1 else N
    if M:
        lib = _lib.load()
        at, need = None, 0
        if M > RAW_MAX_M:
            need = lib.mtc_fp8_gemm_workspace_bytes(W._ref, M)
            ws = _empty((need,), (1,), dtype=torch.uint8, device=dev)
            at = ws.data_ptr()
        rc = lib.mtc_fp8_gemm(W._ref, X.data_ptr(), _TYPES[X.dtype], M, X.stride(0) if M > 1 else K, Y.data_ptr(),
                              y_type, ldy, at, need, W._status_ptr, ep, _raw_stream(index))
        if rc:
            _lib.check(rc, "fp8 gemm")
    return Y
