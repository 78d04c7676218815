"""Mixture-of-experts operators: routing and the experts' gated feed-forward.

``route_experts`` turns router logits into the chosen experts and their
weights; ``experts_forward`` runs the chosen experts, whose matrices are
``FP8Experts`` stacks, on every token:

    y_t = sum_j weights[t, j] * (act(x_t @ gate_e) * (x_t @ up_e)) @ down_e,   e = ids[t, j]

Both enqueue their kernels on the current stream and do not synchronise.  A
wait that ran out in a kernel is reported by ``gate.check_status()``.
Inference only: results carry no gradient.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from .fp8 import _TYPES, FP8Experts, _check_output, _current_device, _empty, _raw_stream, _rows

MAX_EXPERTS = 1024
MAX_TOP_K = 32
MAX_GROUPS = 32


def route_experts(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias=None, n_groups: int = 1,
                  top_groups: int = 1, renormalize: bool = True, scale: float = 1.0):
    """(ids (T, top_k) int32, weights (T, top_k) float32) from router logits (T, E).

    Scores are the softmax over the experts or the sigmoid of the logits.
    The experts are chosen by score + ``bias`` (E finite floats, to balance
    their load), compared in 64 bits (without bias and groups by the logits,
    whose order that is), best first, ties to the lowest index.  With
    ``n_groups`` > 1 only the experts of the ``top_groups`` groups (equal
    consecutive parts of the E experts) with the largest sum of their two best
    choices compete.  The weights are the scores without the bias, divided by
    their sum if ``renormalize``, times ``scale``.

    A logit of -inf or NaN masks its expert: score 0, chosen only when no
    other of the competing ones is left, and never one of a group's two best
    (a group's only free expert counts alone, a group without one comes after
    all others); a row of masked experts gets weights 0.  +inf counts as the
    largest finite number."""
    logits = _rows(logits, "route_experts")
    T, E = logits.shape
    if score not in _lib.SCORES:
        raise ValueError(f"route_experts: unknown score {score!r} (softmax or sigmoid)")
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"route_experts: {E} experts (1..{MAX_EXPERTS})")
    if not 1 <= n_groups <= MAX_GROUPS or E % n_groups or not 1 <= top_groups <= n_groups:
        raise ValueError(f"route_experts: {E} experts in {n_groups} groups, {top_groups} of them kept")
    if not 1 <= top_k <= min(MAX_TOP_K, top_groups * (E // n_groups)):
        raise ValueError(f"route_experts: top_k={top_k} outside 1..{min(MAX_TOP_K, top_groups * (E // n_groups))}")
    dev = logits.device
    if _current_device() != dev.index:
        with torch.cuda.device(dev):
            return route_experts(logits, top_k, score=score, bias=bias, n_groups=n_groups, top_groups=top_groups,
                                 renormalize=renormalize, scale=scale)
    if bias is not None:
        if not (isinstance(bias, torch.Tensor) and bias.dtype == torch.float32 and bias.device == dev
                and bias.dim() == 1 and bias.is_contiguous()):
            bias = torch.as_tensor(bias, dtype=torch.float32, device=dev).reshape(-1).contiguous()
        if bias.shape[0] != E:
            raise ValueError(f"route_experts: bias has {bias.shape[0]} values, there are {E} experts")
    ids = _empty((T, top_k), (top_k, 1), dtype=torch.int32, device=dev)
    weights = _empty((T, top_k), (top_k, 1), dtype=torch.float32, device=dev)
    if T:
        rc = _lib.load().mtc_route_experts(
            logits.data_ptr(), _TYPES[logits.dtype], T, E, logits.stride(0) if T > 1 else E, top_k, _lib.SCORES[score],
            None if bias is None else bias.data_ptr(), n_groups, top_groups, bool(renormalize), scale, ids.data_ptr(),
            weights.data_ptr(), _raw_stream(dev.index))
        if rc:
            _lib.check(rc, "route experts")
    return ids, weights


def experts_forward(X: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, gate: FP8Experts, up: FP8Experts,
                    down: FP8Experts, *, activation: Optional[str] = "silu", Y=None, out_dtype=None) -> torch.Tensor:
    """The weighted sum of the chosen experts' gated feed-forward for every token.

    X: (T, D) CUDA tensor (fp32, bf16, fp16); ids (T, k) integers, weights
    (T, k) floats, as ``route_experts`` gives them; gate and up (E, D, I),
    down (E, I, D).  An id outside 0..E-1 is no expert and adds nothing (a
    padded token, or an expert of another rank).  The activations and the
    gated values act(gate) * up (fp32 until then) are quantized as in
    ``fp8_quantize``; an expert's output and the weighted sum, in the order of
    j, are fp32.  The result is fp32, or rounded once to ``out_dtype``; ``Y``
    takes it if given (it must not overlap an input)."""
    X = _rows(X, "experts_forward")
    for m in (gate, up, down):
        if not isinstance(m, FP8Experts) or len(m.shape) != 3:
            raise TypeError("experts_forward: gate, up and down must be FP8Experts")
    dev = X.device
    index = dev.index
    if _current_device() != index:
        with torch.cuda.device(dev):
            return experts_forward(X, ids, weights, gate, up, down, activation=activation, Y=Y, out_dtype=out_dtype)
    T, D = X.shape
    E, K, I = gate.shape
    assert D == K, f"Shape mismatch: {tuple(X.shape)} vs {gate.shape}"
    if up.shape != gate.shape or down.shape != (E, I, D):
        raise ValueError(f"experts_forward: gate {gate.shape}, up {up.shape} and down {down.shape} do not fit")
    if E > MAX_EXPERTS:
        raise ValueError(f"experts_forward: {E} experts, at most {MAX_EXPERTS}")
    if gate.device != dev or up.device != dev or down.device != dev or ids.device != dev or weights.device != dev:
        raise ValueError(f"experts_forward: all operands must be on {dev}")
    shape = ids.shape
    if len(shape) != 2 or shape[0] != T or shape != weights.shape or not 1 <= shape[1] <= MAX_TOP_K:
        raise ValueError(f"experts_forward: ids {tuple(shape)} and weights {tuple(weights.shape)} for {T} tokens "
                         f"(1..{MAX_TOP_K} experts each)")
    if ids.dtype != torch.int32:
        if ids.dtype.is_floating_point or ids.dtype.is_complex or ids.dtype == torch.bool:
            raise ValueError(f"experts_forward: ids of type {ids.dtype}")
        # (an id that does not fit 32 bits is no expert either)
        ids = ids.to(torch.int64)
        ids = torch.where((ids >= 0) & (ids < E), ids, torch.full_like(ids, -1)).to(torch.int32)
    act = _lib.ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r} (one of relu, silu, gelu_tanh)")
    if weights.dtype != torch.float32:
        weights = weights.to(torch.float32)
    ids, weights = ids.contiguous(), weights.contiguous()
    k = shape[1]
    if Y is None:
        y_type = _TYPES.get(out_dtype)
        if y_type is None:
            if out_dtype is not None:
                raise ValueError(f"experts_forward: output type {out_dtype} (one of float32, bfloat16, float16)")
            out_dtype, y_type = torch.float32, _lib.F32
        Y, ldy = _empty((T, D), (D, 1), dtype=out_dtype, device=dev), D
    else:
        _check_output(Y, (T, D), out_dtype, dev, (X, ids, weights) + tuple(t for m in (gate, up, down)
                                                                           for t in (m._store, m.scales)),
                      "experts_forward")
        y_type, ldy = _TYPES[Y.dtype], Y.stride(0) if T > 1 else D
    if T:
        lib = _lib.load()
        need = lib.mtc_experts_workspace_bytes(gate._ref, T, k, y_type)
        if not need:
            raise ValueError(f"experts_forward: too many rows ({T} x {k})")
        ws = _empty((need,), (1,), dtype=torch.uint8, device=dev)
        rc = lib.mtc_experts_forward(
            gate._ref, up._ref, down._ref, X.data_ptr(), _TYPES[X.dtype], T, X.stride(0) if T > 1 else D,
            ids.data_ptr(), weights.data_ptr(), k, act, Y.data_ptr(), y_type, ldy, ws.data_ptr(), need,
            gate._status_ptr, _raw_stream(index))
        if rc:
            _lib.check(rc, "experts")
    return Y
