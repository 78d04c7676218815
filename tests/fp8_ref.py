"""Plain restatement of the 8-bit operators for the tests (CPU or GPU torch).

Quantization follows the format's own 32-bit steps, so codes and scales are
compared bit for bit; products and sums are in 64 bits.
"""

import math

import torch

F8 = torch.float8_e4m3fn
FLOOR = 2.0 ** -100


def quantize(x):
    """(codes as float64 (M, K), scales as float64 (M, ceil(K/128))) of a matrix."""
    x = x.float()
    M, K = x.shape
    kb = -(-K // 128)
    q = torch.zeros(M, kb * 128, dtype=torch.float32, device=x.device)
    q[:, :K] = x
    g = q.view(M, kb, 128)
    amax = g.abs().amax(-1)
    fine = torch.isfinite(g).all(-1)
    amax = torch.where(fine, amax.clamp_min(FLOOR), torch.ones_like(amax))
    top = torch.full_like(amax, 448.0)
    codes = (g * torch.div(top, amax)[..., None]).clamp(-448, 448).to(F8).double()
    codes = torch.where(fine[..., None], codes, torch.zeros_like(codes))
    scales = torch.where(fine, torch.div(amax, top), torch.full_like(amax, math.nan)).double()
    return codes.view(M, kb * 128)[:, :K], scales


def pack(W):
    """(codes (N, K) float64, scales (ceil(N/128), ceil(K/128)) float64) of a K x N weight."""
    K, N = W.shape
    kb, nb = -(-K // 128), -(-N // 128)
    p = torch.zeros(nb * 128, kb * 128, device=W.device)
    p[:N, :K] = W.float().T
    b = p.view(nb, 128, kb, 128)
    amax = b.abs().amax((1, 3)).clamp_min(FLOOR)
    top = torch.full_like(amax, 448.0)
    codes = (b * torch.div(top, amax)[:, None, :, None]).clamp(-448, 448).to(F8).double()
    return codes.reshape(nb * 128, kb * 128)[:N, :K], torch.div(amax, top).double()


def spread(codes, scales, rows=1):
    s = scales.repeat_interleave(128, -1)[..., :codes.shape[-1]]
    if rows > 1:
        s = s.repeat_interleave(rows, -2)[..., :codes.shape[-2], :]
    return codes * s


def act(y, name):
    if name == "relu":
        return torch.where(y < 0, torch.zeros_like(y), y)
    if name == "silu":
        return y * torch.sigmoid(y)
    if name == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y


def gemm(x, codes, scales, bias=None, activation=None):
    """(result in 64 bits, sum of the absolute products): the second bounds the fp32 rounding."""
    a, b = spread(*quantize(x)), spread(codes.double(), scales.double(), 128)
    y, mag = a @ b.T, a.abs() @ b.abs().T
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return act(y, activation), mag


def route(logits, k, score="softmax", bias=None, n_groups=1, top_groups=1, renormalize=True, scale=1.0):
    z = logits.double()
    z = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z).clamp_max(3.4028234663852886e38)
    masked = z == -math.inf
    if score == "softmax":
        top = torch.where(masked.all(1, keepdim=True), torch.zeros_like(z[:, :1]), z.amax(1, keepdim=True))
        s = torch.exp(z - top)
        s = s / s.sum(1, keepdim=True).clamp_min(1e-300)
    else:
        s = torch.where(masked, torch.zeros_like(z), 1 / (1 + torch.exp(-z)))
    c = s if bias is None else s + bias.double()
    if bias is None and n_groups == 1:
        c = z  # the order of the scores, also where they meet in 64 bits
    c = torch.where(masked, torch.full_like(c, -math.inf), c)
    T, E = c.shape
    dropped = torch.zeros_like(masked)
    if n_groups > 1:
        by = c.view(T, n_groups, -1)
        v = by.sort(dim=-1, descending=True).values[..., :2].sum(-1)
        order = v.sort(dim=1, descending=True, stable=True).indices[:, top_groups:]
        dropped = torch.zeros_like(v, dtype=torch.bool).scatter(1, order, True).repeat_interleave(E // n_groups, 1)
    # three tiers: free experts by choice, masked ones, dropped groups
    low = torch.finfo(torch.float64).min
    key = torch.where(dropped, torch.full_like(c, -math.inf), torch.where(masked, torch.full_like(c, low), c))
    ids = key.sort(dim=1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, ids)
    if renormalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total.clamp_min(1e-300), torch.zeros_like(w))
    return ids.to(torch.int32), w * scale


def experts(x, ids, weights, gate, up, down, activation="silu"):
    """gate, up, down: (codes (E, N, K), scales (E, N/128, K/128)) pairs."""
    E = gate[0].shape[0]
    y = torch.zeros(x.shape[0], down[0].shape[1], dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(y)
    for e in range(E):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if len(t):
            g, _ = gemm(x[t], gate[0][e], gate[1][e])
            u, _ = gemm(x[t], up[0][e], up[1][e])
            o, m = gemm(act(g, activation) * u, down[0][e], down[1][e])
            w = weights[t, j].double()[:, None]
            y.index_add_(0, t, o * w)
            mag.index_add_(0, t, m * w.abs())
    return y, mag
