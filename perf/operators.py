"""What the 8-bit and expert operators are measured on: inputs, plain forms, exact results.

Four operators of a linear stack whose weights are kept in 8-bit floating point (e4m3):

* ``quantize``: activations to e4m3 codes with one fp32 scale per row and group of 128 inputs;
* ``gemm``: Y = act(X @ W + bias), W in e4m3 with one fp32 scale per 128 x 128 block, X quantized on the way;
* ``route``: scores of a router, limited to the best groups, top-k experts and their weights;
* ``experts``: the gated feed-forward of the chosen experts, Y = sum_j w_j (act(X Wg) * (X Wu)) Wd.

The definition of a quantized group x: a = max(max|x|, 2^-100), scale = a / 448, code = e4m3(x * (448 / a)), each
step rounded to nearest in 32 bits.  ``own`` selects the framework's kernels in ``run``; the plain forms below are
elementary torch operations in 32 bits (64 for the router, whose choices fall next to a border).
"""

import math

import numpy as np
import torch

own = False

F8 = torch.float8_e4m3fn
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
WIDTH = {"fp32": 4, "bf16": 2, "fp16": 2}
FLOOR = 2.0 ** -100
BLOCK = 128


def listed():
    return [
        # the activations of one decode batch before a hidden-size product
        {"name": "quantize-16x4096", "op": "quantize", "M": 16, "K": 4096, "x": "bf16"},
        # a prompt's activations before the down projection of an 8B-shaped layer, fp32 as the framework's own output
        {"name": "quantize-4096x14336", "op": "quantize", "M": 4096, "K": 14336, "x": "fp32"},
        # k/v projection of a 0.5B-shaped layer, one token: the smallest product, all latency
        {"name": "gemm-1x896x128", "op": "gemm", "M": 1, "K": 896, "N": 128, "x": "fp32", "y": "fp32", "bias": True, "act": "none"},
        # gate projection of an 8B-shaped layer, one token: streams 59 MB of weights
        {"name": "gemm-1x4096x14336", "op": "gemm", "M": 1, "K": 4096, "N": 14336, "x": "bf16", "y": "bf16", "bias": False, "act": "silu"},
        # down projection of an 8B-shaped layer, a decode batch
        {"name": "gemm-16x14336x4096", "op": "gemm", "M": 16, "K": 14336, "N": 4096, "x": "bf16", "y": "fp32", "bias": False, "act": "none"},
        # a ragged chunk of a prompt through a layer with odd sizes
        {"name": "gemm-333x4864x901", "op": "gemm", "M": 333, "K": 4864, "N": 901, "x": "fp16", "y": "fp16", "bias": True, "act": "gelu_tanh"},
        # a whole prompt through the gate projection of an 8B-shaped layer
        {"name": "gemm-4096x4096x14336", "op": "gemm", "M": 4096, "K": 4096, "N": 14336, "x": "bf16", "y": "bf16", "bias": False, "act": "none"},
        # one decoded token choosing among 64 experts
        {"name": "route-1x64", "op": "route", "T": 1, "E": 64, "k": 8, "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "renorm": True, "scale": 1.0},
        # a prompt choosing among 256 experts in 8 groups, with a bias that balances their load
        {"name": "route-8192x256", "op": "route", "T": 8192, "E": 256, "k": 8, "score": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "renorm": True, "scale": 2.5},
        # one decoded token through its 8 experts
        {"name": "experts-1", "op": "experts", "T": 1, "E": 64, "k": 8, "D": 2048, "I": 1024, "y": "bf16", "act": "silu"},
        # a decode batch: nearly every expert is used by a few tokens
        {"name": "experts-48", "op": "experts", "T": 48, "E": 128, "k": 8, "D": 2048, "I": 768, "y": "bf16", "act": "silu"},
        # a prompt: every expert has hundreds of tokens, of unequal number
        {"name": "experts-4096", "op": "experts", "T": 4096, "E": 64, "k": 8, "D": 2048, "I": 1408, "y": "bf16", "act": "silu"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "gemm", "gemm", "route", "experts", "experts"])
    if op == "quantize":
        return {"op": op, "M": _log(rng, 1, 8192), "K": _log(rng, 100, 7168), "x": rng.choice(["fp32", "bf16", "fp16"])}
    if op == "gemm":
        m = _log(rng, 1, 4096)
        return {"op": op, "M": m, "K": _log(rng, 100, 14336 if m < 1024 else 4096), "N": _log(rng, 60, 14336),
                "x": rng.choice(["fp32", "bf16", "fp16"]), "y": rng.choice(["fp32", "bf16", "fp16"]), "bias": rng.random() < 0.5,
                "act": rng.choice(["none", "relu", "silu", "gelu_tanh"])}
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        top = rng.randint(1, groups)
        size = rng.randint(8, 32) if groups > 1 else rng.randint(8, 300)
        return {"op": op, "T": _log(rng, 1, 16384), "E": groups * size, "k": rng.randint(1, 8), "score": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "groups": groups, "top_groups": top, "renorm": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5])}
    e = rng.choice([8, 24, 60, 64, 128])
    return {"op": op, "T": _log(rng, 1, 4096), "E": e, "k": rng.randint(1, min(8, e)), "D": 16 * rng.randint(24, 128), "I": rng.randint(100, 1100 if e <= 64 else 700),
            "y": rng.choice(["bf16", "fp16"]), "act": rng.choice(["silu", "gelu_tanh"])}


# ---------------------------------------------------------------------------------------------- inputs
def _activations(g, rows, k):
    """Normal rows with one in a hundred input channels fifty times as large, as in transformer activations."""
    x = torch.randn(rows, k, device="cuda", generator=g)
    return x * torch.where(torch.rand(k, device="cuda", generator=g) < 0.01, 50.0, 1.0)


def _weights(g, k, n):
    """(codes (n, k), scales (n/128, k/128)): heavy-tailed weights, the output feature as the row."""
    w = torch.randn(n, k, device="cuda", generator=g)
    w = w * (0.02 + 0.06 * torch.rand(n, k, device="cuda", generator=g) ** 4)
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    p = torch.zeros(nb * BLOCK, kb * BLOCK, device="cuda")
    p[:n, :k] = w
    p = p.view(nb, BLOCK, kb, BLOCK)
    scale = p.abs().amax((1, 3)) / 448.0
    codes = (p / scale[:, None, :, None]).clamp(-448, 448).view(nb * BLOCK, kb * BLOCK)[:n, :k].to(F8).contiguous()
    return codes, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case, "op": op}
    if op == "quantize":
        s["x"] = _activations(g, case["M"], case["K"]).to(TYPES[case["x"]])
    elif op == "gemm":
        s["x"] = _activations(g, case["M"], case["K"]).to(TYPES[case["x"]])
        s["w"] = _weights(g, case["K"], case["N"])
        s["bias"] = torch.randn(case["N"], device="cuda", generator=g) if case["bias"] else None
    elif op == "route":
        s["logits"] = torch.randn(case["T"], case["E"], device="cuda", generator=g)
        s["bias"] = 0.1 * torch.randn(case["E"], device="cuda", generator=g) if case["bias"] else None
    else:
        t, e, k, d, i = (case[n] for n in ("T", "E", "k", "D", "I"))
        s["x"] = torch.randn(t, d, device="cuda", generator=g).to(torch.bfloat16)
        # unequal loads: some experts are liked several times as much as others
        liking = torch.randn(t, e, device="cuda", generator=g) + 0.5 * torch.randn(e, device="cuda", generator=g)
        top = liking.topk(k, dim=1)
        s["ids"] = top.indices.to(torch.int32)
        s["weights"] = torch.softmax(top.values, 1)
        for name, a, b in (("gate", d, i), ("up", d, i), ("down", i, d)):
            each = [_weights(g, a, b) for _ in range(e)]
            s[name] = torch.stack([c.view(torch.uint8) for c, _ in each]).view(F8), torch.stack([v for _, v in each])
        # what bounds the plain form's buffers: the most rows of one expert, and how many experts have any
        count = torch.bincount(s["ids"].reshape(-1).long(), minlength=e)
        s["capacity"], s["used"] = int(count.max()), int((count > 0).sum())
    if own:
        from tensorpack_b200.kernels.fp8 import FP8Experts, FP8Matrix

        if op == "gemm":
            s["handle"] = FP8Matrix.from_codes(*s["w"])
        elif op == "experts":
            s["handles"] = [FP8Experts.from_codes(*s[name]) for name in ("gate", "up", "down")]
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _quantize(x):
    """(codes (rows, K), scales (rows, K/128)) of fp32 rows."""
    rows, k = x.shape
    kb = -(-k // BLOCK)
    p = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(rows, kb, BLOCK)
    a = p.abs().amax(-1).clamp_min(FLOOR)
    top = torch.full_like(a, 448.0)
    q = (p * (top / a)[..., None]).clamp(-448, 448).to(F8).view(rows, kb * BLOCK)[:, :k]
    return q, a / top


def _spread(codes, scales, rows, cols):
    """fp32 values of codes whose scales hold for `rows` x `cols` blocks (last two axes)."""
    s = scales.repeat_interleave(cols, -1)[..., : codes.shape[-1]]
    if rows > 1:
        s = s.repeat_interleave(rows, -2)[..., : codes.shape[-2], :]
    return codes.float() * s


def _act(y, name):
    if name == "relu":
        return torch.where(y < 0, torch.zeros_like(y), y)
    if name == "silu":
        return y / (1 + torch.exp(-y))
    if name == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    return y


def _plain_gemm(s):
    c = s["case"]
    x = _spread(*_quantize(s["x"].float()), 1, BLOCK)
    y = x @ _spread(*s["w"], BLOCK, BLOCK).T
    if s["bias"] is not None:
        y = y + s["bias"]
    return _act(y, c["act"]).to(TYPES[c["y"]])


def _plain_route(s):
    c = s["case"]
    z = s["logits"].double()
    if c["score"] == "softmax":
        score = torch.exp(z - z.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-z))
    choice = score if s["bias"] is None else score + s["bias"].double()
    if c["groups"] > 1:
        by = choice.view(c["T"], c["groups"], -1)
        value = by.sort(dim=-1, descending=True).values[..., :2].sum(-1)
        best = value.sort(dim=1, descending=True, stable=True).indices[:, : c["top_groups"]]
        keep = torch.zeros_like(value, dtype=torch.bool).scatter(1, best, True)
        choice = torch.where(keep[..., None], by, -math.inf).view(c["T"], -1)
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, : c["k"]]
    w = score.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return ids.to(torch.int32), (w * c["scale"]).float()


def _plain_experts(s):
    c = s["case"]
    t, e, k, cap, used = c["T"], c["E"], c["k"], s["capacity"], s["used"]
    flat = s["ids"].reshape(-1).long()
    count = (flat[:, None] == torch.arange(e, device="cuda")).sum(0)
    chosen = (count == 0).to(torch.int32).sort(stable=True).indices[:used]  # the experts that have rows, in order
    place = torch.zeros(e, dtype=torch.long, device="cuda").scatter(0, chosen, torch.arange(used, device="cuda"))
    order = flat.sort(stable=True).indices
    rank = torch.arange(t * k, device="cuda") - (count.cumsum(0) - count)[flat[order]]
    slot = place[flat[order]] * cap + rank
    x = _spread(*_quantize(s["x"].float()), 1, BLOCK)
    rows = torch.zeros(used * cap, c["D"], device="cuda")
    rows[slot] = x[order // k]
    gate, up, down = (_spread(s[n][0].view(torch.uint8)[chosen].view(F8), s[n][1][chosen], BLOCK, BLOCK).mT for n in ("gate", "up", "down"))
    rows = rows.view(used, cap, -1)
    h = _act(rows @ gate, c["act"]) * (rows @ up)
    h = _spread(*_quantize(h.view(used * cap, -1)), 1, BLOCK).view(used, cap, -1)
    out = (h @ down).view(used * cap, -1)
    back = torch.empty_like(slot).scatter(0, order, slot)
    y = (out[back].view(t, k, -1) * s["weights"][..., None]).sum(1)
    return y.to(TYPES[c["y"]])


def run(s):
    c, op = s["case"], s["op"]
    if not own:
        if op == "quantize":
            return _quantize(s["x"].float())
        return {"gemm": _plain_gemm, "route": _plain_route, "experts": _plain_experts}[op](s)
    from tensorpack_b200.kernels import experts, fp8

    if op == "quantize":
        return fp8.fp8_quantize(s["x"])
    if op == "gemm":
        return fp8.fp8_gemm(s["x"], s["handle"], s["bias"], c["act"], out_dtype=TYPES[c["y"]])
    if op == "route":
        return experts.route_experts(s["logits"], c["k"], score=c["score"], bias=s["bias"], n_groups=c["groups"],
                                     top_groups=c["top_groups"], renormalize=c["renorm"], scale=c["scale"])
    return experts.experts_forward(s["x"], s["ids"], s["weights"], *s["handles"], activation=c["act"], out_dtype=TYPES[c["y"]])


# ---------------------------------------------------------------------------------------------- work and exact results
def work(case):
    op = case["op"]
    if op == "quantize":
        m, k = case["M"], case["K"]
        return {"bytes": m * k * (WIDTH[case["x"]] + 1) + 4 * m * -(-k // BLOCK), "flops": 3 * m * k}
    if op == "gemm":
        m, k, n = case["M"], case["K"], case["N"]
        return {"bytes": m * k * WIDTH[case["x"]] + k * n + 4 * -(-k // BLOCK) * -(-n // BLOCK) + m * n * WIDTH[case["y"]] + 4 * n * case["bias"],
                "flops": 2 * m * k * n}
    if op == "route":
        t, e = case["T"], case["E"]
        return {"bytes": 4 * t * e + 8 * t * case["k"] + 4 * e * case["bias"], "flops": 8 * t * e}
    t, e, k, d, i = (case[n] for n in ("T", "E", "k", "D", "I"))
    used = e * (1 - (1 - k / e) ** t)  # experts with rows, were they chosen evenly
    return {"bytes": used * (3 * d * i + 12 * -(-d // BLOCK) * -(-i // BLOCK)) + t * d * (2 + WIDTH[case["y"]]) + 8 * t * k, "flops": 6 * t * k * d * i}


def _codes64(x):
    """Quantized rows (codes and scales as the format stores them, in 64 bits) of 64-bit rows."""
    v = x.float()
    rows, k = v.shape
    out, scales = torch.zeros(rows, k, dtype=torch.float64, device="cuda"), []
    for b in range(0, k, BLOCK):
        part = v[:, b: b + BLOCK]
        a = torch.maximum(part.abs().max(1).values, torch.tensor(FLOOR, device="cuda"))
        top = torch.full_like(a, 448.0)
        out[:, b: b + BLOCK] = torch.clamp(part * torch.div(top, a)[:, None], min=-448.0, max=448.0).to(F8).double()
        scales.append(torch.div(a, top).double())
    return out, torch.stack(scales, 1)


def _product64(q, sq, w, sw):
    """Sum over blocks of 128 inputs of scale x scale x (codes @ codes), in 64 bits."""
    n = w.shape[0]
    y = torch.zeros(q.shape[0], n, dtype=torch.float64, device="cuda")
    for b in range(sq.shape[1]):
        at = slice(b * BLOCK, (b + 1) * BLOCK)
        col = sw[:, b].double().repeat_interleave(BLOCK)[:n]
        y += (q[:, at] @ w[:, at].double().T) * sq[:, b: b + 1] * col
    return y


def _act64(y, name):
    if name == "relu":
        return y.clamp_min(0)
    if name == "silu":
        return y * torch.sigmoid(y)
    if name == "gelu_tanh":
        return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    return y


def _weights64(s, case):
    """The chosen experts' weights, row by row in numpy's 64 bits."""
    z = s["logits"].double().cpu().numpy()
    if case["score"] == "softmax":
        p = np.exp(z - z.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    else:
        p = 0.5 * (1 + np.tanh(z / 2))
    c = p if s["bias"] is None else p + s["bias"].double().cpu().numpy()
    if case["groups"] > 1:
        size = case["E"] // case["groups"]
        by = np.partition(c.reshape(case["T"], -1, size), size - 2, axis=2)[:, :, -2:].sum(2)
        dropped = np.argsort(-by, axis=1, kind="stable")[:, case["top_groups"]:]
        c = c.copy()
        for j in range(dropped.shape[1]):
            np.put_along_axis(c, dropped[:, j, None] * size + np.arange(size), -np.inf, 1)
    w = np.take_along_axis(p, np.argsort(-c, axis=1, kind="stable")[:, : case["k"]], 1)
    return w / w.sum(1, keepdims=True) * case["scale"] if case["renorm"] else w * case["scale"]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _codes64(s["x"].double())
    if op == "gemm":
        y = _product64(*_codes64(s["x"].double()), *s["w"])
        if s["bias"] is not None:
            y += s["bias"].double()
        return _act64(y, case["act"])
    if op == "route":
        return None, _weights64(s, case)
    q, sq = _codes64(s["x"].double())
    y = torch.zeros(case["T"], case["D"], dtype=torch.float64, device="cuda")
    for e in range(case["E"]):
        token, j = torch.nonzero(s["ids"] == e, as_tuple=True)
        if len(token):
            g = _product64(q[token], sq[token], s["gate"][0][e], s["gate"][1][e])
            u = _product64(q[token], sq[token], s["up"][0][e], s["up"][1][e])
            out = _product64(*_codes64(_act64(g, case["act"]) * u), s["down"][0][e], s["down"][1][e])
            y.index_add_(0, token, out * s["weights"][token, j].double()[:, None])
    return y
