"""Routing and the experts' feed-forward on the GPU against the plain
restatement (fp8_ref).

Routing: ids are equal (the choice is made in 64 bits on both sides), weights
agree to one rounding to fp32 (2^-24, twice for the scale).

Experts: the gated values are fp32 (relative error below 1e-5) before they are
quantized, so a value that close to the border of two codes may fall on the
other side: at most 2 * 1e-5 / 2^-4 of them, each then off by at most a step,
2^-3.  That is sqrt(3.2e-4) * 2^-3 = 2.3e-3 of the result's norm; half a step
of the output type comes on top twice (the expert's output, the sum).  A row
may hold a few such values: 5e-2 of its own norm tells it from another row.
"""

import math
import os
import subprocess
import sys

import pytest
import torch

import fp8_ref as R
from test_gpu_fp8 import TYPES, dev, normal  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def same_routing(logits, k, **kw):
    from tensorpack_b200.kernels.experts import route_experts

    ids, w = route_experts(logits, k, **kw)
    rid, rw = R.route(logits, k, **kw)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32 and ids.shape == w.shape == (logits.shape[0], k)
    assert torch.equal(ids, rid)
    assert ((w.double() - rw).abs() <= 2 ** -23 * rw.abs() + 1e-45).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 8), (3, 8, 8), (33, 60, 4), (100, 33, 32), (257, 256, 8),
                                   (20, 513, 7), (9, 1024, 32)])
def test_routing(dev, T, E, k, score):
    z = normal((T, E), T + E, dev, scale=2.0)
    b = normal((E,), 5, dev, scale=0.2)
    same_routing(z, k, score=score)
    same_routing(z, k, score=score, bias=b, scale=2.5)
    same_routing(z, k, score=score, bias=b, renormalize=False)


@pytest.mark.parametrize("E,groups,top,k", [(256, 8, 4, 8), (64, 8, 1, 8), (60, 4, 3, 6), (32, 32, 5, 5), (96, 2, 2, 3),
                                            (1024, 32, 3, 8), (640, 20, 7, 8)])
@pytest.mark.parametrize("biased", [False, True])
def test_group_limit(dev, E, groups, top, k, biased):
    z = normal((70, E), E, dev)
    b = normal((E,), 6, dev, scale=0.1) if biased else None
    for score in ("softmax", "sigmoid"):
        same_routing(z, k, score=score, bias=b, n_groups=groups, top_groups=top)


def test_routing_types_strides_ties(dev):
    from tensorpack_b200.kernels.experts import route_experts

    wide = normal((50, 200), 7, dev)
    for z in (wide[:, 3:67], wide[::2, :64], wide.bfloat16()[:, :64], wide.half()[:, 1:33], wide[3:4, :64].expand(5, -1),
              wide.T[:40, :48], wide[:, :64].round(), torch.zeros(4, 64, device=dev)):
        same_routing(z, 8)
        same_routing(z, 8, score="sigmoid", n_groups=8, top_groups=3)
    # values that 32 bits of a score cannot tell apart
    z = torch.zeros(1, 64, device=dev)
    z[0, ::2] = 1e-9 * torch.arange(32, device=dev)
    z[0, 1] = 5.0
    same_routing(z, 8)
    same_routing(z, 8, bias=torch.zeros(64, device=dev))
    ids, w = route_experts(wide[:0, :64], 8)
    assert ids.shape == (0, 8) and w.shape == (0, 8)


def test_masked_experts_and_rows(dev):
    inf = math.inf
    z = normal((6, 40), 8, dev)
    z[0, 5:] = -inf          # fewer free experts than chosen ones
    z[1] = -inf              # none
    z[2, 7], z[2, 9] = math.nan, inf
    z[3] = 60000.0
    z[4, 20:] = torch.finfo(torch.float32).min
    z[5, ::2] = -inf
    b = normal((40,), 9, dev)
    for score in ("softmax", "sigmoid"):
        same_routing(z, 8, score=score)
        same_routing(z, 8, score=score, bias=b, renormalize=False)
        same_routing(z, 8, score=score, bias=b, n_groups=4, top_groups=2)
        same_routing(z, 8, score=score, n_groups=4, top_groups=1)


def stack(E, K, N, seed, dev):
    from tensorpack_b200.kernels.fp8 import FP8Experts

    return FP8Experts.from_tensor(normal((E, K, N), seed, dev, scale=K ** -0.5))


def pairs(*stacks):
    return [(s.codes, s.scales) for s in stacks]


def near(y, ref, dtype):
    tol = 2.5e-3 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps)
    d = y.double() - ref
    assert torch.isfinite(d).all()
    assert d.norm() <= tol * ref.norm() + 1e-30
    assert (d.norm(dim=1) <= 5e-2 * ref.norm(dim=1) + 1e-30).all()


def forward(dev, T, E, k, D, I, dtype, activation="silu", ids=None, seed=0):
    from tensorpack_b200.kernels.experts import experts_forward

    gate, up, down = stack(E, D, I, seed + 1, dev), stack(E, D, I, seed + 2, dev), stack(E, I, D, seed + 3, dev)
    x = normal((T, D), seed + 4, dev, dtype)
    if ids is None:
        ids = normal((T, E), seed + 5, dev).topk(k, 1).indices.to(torch.int32)
    w = torch.softmax(normal(tuple(ids.shape), seed + 6, dev), 1)
    y = experts_forward(x, ids, w, gate, up, down, activation=activation, out_dtype=dtype)
    torch.cuda.synchronize()
    gate.check_status()
    ref, _ = R.experts(x, ids, w, *pairs(gate, up, down), activation=activation)
    assert y.shape == (T, D) and y.dtype == dtype
    near(y, ref, dtype)
    return x, ids, w, (gate, up, down), y


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,E,k,D,I", [
    (1, 1, 1, 16, 1), (1, 64, 8, 256, 130), (3, 8, 2, 100, 60), (40, 16, 4, 300, 257),      # a few rows per expert
    (90, 8, 1, 128, 128), (120, 16, 4, 260, 200), (300, 8, 4, 144, 96),                     # tens
    (700, 4, 2, 200, 150), (1000, 3, 2, 384, 300),                                          # hundreds
    (48, 128, 8, 512, 300), (250, 96, 8, 256, 700), (150, 32, 8, 256, 900),                 # several tiles per SM
])
def test_experts(dev, T, E, k, D, I, dtype):
    forward(dev, T, E, k, D, I, TYPES[dtype], activation="gelu_tanh" if T % 2 else "silu", seed=T)


@pytest.mark.parametrize("rows", [11, 12, 13, 20, 21, 48, 49])
def test_experts_on_both_sides_of_their_variants(dev, rows):
    """`rows` rows per expert on average, all tokens and only some of them
    at real experts."""
    E, k = 6, 2
    T = -(-rows * E // k)
    _, ids, _, _, _ = forward(dev, T, E, k, 272, 264, torch.float32, seed=rows)
    ids = ids.clone()
    ids[::3] = -1
    forward(dev, T, E, k, 272, 264, torch.bfloat16, ids=ids, seed=rows)


@pytest.mark.parametrize("T", [1, 30, 300, 1500])
def test_uneven_experts(dev, T):
    """All tokens at one expert, experts without tokens, the same expert
    twice, ids that name no expert."""
    E, k = 8, 4
    one = torch.full((T, k), 5, dtype=torch.int32, device=dev)
    forward(dev, T, E, k, 144, 130, torch.float32, ids=one, seed=1)
    two = one.clone()
    two[:, 1], two[::2, 2], two[:, 3] = 7, -1, 8
    forward(dev, T, E, k, 144, 130, torch.float32, ids=two, seed=2)
    skew = (normal((T, k), 3, dev).abs() * 1.5).floor().clamp_max(7).to(torch.int32)
    forward(dev, T, E, k, 144, 130, torch.bfloat16, ids=skew, seed=3)


def test_no_expert_and_wide_ids(dev):
    from tensorpack_b200.kernels.experts import experts_forward

    x, ids, w, mats, y = forward(dev, 20, 8, 2, 64, 48, torch.float32)
    wide = ids.long()
    assert torch.equal(y, experts_forward(x, wide, w, *mats))
    wide[3], wide[4, 0] = -1, 2 ** 32 + int(ids[4, 0])
    z = experts_forward(x, wide, w, *mats)
    assert (z[3] == 0).all()
    ref, _ = R.experts(x[4:5], torch.cat([torch.full_like(ids[4:5, :1], -1), ids[4:5, 1:]], 1), w[4:5], *pairs(*mats))
    near(z[4:5], ref, torch.float32)
    assert (experts_forward(x, torch.full_like(ids, -1), w, *mats) == 0).all()
    assert experts_forward(x[:0], ids[:0], w[:0], *mats).shape == (0, 64)


@pytest.mark.parametrize("T", [7, 200, 1200])
def test_output_views_and_repeats(dev, T):
    from tensorpack_b200.kernels.experts import experts_forward

    x, ids, w, mats, y = forward(dev, T, 4, 2, 100, 90, torch.bfloat16)
    hold = torch.full((T + 2, 109), 7.0, device=dev, dtype=torch.bfloat16)
    out = hold[1:T + 1, 5:105]
    assert experts_forward(x, ids, w, *mats, Y=out) is out and torch.equal(out, y)
    edge = torch.ones_like(hold, dtype=torch.bool)
    edge[1:T + 1, 5:105] = False
    assert (hold[edge] == 7).all()
    wide = torch.zeros(T, 120, device=dev, dtype=torch.bfloat16)
    wide[:, 3:103] = x
    assert torch.equal(experts_forward(wide[:, 3:103], ids, w, *mats, out_dtype=torch.bfloat16), y)


def test_a_bad_token_stays_alone(dev):
    from tensorpack_b200.kernels.experts import experts_forward

    for T in (20, 300, 1200):
        x, ids, w, mats, y = forward(dev, T, 4, 2, 128, 64, torch.float32, seed=T)
        x = x.clone()
        x[3, 7] = math.nan
        z = experts_forward(x, ids, w, *mats)
        others = torch.arange(T, device=dev) != 3
        assert torch.isnan(z[3]).all() and torch.equal(z[others], y[others])


@pytest.mark.parametrize("T", [1, 100, 1200])
def test_the_layer_with_a_packed_router(dev, T):
    """Router logits from the packed linear layer, routing, experts: the run
    of them that a model makes, eagerly, on another stream and captured."""
    from tensorpack_b200.kernels.experts import experts_forward, route_experts
    from tensorpack_b200.nn import ExpertsFP8, LinearMTCAdaptive

    E, D, I, k = 16, 128, 96, 4
    router = LinearMTCAdaptive(D, E, seed=3)
    mats = stack(E, D, I, 1, dev), stack(E, D, I, 2, dev), stack(E, I, D, 3, dev)
    bias = normal((E,), 4, dev, scale=0.05)
    layer = ExpertsFP8(router, *mats, k, score="sigmoid", bias=bias, n_groups=4, top_groups=2, scale=1.5)
    x = normal((T, D), 5, dev)
    y = layer(x)
    ids, w = route_experts(router(x), k, score="sigmoid", bias=bias, n_groups=4, top_groups=2, scale=1.5)
    assert torch.equal(y, experts_forward(x, ids, w, *mats))
    ref, _ = R.experts(x, *R.route(router(x), k, score="sigmoid", bias=bias, n_groups=4, top_groups=2, scale=1.5),
                       *pairs(*mats))
    near(y, ref, torch.float32)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        z = layer(x)
    torch.cuda.synchronize()
    assert torch.equal(z, y)
    graphs, outs, held = [], [], [x.clone(), x.flip(0).contiguous()]
    for h in held:
        logits = router(h)  # eager: the packed layer keeps its own workspaces
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(experts_forward(h, *route_experts(logits, k), *mats))
        graphs.append((g, logits))
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for h, o, (_, logits) in zip(held, outs, graphs):
        assert torch.equal(o, experts_forward(h, *route_experts(logits, k), *mats))
    assert layer.weight_bytes == sum(m.weight_bytes for m in mats)


def test_refusals(dev):
    from tensorpack_b200.kernels.experts import experts_forward, route_experts
    from tensorpack_b200.nn import ExpertsFP8

    z = normal((4, 16), 1, dev)
    for kw in (dict(top_k=0), dict(top_k=17), dict(top_k=2, score="tanh"), dict(top_k=2, n_groups=3),
               dict(top_k=2, n_groups=4, top_groups=5), dict(top_k=9, n_groups=4, top_groups=2),
               dict(top_k=2, bias=torch.zeros(15, device=dev))):
        with pytest.raises(ValueError):
            route_experts(z, **kw)
    with pytest.raises(ValueError):
        route_experts(torch.zeros(2, 1025, device=dev), 2)
    with pytest.raises(ValueError):
        route_experts(z[0], 2)
    gate, up, down = stack(4, 64, 48, 1, dev), stack(4, 64, 48, 2, dev), stack(4, 48, 64, 3, dev)
    x, ids, w = normal((5, 64), 4, dev), torch.zeros(5, 2, dtype=torch.int32, device=dev), torch.ones(5, 2, device=dev)
    with pytest.raises(AssertionError, match="Shape mismatch"):
        experts_forward(x[:, :60], ids, w, gate, up, down)
    with pytest.raises(ValueError, match="fit"):
        experts_forward(x, ids, w, gate, up, gate)
    with pytest.raises(TypeError):
        experts_forward(x, ids, w, gate, up, None)
    for i, v in ((ids[:4], w), (ids, w[:, :1]), (ids[:, :0], w[:, :0]), (ids.float(), w),
                 (ids[:, :1].expand(-1, 33), w[:, :1].expand(-1, 33))):
        with pytest.raises(ValueError):
            experts_forward(x, i, v, gate, up, down)
    with pytest.raises(ValueError, match="must be on"):
        experts_forward(x, ids.cpu(), w, gate, up, down)
    with pytest.raises(ValueError, match="activation"):
        experts_forward(x, ids, w, gate, up, down, activation="tanh")
    with pytest.raises(ValueError, match="overlaps"):
        experts_forward(x, ids, w, gate, up, down, Y=x)
    with pytest.raises(ValueError, match="logits"):
        ExpertsFP8(lambda v: v, gate, up, down, 2)(x)
    with pytest.raises(ValueError, match="fit"):
        ExpertsFP8(lambda v: v, gate, up, gate, 2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_choices_next_to_a_border(dev, score):
    """Choices closer than fp32 tells apart, at the last place and at the
    groups' border: decided in 64 bits."""
    g = torch.Generator(device=dev).manual_seed(1)
    base = torch.randn(200, 1, device=dev, generator=g).expand(-1, 64)
    z = base + 2e-7 * torch.randn(200, 64, device=dev, generator=g)
    b = 1e-8 * torch.randn(64, device=dev, generator=g)
    same_routing(z, 8, score=score)
    same_routing(z, 8, score=score, bias=b)
    same_routing(z, 8, score=score, bias=b, n_groups=8, top_groups=3)
    same_routing(z, 6, score=score, n_groups=4, top_groups=2, renormalize=False)
    same_routing(torch.zeros(5, 64, device=dev), 8, score=score, bias=b, n_groups=8, top_groups=2)
    signs = torch.where(torch.randn(20, 64, device=dev, generator=g) < 0, -0.0, 0.0)
    same_routing(signs, 8, score=score)
    same_routing(signs, 8, score=score, n_groups=8, top_groups=2)


def test_one_token_with_rows_of_no_expert(dev):
    ids = torch.tensor([[3, -1, 7, 3, 8, 2 ** 30]], dtype=torch.int32, device=dev)
    forward(dev, 1, 8, 6, 200, 130, torch.float32, ids=ids)
    forward(dev, 1, 8, 6, 200, 130, torch.bfloat16, ids=torch.full_like(ids, -5))


FIRST_CALLS = """
import torch
from tensorpack_b200.kernels import experts, fp8
dev = torch.device("cuda")
g = torch.Generator(device=dev).manual_seed(1)
w = fp8.FP8Matrix.from_tensor(torch.randn(2048, 512, device=dev, generator=g))
mats = [fp8.FP8Experts.from_tensor(torch.randn(4, a, b, device=dev, generator=g)) for a, b in
        ((512, 128), (512, 128), (128, 512))]
def run(x):
    y = fp8.fp8_gemm(x, w, activation="silu")
    ids, weights = experts.route_experts(y[:, :4], 2)
    return experts.experts_forward(y, ids, weights, *mats)
xs = [torch.randn(n, 2048, device=dev, generator=g) for n in (1, 5, 30, 300)]
s = torch.cuda.Stream()
graphs, outs = [], []
for x in xs:   # every kernel's first launch is a captured one
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        outs.append(run(x))
    graphs.append(graph)
for _ in range(3):
    for graph in graphs:
        graph.replay()
torch.cuda.synchronize()
w.check_status()
for x, y in zip(xs, outs):
    assert y.isfinite().all() and y.abs().max() > 0 and torch.equal(y, run(x))
"""


def test_first_calls_inside_a_capture(dev):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_an_output_on_top_of_the_weights_is_refused(dev):
    from tensorpack_b200.kernels.experts import experts_forward
    from tensorpack_b200.kernels.fp8 import FP8Matrix, fp8_gemm

    codes = torch.zeros(128, 256, dtype=torch.uint8, device=dev)
    m = FP8Matrix.from_codes(codes, torch.ones(1, 2, device=dev))
    x = torch.ones(3, 256, device=dev)
    with pytest.raises(ValueError, match="overlaps"):
        fp8_gemm(x, m, Y=codes.view(-1).view(torch.float32)[:3 * 128].view(3, 128))
    E, D, I = 2, 128, 128
    mats = stack(E, D, I, 1, dev), stack(E, D, I, 2, dev), stack(E, I, D, 3, dev)
    ids = torch.zeros(3, 1, dtype=torch.int32, device=dev)
    y = mats[2]._store.view(-1).view(torch.float32)[:3 * D].view(3, D)
    with pytest.raises(ValueError, match="overlaps"):
        experts_forward(x[:, :D], ids, ids.float(), *mats, Y=y)
