"""Group-limited routing with masked experts.

A group's value is the sum of its two best free choices; a group with one free
expert counts by that one, a group without any comes after all others.
Expected ids are written out, or come from the loops below (64 bits).
"""

import math

import numpy as np
import pytest
import torch

from test_gpu_fp8 import dev, normal  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu
INF = math.inf


def routed(z, k, score, bias, groups, top):
    """ids and weights (divided by their sum), one row and expert at a time."""
    ids, weights = [], []
    for row in z.double().cpu().numpy():
        row = np.where(np.isnan(row), -INF, row)
        free = row > -INF
        s = np.zeros(len(row))
        if score == "softmax":
            s[free] = np.exp(row[free] - row[free].max(initial=-INF))
            s /= max(s.sum(), 1e-300)
        else:
            s[free] = 1 / (1 + np.exp(-row[free]))
        c = s if bias is None else s + bias.double().cpu().numpy()
        size = len(row) // groups
        value = []
        for g in range(groups):
            best = sorted((c[e] for e in range(g * size, (g + 1) * size) if free[e]), reverse=True)[:2]
            value.append(sum(best) if best else -INF)
        kept = sorted(range(groups), key=lambda g: (-value[g], g))[:top]
        order = sorted((e for e in range(len(row)) if e // size in kept),
                       key=lambda e: (not free[e], -c[e] if free[e] else 0.0, e))[:k]
        w = s[order]
        ids.append(order)
        weights.append(w / w.sum() if w.sum() > 0 else 0 * w)
    return torch.tensor(ids, dtype=torch.int32), torch.from_numpy(np.array(weights))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_group_with_one_free_expert(dev, score, dtype):
    from tensorpack_b200.kernels.experts import route_experts

    def ids(rows, k, groups, top, bias=None):
        z = torch.tensor(rows, device=dev, dtype=dtype)
        b = None if bias is None else torch.tensor(bias, device=dev)
        got, w = route_experts(z, k, score=score, bias=b, n_groups=groups, top_groups=top)
        assert torch.isfinite(w).all()
        return got.tolist(), w.tolist()

    zero = [0.0] * 4
    for bias in (None, zero):
        # the only free expert, behind a group without any
        got, w = ids([[-INF, -INF, 2.0, -INF], [-INF, math.nan, -INF, 2.0]], 1, 2, 1, bias)
        assert got == [[2], [3]] and w == [[1.0], [1.0]]
        # one strong expert against two weak ones
        assert ids([[3.0, -INF, -4.0, -4.0]], 1, 2, 1, bias)[0] == [[0]]
    eight = [-INF, -INF, 1.0, -INF, 2.0, -INF, 3.0, -INF]
    assert ids([eight], 2, 4, 1) == ([[6, 7]], [[1.0, 0.0]])
    assert ids([eight], 2, 4, 2)[0] == [[6, 4]]
    assert ids([eight], 3, 4, 3)[0] == [[6, 4, 2]]
    # a bias is part of the choice, also of a single one
    assert ids([eight], 1, 4, 1, [0.0, 0, 9, 0, 0, 0, 0, 0])[0] == [[2]]
    assert ids([eight], 1, 4, 1, [9.0, 9, 0, 0, 0, 0, -9, 0])[0] == [[4]]
    # no free expert at all: by index
    assert ids([[-INF] * 8], 2, 4, 1) == ([[0, 1]], [[0.0, 0.0]])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("E,groups,top,k", [(8, 4, 1, 2), (40, 4, 2, 8), (256, 8, 4, 8), (64, 32, 3, 5), (640, 20, 7, 8),
                                            (1024, 32, 3, 8), (32, 32, 5, 5)])
def test_masked_rows_against_the_loops(dev, E, groups, top, k, biased, score):
    from tensorpack_b200.kernels.experts import route_experts

    z = normal((60, E), E, dev)
    b = normal((E,), 3, dev, scale=0.1) if biased else None
    # rows with ever fewer free experts, down to none
    g = torch.Generator(device=dev).manual_seed(E)
    z[torch.rand(60, E, device=dev, generator=g) < torch.linspace(0.3, 1.01, 60, device=dev)[:, None]] = -INF
    ids, w = route_experts(z, k, score=score, bias=b, n_groups=groups, top_groups=top)
    rid, rw = routed(z, k, score, b, groups, top)
    assert torch.equal(ids.cpu(), rid)
    assert ((w.double().cpu() - rw).abs() <= 2 ** -23 * rw + 1e-45).all()
