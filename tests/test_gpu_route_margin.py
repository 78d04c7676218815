"""Routing where the scores of a whole row are tiny or spread far apart.

The choice is by 64-bit scores, whatever the 32-bit ones that reach it
first are off by: a sigmoid of a logit near -60 by some 70 ulp of itself, so
two choices further apart than that can change places in 32 bits.
"""

import pytest
import torch

from test_gpu_experts import same_routing
from test_gpu_fp8 import dev, normal  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E", [16, 32, 64, 200])
@pytest.mark.parametrize("level", [-20.0, -45.0, -60.0, -80.0, -88.0, -100.0, 30.0])
def test_sigmoids_of_rows_at_one_level(dev, E, level):
    for step in (1e-6, 1e-5, 1e-3, 1.0):
        # logits near one level: neighbours, or groups, that few ulp of a score set apart
        z = level + step * normal((4000, E), int(-level) + E, dev)
        same_routing(z, 6, score="sigmoid", n_groups=8, top_groups=3, renormalize=False)
        same_routing(z, 4, score="sigmoid", n_groups=4, top_groups=1, renormalize=False,
                     bias=1e-30 * normal((E,), 1, dev))


@pytest.mark.parametrize("E", [32, 64, 256, 1024])
def test_softmax_of_spread_rows(dev, E):
    for spread in (1e-5, 0.1, 3.0, 30.0, 100.0):
        z = spread * normal((3000, E), E, dev)
        same_routing(z, 8, n_groups=8, top_groups=4)
        same_routing(z, 8, n_groups=4, top_groups=2, bias=1e-4 * normal((E,), 2, dev))
