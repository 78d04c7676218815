"""Every activation of the gate in every form of the experts' products."""

import pytest
import torch

from test_gpu_experts import dev, forward  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("T,E,k,D,I", [(1, 16, 4, 200, 130), (1, 16, 4, 2048, 130), (9, 16, 4, 300, 260),
                                       (120, 16, 2, 260, 200), (700, 4, 2, 200, 150)])
def test_gate_activations(dev, T, E, k, D, I, activation):
    forward(dev, T, E, k, D, I, torch.float32, activation=activation, seed=T)
