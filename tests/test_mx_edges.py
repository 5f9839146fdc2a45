"""MXFP4 operators at their edges: where arguments live, how they are laid out,
what happens after an error. Definitions and bounds are those of ``test_mx``."""

from __future__ import annotations

import pytest
import torch

from mlx_iqk_b200 import MxSwitchGLU
from mlx_iqk_b200 import kernels as K


# ------------------------------------------------------ the layer's arguments


def small_layer(device):
    layer = MxSwitchGLU(4, 64, 32, device=device)
    x = torch.ones((3, 64), device=device)
    idx = torch.zeros((3, 2), dtype=torch.int32, device=device)
    return layer, x, idx


def test_layer_refuses_scores_elsewhere():
    layer, x, idx = small_layer("cpu")
    for scores in (torch.ones((3, 2), device="meta"), [[1.0, 1.0]] * 3):
        with pytest.raises(K.IqkRuntimeError, match="scores"):
            layer(x, idx, scores)


@pytest.mark.gpu
def test_layer_refuses_host_scores(cuda):
    layer, x, idx = small_layer("cuda")
    with pytest.raises(K.IqkRuntimeError, match="scores"):
        layer(x, idx, torch.ones((3, 2)))
    assert layer(x, idx, torch.ones((3, 2), device="cuda")).shape == (3, 64)
