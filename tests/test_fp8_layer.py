"""CPU: Fp8Linear as a module."""

from __future__ import annotations

import torch

from convrot_mlx_amd import Fp8Linear

FP8 = torch.float8_e4m3fn


def test_moved_without_a_bias():
    """A bias taken away (None, which the call accepts) stays away where the layer is cast or moved."""
    layer = Fp8Linear(16, 8)
    layer.bias = None
    for moved in (layer.half(), layer.to("cpu"), torch.nn.Sequential(layer).to(torch.bfloat16)[0], layer.to("meta")):
        assert moved.bias is None and moved.qweight.dtype == FP8 and moved.scales.dtype == torch.float32
    assert moved.qweight.device.type == "meta"
