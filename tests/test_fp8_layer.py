"""CPU: Fp8Linear as a module."""

from __future__ import annotations

import contextlib

import torch

from convrot_mlx_amd import Fp8Linear, _native, fp8

FP8 = torch.float8_e4m3fn


def test_moved_without_a_bias():
    """A bias taken away (None, which the call accepts) stays away where the layer is cast or moved."""
    layer = Fp8Linear(16, 8)
    layer.bias = None
    for moved in (layer.half(), layer.to("cpu"), torch.nn.Sequential(layer).to(torch.bfloat16)[0], layer.to("meta")):
        assert moved.bias is None and moved.qweight.dtype == FP8 and moved.scales.dtype == torch.float32
    assert moved.qweight.device.type == "meta"


def test_norm_on_the_device_of_its_rows(monkeypatch):
    """Every launch of a call has the rows' device as the current one, the norm's in front of the linear too."""
    current, seen = [], []

    @contextlib.contextmanager
    def on(device):
        current.append(device)
        yield
        current.pop()

    def norm(x, **kw):
        seen.append(list(current))
        return x

    monkeypatch.setattr(_native, "on", on)
    monkeypatch.setattr(fp8, "hip_layer_norm", norm)
    layer = Fp8Linear(16, 8)
    monkeypatch.setattr(layer, "forward", lambda x, **kw: x)
    x = torch.zeros(2, 16)
    assert layer.forward_modulated(x, x[:1], x[:1]) is x
    assert seen == [[x.device]]
