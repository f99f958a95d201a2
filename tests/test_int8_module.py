"""CPU: Int8Linear and replace_int8_linears as modules (buffers, state, refusals); no GPU is touched."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from convrot_mlx_amd import Int8Linear, replace_int8_linears


def test_buffers_and_state():
    layer = Int8Linear(50, 7)
    assert layer.qweight.shape == (7, 50) and layer.qweight.dtype == torch.int8
    assert layer.scales.dtype == layer.bias.dtype == torch.float32
    assert set(layer.state_dict()) == {"qweight", "scales", "bias"}
    other = Int8Linear(50, 7)
    layer.qweight.random_(-127, 127), layer.scales.uniform_(), layer.bias.normal_()
    other.load_state_dict(layer.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(layer.state_dict().values(), other.state_dict().values()))
    assert "in_features=50" in repr(layer)


def test_refusals():
    with pytest.raises(ValueError, match="1 to 65536 features"):
        Int8Linear(0, 4)
    with pytest.raises(ValueError, match="1 to 65536 features"):
        Int8Linear(65537, 4)
    layer = Int8Linear(32, 4)
    with pytest.raises(ValueError, match="expected K=32"):
        layer(torch.zeros(2, 16))
    with pytest.raises(ValueError, match="expected K=32"):
        layer.forward_modulated(torch.zeros(2, 16), torch.zeros(16), torch.zeros(16))
    with pytest.raises(ValueError, match="must have shape"):
        layer.load_weight(torch.zeros(4, 16))
    with pytest.raises(RuntimeError, match="ROCm device"):
        layer(torch.zeros(2, 32))
    with pytest.raises(RuntimeError, match="ROCm device"):
        layer.load_weight(torch.zeros(4, 32))


def test_replacement_without_conversion():
    model = nn.Sequential(nn.Linear(12, 8), nn.ReLU(), nn.Sequential(nn.Linear(8, 5, bias=False)))
    assert replace_int8_linears(model, select=lambda name, m: m.in_features == 8, convert=False) == ["2.0"]
    assert isinstance(model[0], nn.Linear) and isinstance(model[2][0], Int8Linear)
    assert not model[2][0].source_has_bias and not model[2][0].qweight.any()
    assert replace_int8_linears(model, convert=False) == ["0"]
    assert replace_int8_linears(model, convert=False) == []
