"""CPU: what Int8Linear checks of its own tensors, which a state dict or an assignment may have replaced,
before a kernel reads as far as the layer's shape says."""

from __future__ import annotations

import pytest
import torch

from convrot_mlx_amd import Int8Linear


def calls(layer, rows=2):
    x = torch.zeros(rows, layer.in_features)
    yield lambda: layer(x)
    yield lambda: layer.forward_modulated(x, torch.zeros(layer.in_features), torch.zeros(layer.in_features))


@pytest.mark.parametrize("name,value,text", [
    ("scales", torch.ones(1), "weight scales must have shape"), ("scales", torch.ones(6, 1), "weight scales"),
    ("bias", torch.ones(5), "bias must have shape"), ("qweight", torch.zeros(5, 32, dtype=torch.int8), "weight scales"),
    ("qweight", torch.zeros(6, 48, dtype=torch.int8), "N x K with K=32"),
    ("qweight", torch.zeros(6, 32, dtype=torch.uint8), "2D int8"),
])
def test_replaced_tensors_of_another_size(name, value, text):
    layer = Int8Linear(32, 6)
    setattr(layer, name, value)
    for call in calls(layer):
        with pytest.raises(ValueError, match=text):
            call()


def test_weight_and_scales_of_another_width_together():
    layer = Int8Linear(32, 6)
    layer.qweight, layer.scales, layer.bias = torch.zeros(5, 32, dtype=torch.int8), torch.ones(5), torch.zeros(5)
    for call in calls(layer):
        with pytest.raises(ValueError, match="must have 6 rows"):
            call()


def test_loaded_bias_of_another_size():
    layer = Int8Linear(32, 6)
    with pytest.raises(ValueError, match="bias must have shape"):
        layer.load_weight(torch.zeros(6, 32), torch.zeros(1))


@pytest.mark.parametrize("k", [64, 50])
def test_strided_weight_is_read_in_order(k):
    """A weight assigned as a view whose features are not adjacent, or whose rows are not whole 16-byte
    steps apart, reaches the kernels as the values it holds."""
    q = torch.randint(-127, 128, (4, 2 * k), dtype=torch.int8)
    for view in (q[:, ::2], q[:, :k], q[:, 1: k + 1], q.t().contiguous().t()[:, :k]):
        layer = Int8Linear(k, 4)
        layer.load_state_dict({**layer.state_dict(), "qweight": view}, assign=True)
        w = layer._weight()
        assert w.stride(1) == 1 and w.stride(0) % 16 == 0 and w.data_ptr() % 16 == 0
        assert torch.equal(w[:, :k], view) and not w[:, k:].any()


def test_weights_of_inference_mode():
    with torch.inference_mode():
        layer = Int8Linear(50, 4)
        layer.qweight.random_(-127, 128)
        for _ in range(2):
            assert torch.equal(layer._weight()[:, :50], layer.qweight)
            layer.qweight.neg_()


def test_copies_of_a_layer_read_their_own_weight():
    import copy
    import pickle

    layer = Int8Linear(50, 4)
    layer.qweight.random_(-127, 128)
    layer._weight()
    for other in (copy.deepcopy(layer), pickle.loads(pickle.dumps(layer))):
        assert torch.equal(other._weight(), layer._weight())
        other.qweight.neg_()
        assert torch.equal(other._weight()[:, :50], -layer.qweight)
    assert torch.equal(layer._weight()[:, :50], layer.qweight)


def test_single_row_operands_stay_in_place():
    from convrot_mlx_amd import int8

    wide = torch.zeros((2, 69), dtype=torch.int8)
    for t in (wide[:1, :64], torch.zeros((64, 1), dtype=torch.int8).t()):
        assert int8._operand(t, True) is t and int8._row_stride(t) == 64
    t = wide[:1, :50]  # the kernels read 64 bytes: of codes any, of a weight zeros
    assert int8._operand(t, False) is t and int8._row_stride(t) == 64
    assert int8._operand(t, True) is not t
    end = torch.zeros(50, dtype=torch.int8)[None]  # 64 bytes would pass the end of its memory
    assert int8._operand(end, False).shape == (1, 64)
