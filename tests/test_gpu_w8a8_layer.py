"""GPU: Int8Linear and the 8-bit functions around their product: where operands lie, streams, graphs."""

from __future__ import annotations

import pytest
import torch

from test_gpu_w8a8 import BF16, operands, product_plain, quantize_plain

pytestmark = pytest.mark.gpu


def layer_and_rows(seed, k, n, rows, dev):
    """A layer of random codes, bf16 rows, and what the layer gives for them."""
    from convrot_mlx_amd import Int8Linear

    host, (_, qw, _, ws, bias) = operands(seed, rows, n, k, dev)
    layer = Int8Linear(k, n, device=dev)
    layer.qweight, layer.scales, layer.bias = qw, ws, bias
    x = torch.randn((rows, k), generator=torch.Generator().manual_seed(seed)).to(BF16)
    codes, xs = quantize_plain(x)
    return layer, x.to(dev), product_plain(codes, host[1], xs, *host[3:], BF16)


@pytest.mark.parametrize("name", ["scales", "bias", "qweight"])
def test_tensors_elsewhere_are_refused(dev, name):
    layer, x, _ = layer_and_rows(1, 64, 8, 3, dev)
    setattr(layer, name, getattr(layer, name).cpu())
    shift = torch.zeros(64, dtype=BF16, device=dev)
    for call in (lambda: layer(x), lambda: layer.forward_modulated(x, shift, shift)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


@pytest.mark.parametrize("k", [64, 50])
def test_strided_weight(dev, k):
    layer, x, want = layer_and_rows(2, k, 40, 5, dev)
    wide = torch.zeros((40, 2 * k), dtype=torch.int8, device=dev)
    wide[:, ::2] = layer.qweight
    layer.load_state_dict({**layer.state_dict(), "qweight": wide[:, ::2]}, assign=True)
    assert torch.equal(layer(x).cpu(), want)
