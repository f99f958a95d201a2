"""GPU: the forms that ConvRotLinear makes of its weight (FP6 operands, the CDNA4 repack of a K x packed-N
weight) follow the weight."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
M, K, N, G = 512, 1024, 768, 64


def packed(seed, dev):
    """(NK-packed codes, scales) of a random weight."""
    from convrot_mlx_amd import quantize_convrot_weight

    gen = torch.Generator(dev).manual_seed(seed)
    return quantize_convrot_weight((torch.randn((N, K), generator=gen, device=dev) * 0.02).to(torch.bfloat16), G)


def layer_of(backend, qw, ws, dev):
    from convrot_mlx_amd import ConvRotLinear

    return ConvRotLinear(K, N, group_size=G, backend=backend, device=dev).load_nk_weight(qw, ws)


@pytest.mark.parametrize("backend", ["hip-w4a4", "mpp-w4a4", "mpp-w4a16"])
def test_weights_assigned_one_after_the_other(dev, backend):
    """A weight whose memory is that of an earlier one, which the layer's kept forms were made of, is another
    weight."""
    x = torch.randn((M, K), generator=torch.Generator(dev).manual_seed(1), device=dev).to(torch.bfloat16)
    states = [packed(seed, dev) for seed in range(4)]
    want = [layer_of(backend, *s, dev)(x) for s in states]
    layer, places = layer_of(backend, *states[0], dev), set()
    for (qw, ws), w in zip(states, want):
        layer.qweight = None
        layer.load_nk_weight(qw, ws)
        places.add(layer.qweight.data_ptr())
        assert torch.equal(layer(x), w)
