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


CYCLES = 100_000_000  # of a spinning kernel: some tens of milliseconds


@pytest.mark.parametrize("backend", ["hip-w4a4", "mpp-w4a4", "mpp-w4a16"])
def test_forms_made_on_another_stream(dev, backend, fp6_form):
    """A form made by a call on one stream is read by a call on another only once it is written."""
    fp6_form("full")
    x = torch.randn((M, K), generator=torch.Generator(dev).manual_seed(1), device=dev).to(torch.bfloat16)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for seed in range(3):
        state = packed(seed, dev)
        want = layer_of(backend, *state, dev)(x)
        layer = layer_of(backend, *state, dev)
        for s in (a, b):  # each stream's workspace
            with torch.cuda.stream(s):
                layer_of(backend, *state, dev)(x)
        with torch.cuda.stream(a):
            for size in (K * N // 2, K * N * 3 // 4):  # what the forms' memory may hold before
                torch.full((size,), 77, dtype=torch.uint8, device=dev)
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            torch.cuda._sleep(CYCLES)
            first = layer(x)
        with torch.cuda.stream(b):
            second = layer(x)
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(second, want)


@pytest.mark.parametrize("backend", ["hip-w4a4", "mpp-w4a4", "mpp-w4a16"])
def test_forms_made_under_capture_are_the_graphs(dev, backend, fp6_form):
    """A layer first called under capture: its forms are written when the graph runs, so an eager call before
    that makes its own."""
    fp6_form("full")
    x = torch.randn((M, K), generator=torch.Generator(dev).manual_seed(1), device=dev).to(torch.bfloat16)
    state = packed(5, dev)
    want = layer_of(backend, *state, dev)(x)
    layer = layer_of(backend, *state, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer_of(backend, *state, dev)(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            static = layer(x)
        eager = layer(x)
        side.synchronize()
        assert torch.equal(eager, want)
        for _ in range(3):
            static.zero_()
            graph.replay()
            side.synchronize()
            assert torch.equal(static, want) and torch.equal(layer(x), want)


def test_copies_of_a_layer(dev):
    import copy
    import pickle

    x = torch.randn((M, K), generator=torch.Generator(dev).manual_seed(1), device=dev).to(torch.bfloat16)
    layer = layer_of("mpp-w4a4", *packed(6, dev), dev)
    want = layer(x)
    for other in (copy.deepcopy(layer), pickle.loads(pickle.dumps(layer))):
        assert torch.equal(other(x), want)


@pytest.mark.parametrize("backend", ["hip-w4a4", "mpp-w4a4", "hip-w4a16", "mpp-w4a16"])
def test_weights_of_inference_mode(dev, backend):
    x = torch.randn((M, K), generator=torch.Generator(dev).manual_seed(1), device=dev).to(torch.bfloat16)
    states = [packed(seed, dev) for seed in (7, 8)]
    want = [layer_of(backend, *s, dev)(x) for s in states]
    with torch.inference_mode():
        layer, other = (layer_of(backend, *s, dev) for s in states)
        assert layer.qweight.is_inference()
        for _ in range(2):
            assert torch.equal(layer(x), want[0])
        layer.qweight.copy_(other.qweight), layer.scales.copy_(other.scales)
        assert torch.equal(layer(x), want[1])
    assert torch.equal(layer(x), want[1])
