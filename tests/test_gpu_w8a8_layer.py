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


CYCLES = 100_000_000  # of a spinning kernel: some tens of milliseconds


def test_padded_weight_on_two_streams(dev):
    """The copy with padded rows is written on the first caller's stream; a call on another stream, which
    that caller has not been ordered before, waits for it."""
    for seed in range(3):
        layer, x, want = layer_and_rows(seed, 250, 96, 40, dev)
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        for s in (a, b):  # workspaces, and kernels loaded
            with torch.cuda.stream(s):
                layer_and_rows(9, 256, 96, 40, dev)[0](torch.zeros((40, 256), dtype=BF16, device=dev))
        with torch.cuda.stream(a):
            torch.full((96, 256), 77, dtype=torch.int8, device=dev)  # what the copy's memory may hold before
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            torch.cuda._sleep(CYCLES)
            first = layer(x)
        with torch.cuda.stream(b):
            second = layer(x)
        torch.cuda.synchronize()
        assert torch.equal(first.cpu(), want) and torch.equal(second.cpu(), want)


def test_replaced_copy_is_kept_for_its_readers(dev):
    """A weight changed in place gets a new copy; the old one's memory stays until a delayed call on
    another stream has read it."""
    layer, x, want = layer_and_rows(5, 250, 96, 40, dev)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        layer(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(b):
        torch.cuda._sleep(CYCLES)
        late = layer(x)
    with torch.cuda.stream(a):
        layer.qweight.neg_()
        layer(x)
        spoil = [torch.full((96, 256), 77, dtype=torch.int8, device=dev) for _ in range(8)]
    torch.cuda.synchronize()
    assert len(spoil) == 8 and torch.equal(late.cpu(), want)


def test_captured_layer_follows_its_weight(dev):
    layer, x, want = layer_and_rows(6, 250, 96, 40, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            static = layer(x)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(static, layer(x))
        if i == 0:
            assert torch.equal(static.cpu(), want)
        layer.qweight.neg_()  # seen by the next replay and the next eager call
        torch.cuda.synchronize()


@pytest.mark.parametrize("k", [16, 64, 1040, 50])
def test_single_rows_at_any_stride(dev, k):
    """A single row of codes, or the weight of a single output: the stride of its row says nothing."""
    from convrot_mlx_amd import hip_w8a8_linear, hip_w8a8_matmul

    host, (qa, qw, xs, ws, bias) = operands(k, 1, 1, k, dev)
    want = product_plain(*host, torch.float32)

    def forms(t):
        wide = torch.full((2, k + 5), 99, dtype=torch.int8, device=dev)
        wide[0, :k] = t[0]
        yield wide[:1, :k]  # the next row k + 5 bytes on
        yield t.t().contiguous().t()  # [k, 1] turned: a stride of one
        yield wide.flatten().as_strided((1, k), (7, 1))

    for a in forms(qa):
        for w in forms(qw):
            assert torch.equal(hip_w8a8_matmul(a, w, xs, ws, bias, output_dtype=torch.float32).cpu(), want)
    x = torch.randn((3, k), generator=torch.Generator().manual_seed(k)).to(BF16)
    codes, scales = quantize_plain(x)
    for w in forms(qw):
        assert torch.equal(hip_w8a8_linear(x.to(dev), w, ws, bias).cpu(), product_plain(codes, host[1], scales, *host[3:],
                                                                                      BF16))


def test_rows_too_far_apart_are_copied(dev):
    from convrot_mlx_amd import hip_w8a8_matmul

    host, (qa, qw, xs, ws, bias) = operands(3, 2, 2, 64, dev)
    far = torch.zeros(((1 << 22) + 16 + 64,), dtype=torch.int8, device=dev).as_strided((2, 64), ((1 << 22) + 16, 1))
    for codes, swap in ((qa, False), (qw, True)):
        far.copy_(codes)
        got = hip_w8a8_matmul(*((qa, far) if swap else (far, qw)), xs, ws, bias, output_dtype=BF16)
        assert torch.equal(got.cpu(), product_plain(*host, BF16))


SHARED = [(24, 1024, 12288), (4, 1024, 12288), (1, 512, 8192)]  # tiles and few rows whose workgroups share K


@pytest.mark.parametrize("m,n,k", SHARED)
def test_graphs_with_shared_k_side_by_side(dev, m, n, k):
    """Two graphs captured on one stream, replayed on two others beside eager calls on it: each product has
    counters and partial sums of its own."""
    from convrot_mlx_amd import _native, hip_w8a8_linear, hip_w8a8_matmul, quantize_int8_rowwise

    assert _native.load().convrot_w8a8_workspace_bytes(m, n, k) > 32768
    _, (_, qw, _, ws, bias) = operands(m, 1, n, k, dev)
    xs = [torch.randn((m, k), generator=torch.Generator().manual_seed(i)).to(BF16).to(dev) for i in range(3)]
    want = [hip_w8a8_linear(x, qw, ws, bias).clone() for x in xs]
    capture, others = torch.cuda.Stream(), [torch.cuda.Stream(), torch.cuda.Stream()]
    capture.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(capture):
        hip_w8a8_linear(xs[0], qw, ws, bias)  # the stream has a workspace
        for x in xs[:2]:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=capture):
                codes, scales = quantize_int8_rowwise(x)
                outs.append([o for _ in range(8) for o in (
                    hip_w8a8_linear(x, qw, ws, bias),
                    hip_w8a8_matmul(codes, qw, scales, ws, bias, output_dtype=BF16))])
            graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(5):
        for out in outs:
            for o in out:
                o.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, others):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(capture):
            eager = [hip_w8a8_linear(xs[2], qw, ws, bias) for _ in range(16)]
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert all(torch.equal(o, w) for o in out)
        assert all(torch.equal(o, want[2]) for o in eager)


@pytest.mark.parametrize("split", [2, 3, 7, 64])
@pytest.mark.parametrize("tile,m", [("160x128", 200), ("128x160", 150)])
def test_shared_k_of_the_largest_tiles(dev, tuning, tile, m, split):
    from convrot_mlx_amd import hip_w8a8_matmul

    tuning.set("w8a8_tile", tile)
    tuning.set("w8a8_split", split)
    for n, k in ((70, 992), (200, 4112)):
        host, (qa, qw, xs, ws, bias) = operands(m + k, m, n, k, dev)
        want = product_plain(*host, BF16)
        for _ in range(3):
            assert torch.equal(hip_w8a8_matmul(qa, qw, xs, ws, bias, output_dtype=BF16).cpu(), want)


@pytest.mark.parametrize("inplace", [False, True])
def test_no_gradient_is_lost_in_silence(dev, inplace):
    """A layer between trained ones keeps its result in grad mode, and the backward pass that reaches it raises."""
    layer, x, _ = layer_and_rows(8, 64, 24, 5, dev)
    res = torch.randn((5, 24), generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    shift = torch.zeros(64, dtype=BF16, device=dev)
    for call in (lambda t, **kw: layer(t, **kw), lambda t, **kw: layer.forward_modulated(t, shift, shift, **kw)):
        with torch.no_grad():
            want = call(x, residual=res)
        leaf = x.clone().requires_grad_()
        target = res.clone()
        got = call(leaf * 1, residual=target, inplace=inplace)
        assert torch.equal(got, want) and (got is target) == inplace
        with pytest.raises(RuntimeError, match="Int8Linear has no gradient"):
            got.sum().backward()
        assert leaf.grad is None
