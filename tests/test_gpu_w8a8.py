"""GPU: 8-bit linears, bit for bit against the definition (exact integer sums, the epilogue and the
quantizer as the same sequence of float32 operations in numpy)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def quantize_plain(x: torch.Tensor):
    v = x.float().cpu().numpy()
    a = np.abs(v).max(axis=1, initial=0.0)
    zero = a < np.float32(2.0 ** -100)
    inv = np.where(zero, np.float32(0), np.float32(127) / np.where(zero, np.float32(1), a)).astype(np.float32)
    codes = np.rint(v * inv[:, None]).astype(np.int8)
    return codes, np.where(zero, np.float32(0), a * np.float32(1.0 / 127.0)).astype(np.float32)


def product_plain(qa, qw, xs, ws, bias, dtype):
    dot = qa.astype(np.float64) @ qw.astype(np.float64).T  # exact: below 2^53
    v = dot.astype(np.float32) * xs[:, None]
    v = v * ws[None]
    if bias is not None:
        v = v + bias[None]
    return torch.from_numpy(v).to(dtype)


def operands(seed, m, n, k, dev):
    g = np.random.default_rng(seed)
    qa = g.integers(-127, 128, (m, k), dtype=np.int8)
    qw = g.integers(-128, 128, (n, k), dtype=np.int8)
    xs, ws = (g.uniform(0.001, 0.02, s).astype(np.float32) for s in (m, n))
    bias = g.normal(size=n).astype(np.float32)
    return (qa, qw, xs, ws, bias), tuple(torch.from_numpy(t).to(dev) for t in (qa, qw, xs, ws, bias))


SHAPES = [
    (1, 64, 64), (1, 1, 16), (1, 1000, 4096), (3, 33, 48), (5, 16, 32), (16, 160, 144), (17, 48, 400), (32, 130, 1024),
    (33, 64, 2048), (64, 96, 640), (65, 128, 128), (77, 300, 528), (128, 128, 256), (200, 515, 1040), (255, 255, 272),
    (512, 512, 512), (513, 700, 384), (600, 1000, 2064), (1030, 520, 144), (700, 2685, 896),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(dev, m, n, k, dtype):
    from convrot_mlx_amd import hip_w8a8_matmul

    host, (qa, qw, xs, ws, bias) = operands(m + n + k, m, n, k, dev)
    got = hip_w8a8_matmul(qa, qw, xs, ws, bias, output_dtype=dtype)
    assert torch.equal(got.cpu(), product_plain(*host, dtype))
    got = hip_w8a8_matmul(qa, qw, xs, ws, output_dtype=dtype)
    assert torch.equal(got.cpu(), product_plain(*host[:4], None, dtype))


TILES = ["256x256", "256x224", "224x256", "256x192", "192x256", "256x128", "128x256", "192x192", "192x128", "128x192",
         "160x128", "128x160", "128x128", "128x64", "64x128", "64x64"]


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (31, 70, 256), (130, 300, 1168), (520, 513, 384), (300, 264, 4000)])
def test_every_kernel(dev, tuning, tile, m, n, k):
    from convrot_mlx_amd import hip_w8a8_matmul

    tuning.set("w8a8_tile", tile)
    for dtype in (BF16, F32):
        host, (qa, qw, xs, ws, bias) = operands(m + k, m, n, k, dev)
        assert torch.equal(hip_w8a8_matmul(qa, qw, xs, ws, bias, output_dtype=dtype).cpu(), product_plain(*host, dtype))


@pytest.mark.parametrize("split", [2, 3, 7, 64])
@pytest.mark.parametrize("tile,m", [(None, 1), (None, 16), ("64x64", 70), ("128x64", 200), ("64x128", 65), ("128x128", 300)])
def test_shared_k(dev, tuning, tile, m, split):
    """Workgroups that share a tile's K add integer sums: the same bits, launch after launch."""
    from convrot_mlx_amd import hip_w8a8_matmul

    tuning.set("w8a8_tile", tile)
    tuning.set("w8a8_split", split)
    for n, k in ((70, 1000), (200, 4112)):
        k16 = k - k % 16
        host, (qa, qw, xs, ws, bias) = operands(m + k, m, n, k16, dev)
        want = product_plain(*host, BF16)
        for _ in range(3):
            assert torch.equal(hip_w8a8_matmul(qa, qw, xs, ws, bias, output_dtype=BF16).cpu(), want)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k", [(1, 16), (1, 3072), (1, 12288), (1, 24576), (2, 4112), (3, 128), (7, 1040), (8, 3072),
                                 (16, 1536), (16, 1600), (5, 6144)])
def test_few_rows_quantized_in_the_launch(dev, m, k, dtype):
    from convrot_mlx_amd import hip_w8a8_linear, hip_w8a8_matmul, quantize_int8_rowwise

    n = 150
    host, (_, qw, _, ws, bias) = operands(m + k, m, n, k, dev)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)) * 2
    if m > 2:
        x[1], x[2, k // 2] = 0.0, float("nan")
    x = x.to(dtype).to(dev)
    got = hip_w8a8_linear(x, qw, ws, bias)
    codes, scales = quantize_int8_rowwise(x)
    want = hip_w8a8_matmul(codes, qw, scales, ws, bias, output_dtype=dtype)
    assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(want, nan=7.0))
    clean = [r for r in range(m) if not (m > 2 and r == 2)]
    plain = product_plain(codes.cpu().numpy(), host[1], scales.cpu().numpy(), *host[3:], dtype)
    assert torch.equal(got.cpu()[clean], plain[clean])
    if m > 2:
        assert got[2].isnan().all()


@pytest.mark.parametrize("m,k", [(20, 64), (70, 2000), (300, 528), (40, 12288), (5000, 4096)])
def test_codes_in_the_workspace_or_apart(dev, m, k):
    """The codes between the two launches lie at the end of the stream's workspace where they are at
    most a quarter of it, beside partial sums (40 rows of 12288) or not, else in memory of their own."""
    from convrot_mlx_amd import core, hip_w8a8_linear

    host, (_, qw, _, ws, bias) = operands(m, m, 96, k, dev)
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)).to(BF16)
    codes, scales = quantize_plain(x)
    want = product_plain(codes, host[1], scales, *host[3:], BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            for _ in range(2):
                assert torch.equal(hip_w8a8_linear(x.to(dev), qw, ws, bias).cpu(), want)
    assert (dev.index or 0, side.cuda_stream) in core._WORKSPACES


def test_few_rows_in_place_over_their_input(dev):
    """x as its own residual: every workgroup reads all of x, so the rows are quantized first."""
    from convrot_mlx_amd import hip_w8a8_linear

    _, (_, qw, _, ws, bias) = operands(3, 4, 256, 256, dev)
    x = torch.randn((4, 256), generator=torch.Generator().manual_seed(3)).to(BF16).to(dev)
    want = hip_w8a8_linear(x, qw, ws, bias, residual=x.clone())
    got = hip_w8a8_linear(x, qw, ws, bias, residual=x, inplace=True)
    assert got.data_ptr() == x.data_ptr() and torch.equal(x, want)


@pytest.mark.parametrize("k", [1, 5, 15, 17, 100, 127, 129, 1001])
@pytest.mark.parametrize("m,n", [(1, 5), (40, 37), (300, 150)])
def test_any_features(dev, m, n, k):
    """K that fills no 16 bytes: operands are padded, through the functions and through the layer."""
    from convrot_mlx_amd import Int8Linear, hip_w8a8_linear, hip_w8a8_matmul

    host, (qa, qw, xs, ws, bias) = operands(k, m, n, k, dev)
    assert torch.equal(hip_w8a8_matmul(qa, qw, xs, ws, bias, output_dtype=F32).cpu(), product_plain(*host, F32))
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)).to(BF16)
    codes, scales = quantize_plain(x)
    want = product_plain(codes, host[1], scales, *host[3:], BF16)
    assert torch.equal(hip_w8a8_linear(x.to(dev), qw, ws, bias).cpu(), want)
    layer = Int8Linear(k, n, device=dev)
    layer.qweight, layer.scales, layer.bias = qw, ws, bias
    assert torch.equal(layer(x.to(dev)).cpu(), want)
    assert torch.equal(layer(x.to(dev)).cpu(), want)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 16), (3, 40), (5, 130), (4, 512), (2, 1000), (3, 1024), (2, 2056), (2, 3072),
                                 (2, 5120), (1, 7777), (2, 8192), (2, 10001), (1, 15360), (1, 33000), (1, 65536)])
def test_quantizer(dev, m, k, dtype):
    from convrot_mlx_amd import quantize_int8_rowwise

    x = torch.randn((m, k), generator=torch.Generator().manual_seed(k)) * 3
    x[:, : max(1, k // 200)] *= 20
    x = x.to(dtype)
    codes, scales = quantize_int8_rowwise(x.to(dev))
    want, wscales = quantize_plain(x)
    assert np.array_equal(codes.cpu().numpy(), want) and np.array_equal(scales.cpu().numpy(), wscales)


def test_quantizer_of_views_and_odd_rows(dev):
    from convrot_mlx_amd import hip_w8a8_linear, quantize_int8_rowwise

    base = torch.randn((9, 300), generator=torch.Generator().manual_seed(3))
    for view in (base[:, 8:264], base[:, 1:129], base[::2, :256], base.t()[:, :8], base[:1].expand(4, 300)):
        codes, scales = quantize_int8_rowwise(view.to(BF16).to(dev) if view.stride(0) else view.to(dev))
        want, wscales = quantize_plain(view.to(BF16) if view.stride(0) else view)
        assert np.array_equal(codes.cpu().numpy(), want) and np.array_equal(scales.cpu().numpy(), wscales)
    dbase = base.to(BF16).to(dev)
    codes, _ = quantize_int8_rowwise(dbase[:, 3:259])
    assert np.array_equal(codes.cpu().numpy(), quantize_plain(base.to(BF16)[:, 3:259])[0])
    x = torch.zeros((6, 64))
    x[1, 3], x[2, 9], x[3, 5], x[4] = float("nan"), float("inf"), -float("inf"), 2.0 ** -110
    x[5, 0], x[5, 1] = 3e38, -1.0
    codes, scales = quantize_int8_rowwise(x.to(dev))
    assert not codes[:5].any() and scales[0] == 0 and scales[4] == 0 and scales[1:4].isnan().all()
    assert codes[5, 0] == 127 and scales[5].isfinite()
    w = torch.ones((8, 64), dtype=torch.int8, device=dev)
    out = hip_w8a8_linear(x.to(dev), w, torch.ones(8, device=dev), torch.full((8,), 0.5, device=dev))
    assert out[1:4].isnan().all() and (out[[0, 4]] == 0.5).all() and out[5].isfinite().all()
    codes, scales = quantize_int8_rowwise(x[:0].to(dev))
    assert codes.shape == (0, 64) and scales.shape == (0,)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n", [(1, 64), (6, 50), (40, 136), (300, 264), (520, 515), (528, 1024)])
def test_gated_residual(dev, m, n, dtype):
    """residual + gate * linear in float32, rounded once, out of place and in place."""
    from convrot_mlx_amd import hip_w8a8_matmul

    host, (qa, qw, xs, ws, bias) = operands(m + n, m, n, 192, dev)
    lin = product_plain(*host, F32)
    g = torch.Generator().manual_seed(n)
    res = torch.randn((m, n), generator=g).to(dtype)
    for gate in (None, torch.randn((1, n), generator=g).to(dtype), torch.randn((m, n), generator=g).to(dtype)):
        want = (res.float() + lin if gate is None else res.float() + gate.float() * lin).to(dtype)
        r, gd = res.to(dev), None if gate is None else gate.to(dev)
        got = hip_w8a8_matmul(qa, qw, xs, ws, bias, output_dtype=dtype, residual=r, gate=gd)
        assert torch.equal(got.cpu(), want)
        got = hip_w8a8_matmul(qa, qw, xs, ws, bias, output_dtype=dtype, residual=r, gate=gd, inplace=True)
        assert got.data_ptr() == r.data_ptr() and torch.equal(r.cpu(), want)
    if m % 2 == 0:
        gate = torch.randn((2, 1, n), generator=g).to(dtype)
        want = (res.float().reshape(2, m // 2, n) + gate.float() * lin.reshape(2, m // 2, n)).to(dtype)
        got = hip_w8a8_matmul(qa, qw, xs, ws, bias, output_dtype=dtype, residual=res.reshape(2, m // 2, n).to(dev),
                              gate=gate.to(dev))
        assert torch.equal(got.cpu(), want.reshape(m, n))


def test_strided_operands(dev):
    """Row-strided codes and weights are read in place; the last row of a view may end its memory."""
    from convrot_mlx_amd import hip_w8a8_matmul

    host, (qa, qw, xs, ws, bias) = operands(1, 90, 70, 320, dev)
    want = product_plain(*host, BF16)
    big = torch.full((90, 512), 99, dtype=torch.int8, device=dev)
    bigw = torch.full((70, 400), -77, dtype=torch.int8, device=dev)
    big[:, 192:], bigw[:, 80:] = qa, qw
    assert torch.equal(hip_w8a8_matmul(big[:, 192:], bigw[:, 80:], xs, ws, bias, output_dtype=BF16).cpu(), want)
    odd = torch.empty((90, 327), dtype=torch.int8, device=dev)
    odd[:, 7:] = qa
    assert torch.equal(hip_w8a8_matmul(odd[:, 7:], qw, xs, ws, bias, output_dtype=BF16).cpu(), want)
    t = qw.t().contiguous().t()
    assert torch.equal(hip_w8a8_matmul(qa, t, xs, ws, bias, output_dtype=BF16).cpu(), want)


def test_layer(dev):
    """Int8Linear: a dense weight quantized row by row, leading shapes, the fused modulated norm."""
    from convrot_mlx_amd import Int8Linear, hip_layer_norm, quantize_int8_rowwise

    g = torch.Generator().manual_seed(4)
    w, b = (torch.randn((150, 256), generator=g) * 0.05).to(BF16), torch.randn(150, generator=g)
    layer = Int8Linear(256, 150, device=dev).load_weight(w.to(dev), b.to(dev))
    qw, ws = quantize_plain(w)
    assert np.array_equal(layer.qweight.cpu().numpy(), qw)
    x = torch.randn((2, 7, 256), generator=g).to(BF16)
    codes, xs = quantize_plain(x.reshape(14, 256))
    lin = product_plain(codes, qw, xs, ws, b.numpy(), F32).reshape(2, 7, 150)
    want = lin.to(BF16)
    y = layer(x.to(dev))
    assert torch.equal(y.cpu(), want)
    res, gate = torch.randn((2, 7, 150), generator=g).to(BF16), torch.randn((2, 1, 150), generator=g).to(BF16)
    gated = (res.float() + gate.float() * lin).to(BF16)
    assert torch.equal(layer(x.to(dev), residual=res.to(dev), gate=gate.to(dev)).cpu(), gated)
    assert layer(x[:0].to(dev)).shape == (0, 7, 150)
    # the norm's result goes to codes from float32: the product of those codes, which are the
    # quantizer's of the same norm in float32
    shift, scale = (torch.randn((2, 1, 256), generator=g).to(BF16).to(dev) * 0.3 for _ in range(2))
    n32 = hip_layer_norm(x.float().to(dev), scale=scale.float(), shift=shift.float(), eps=1e-6)
    c32, s32 = quantize_int8_rowwise(n32.reshape(14, 256))
    lin = product_plain(c32.cpu().numpy(), qw, s32.cpu().numpy(), ws, b.numpy(), F32).reshape(2, 7, 150)
    assert torch.equal(layer.forward_modulated(x.to(dev), shift, scale, eps=1e-6).cpu(), lin.to(BF16))
    got = layer.forward_modulated(x.to(dev), shift, scale, residual=res.to(dev), gate=gate.to(dev))
    assert torch.equal(got.cpu(), (res.float() + gate.float() * lin).to(BF16))


def test_layer_follows_its_weight(dev):
    """A layer whose rows need padding reads the weight it has now: assigned anew (its memory may be
    the old one's), or changed in place."""
    from convrot_mlx_amd import Int8Linear, hip_w8a8_linear

    g = torch.Generator().manual_seed(5)
    layer = Int8Linear(50, 40, device=dev)
    x = torch.randn((3, 50), generator=g).to(BF16).to(dev)
    for seed in range(4):
        layer.qweight = None
        layer.qweight = torch.randint(-127, 128, (40, 50), generator=g, dtype=torch.int8).to(dev)
        assert torch.equal(layer(x), hip_w8a8_linear(x, layer.qweight, layer.scales, layer.bias))
        layer.qweight.neg_()
        assert torch.equal(layer(x), hip_w8a8_linear(x, layer.qweight, layer.scales, layer.bias))


def test_replace_int8_linears(dev):
    from torch import nn

    from convrot_mlx_amd import ConvRotLinear, Int8Linear, replace_convrot_linears, replace_int8_linears

    model = nn.Sequential(nn.Linear(50, 256), nn.GELU(), nn.Linear(256, 256), nn.Linear(256, 30, bias=False)).to(dev)
    dense = [m.weight.detach().clone() for m in model if isinstance(m, nn.Linear)]
    assert replace_int8_linears(model, select=lambda name, m: name != "2") == ["0", "3"]
    assert replace_convrot_linears(model) == ["2"]
    assert isinstance(model[0], Int8Linear) and isinstance(model[2], ConvRotLinear) and isinstance(model[3], Int8Linear)
    x = torch.randn((5, 50), generator=torch.Generator().manual_seed(2)).to(dev)
    # symmetric 8-bit rows: a product is off by at most half a step of each operand
    want = torch.nn.functional.linear(x, dense[0], model[0].bias)
    step = (x.abs().amax(1, keepdim=True) / 254) @ dense[0].abs().sum(1)[None] + \
        x.abs().sum(1, keepdim=True) @ (dense[0].abs().amax(1)[None] / 254)
    assert ((model[0](x) - want).abs() <= 1.01 * step).all()
    assert model(x).shape == (5, 30)


def test_side_stream_and_graph_replays(dev):
    from convrot_mlx_amd import hip_w8a8_linear

    for m in (3, 100, 600):
        _, (_, qw, _, ws, bias) = operands(m, 1, 520, 256, dev)
        x = torch.randn((m, 256), generator=torch.Generator().manual_seed(m)).to(BF16).to(dev)
        side = torch.cuda.Stream()
        eager = hip_w8a8_linear(x, qw, ws, bias).clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = hip_w8a8_linear(x, qw, ws, bias)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                static = hip_w8a8_linear(x, qw, ws, bias)
        side.synchronize()
        assert torch.equal(eager, other)
        for i in range(3):
            x.mul_(-1.5)
            want = hip_w8a8_linear(x, qw, ws, bias).clone()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(static, want)


def test_refusals(dev):
    from convrot_mlx_amd import Int8Linear, hip_w8a8_linear, hip_w8a8_matmul, quantize_int8_rowwise

    _, (qa, qw, xs, ws, bias) = operands(1, 4, 6, 64, dev)
    with pytest.raises(ValueError, match="activation must be 2D int8"):
        hip_w8a8_matmul(qa.float(), qw, xs, ws, output_dtype=BF16)
    with pytest.raises(ValueError, match="weight must be 2D int8"):
        hip_w8a8_matmul(qa, qw.to(torch.uint8), xs, ws, output_dtype=BF16)
    with pytest.raises(ValueError, match="N x K with K=64"):
        hip_w8a8_matmul(qa, qw[:, :48], xs, ws, output_dtype=BF16)
    with pytest.raises(ValueError, match="activation scales must have shape"):
        hip_w8a8_matmul(qa, qw, xs[:3], ws, output_dtype=BF16)
    with pytest.raises(ValueError, match="weight scales must have shape"):
        hip_w8a8_matmul(qa, qw, xs, ws[:3], output_dtype=BF16)
    with pytest.raises(ValueError, match="bias must have shape"):
        hip_w8a8_matmul(qa, qw, xs, ws, bias[:2], output_dtype=BF16)
    with pytest.raises(ValueError, match="unsupported dtype"):
        hip_w8a8_matmul(qa, qw, xs, ws, output_dtype=torch.int32)
    with pytest.raises(ValueError, match="gate and inplace need a residual"):
        hip_w8a8_matmul(qa, qw, xs, ws, output_dtype=BF16, gate=bias)
    with pytest.raises(ValueError, match="must hold the"):
        hip_w8a8_matmul(qa, qw, xs, ws, output_dtype=BF16, residual=torch.zeros((3, 6), dtype=BF16, device=dev))
    with pytest.raises(ValueError, match="1 to 65536 features"):
        hip_w8a8_matmul(qa[:, :0], qw[:, :0], xs, ws, output_dtype=BF16)
    with pytest.raises(ValueError, match="2D input"):
        quantize_int8_rowwise(bias)
    with pytest.raises(ValueError, match="unsupported dtype"):
        hip_w8a8_linear(qa, qw, ws)
    with pytest.raises(RuntimeError, match="ROCm device"):
        hip_w8a8_linear(torch.zeros(2, 64), qw.cpu(), ws.cpu())
    with pytest.raises(ValueError, match="expected K=64"):
        Int8Linear(64, 6, device=dev)(torch.zeros((2, 32), device=dev))
    with pytest.raises(ValueError, match="output shape"):
        Int8Linear(64, 6, device=dev)(torch.zeros((2, 64), device=dev), residual=torch.zeros((1, 2, 6), device=dev))
    assert hip_w8a8_matmul(qa[:0], qw, xs[:0], ws, output_dtype=BF16).shape == (0, 6)
    assert hip_w8a8_matmul(qa, qw[:0], xs, ws[:0], output_dtype=BF16).shape == (4, 0)
