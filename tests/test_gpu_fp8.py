"""GPU: linears in 8-bit floating point against their definition in 64 bits (codes and scales exactly)."""

from __future__ import annotations

import pytest
import torch

from tests import _plain_fp8 as plain
from tests._plain64 import U, assert_within

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
FP8 = torch.float8_e4m3fn
TILES = ["256x256", "128x128", "64x128", "64x64", "32x64"]


def normal(seed, *shape, std=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std


def weight(seed, n, k, dev):
    """Codes, and scales that are no powers of two."""
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn((n, k), generator=g) * 60).clamp(-448, 448).to(FP8)
    ws = torch.rand(((n + 127) // 128, (k + 127) // 128), generator=g) * 1e-3 + 1e-5
    return q.to(dev), ws.to(dev)


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double().cpu(), nan=-1e9), torch.nan_to_num(b.double().cpu(), nan=-1e9))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 130), (16, 256), (17, 1000), (33, 4096), (300, 72), (5, 8191)])
def test_quantizer(dev, m, k, dtype):
    from convrot_mlx_amd import quantize_fp8_blockwise

    x = normal(m + k, m, k) * torch.exp(normal(k, m, 1) * 3)
    if m > 4:
        x[1], x[2], x[3, k // 2], x[4, 0] = 0.0, 2.0 ** -120, float("nan"), float("-inf")
    x = x.to(dtype)
    x[0, 0] = x[0].abs().max()
    q, s = plain.codes(x)
    for view in (x.to(dev), x.to(dev).t().contiguous().t(), torch.cat([x, x], 1).to(dev)[:, :k]):
        got, scales = quantize_fp8_blockwise(view)
        assert got.dtype == FP8 and got.shape == x.shape and scales.shape == s.shape
        assert same(got.float(), q) and same(scales, s)


def test_quantizer_borders(dev):
    """Largest magnitudes at and beside 448 times a power of two, ties between codes, the smallest codes."""
    from convrot_mlx_amd import quantize_fp8_blockwise

    rows = []
    for a in (448.0, 448.0 * (1 + 2 ** -23), 448.0 * (1 - 2 ** -24), 447.0, 256.0, 1.75 * 2 ** -90, 2.0 ** -100,
              2.0 ** -100 * (1 - 2 ** -24), 3.0e38, 1.0):
        x = torch.zeros(128, dtype=F32)
        x[0] = a
        x[1:64] = a * torch.arange(1, 64) / 64 * 2.0 ** (-torch.arange(1, 64) // 4)
        x[64:] = a / 448 * (torch.arange(64) - 32) * 2.0 ** -10
        rows.append(x)
    x = torch.stack(rows)
    q, s = plain.codes(x)
    got, scales = quantize_fp8_blockwise(x.to(dev))
    assert same(got.float(), q) and same(scales, s)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 16), (128, 128), (130, 300), (515, 1000), (3, 70, 200)])
def test_weight_quantizer(dev, shape, dtype):
    from convrot_mlx_amd import quantize_fp8_weight

    w = normal(shape[-1], *shape, std=0.02).to(dtype)
    q, s = quantize_fp8_weight(w.to(dev))
    assert q.shape == w.shape and q.dtype == FP8 and q.is_contiguous()
    for one, qe, se in zip(w.reshape(-1, *shape[-2:]), q.reshape(-1, *shape[-2:]), s.reshape(-1, *s.shape[-2:])):
        for i in range(se.shape[0]):
            for j in range(se.shape[1]):
                at = (slice(128 * i, 128 * i + 128), slice(128 * j, 128 * j + 128))
                want, scale = plain.codes(one[at].abs().max().reshape(1, 1))
                assert se[i, j].item() == scale.item()
                v = one[at].double() / scale.item()
                step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
                assert same(qe[at].float(), torch.round(v / step) * step)


SHAPES = [(1, 1, 16), (1, 64, 128), (5, 33, 48), (16, 160, 144), (31, 70, 256), (32, 130, 1024), (33, 64, 2048),
          (65, 128, 128), (77, 300, 528), (130, 300, 1168), (255, 255, 272), (300, 264, 4000), (520, 513, 384),
          (1030, 520, 144)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(dev, m, n, k, dtype):
    from convrot_mlx_amd import hip_fp8_linear, hip_fp8_matmul, quantize_fp8_blockwise

    q, ws = weight(n + k, n, k, dev)
    bias = normal(n, n).to(dev)
    x = normal(m + k, m, k).to(dtype)
    xq, xs = plain.codes(x)
    want, spread = plain.product(plain.row_values(xq, xs).to(dev), plain.weight_values(q, ws), dtype == F32)
    got = hip_fp8_linear(x.to(dev), q, ws, bias)
    assert got.dtype == dtype and got.shape == (m, n)
    spread = spread + U * bias.abs().double()
    assert_within(got, want + bias.double(), spread + U * want.abs())
    codes, scales = quantize_fp8_blockwise(x.to(dev))
    assert torch.equal(hip_fp8_matmul(codes, q, scales, ws, bias, output_dtype=dtype), got)
    assert_within(hip_fp8_matmul(codes, q, scales.contiguous(), ws, output_dtype=dtype), want, spread)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (31, 70, 256), (130, 300, 1168), (520, 513, 384), (300, 264, 4000)])
def test_every_tile(dev, tuning, tile, m, n, k):
    from convrot_mlx_amd import hip_fp8_linear

    tuning.set("fp8_tile", tile)
    q, ws = weight(n + k, n, k, dev)
    bias = normal(n, n).to(dev)
    for dtype in (BF16, F32):
        x, res, gate = (normal(i, *s).to(dtype) for i, s in enumerate(((m, k), (m, n), (1, n))))
        want, spread = plain.product(plain.row_values(*plain.codes(x)).to(dev), plain.weight_values(q, ws), dtype == F32)
        want, spread = want + bias.double(), spread + U * (bias.abs().double() + want.abs())
        assert_within(hip_fp8_linear(x.to(dev), q, ws, bias), want, spread, tile)
        res, gate = res.to(dev), gate.to(dev)
        got = hip_fp8_linear(x.to(dev), q, ws, bias, residual=res, gate=gate)
        full = res.double() + gate.double() * want
        assert_within(got, full, gate.double().abs() * spread + U * ((gate.double() * want).abs() + full.abs()), tile)
        into = res.clone()
        assert hip_fp8_linear(x.to(dev), q, ws, bias, residual=into, gate=gate, inplace=True) is into
        assert torch.equal(into, got)


@pytest.mark.parametrize("split", [2, 3, 7, 64])
@pytest.mark.parametrize("tile,m", [("32x64", 1), ("32x64", 33), ("64x128", 65), ("128x128", 200), ("64x64", 70), ("64x64", 300),
                                    ("256x256", 300)])
def test_shared_k(dev, tuning, tile, m, split):
    """Workgroups that share a tile's K: sums in the parts' order, the same bits launch after launch."""
    from convrot_mlx_amd import hip_fp8_linear

    tuning.set("fp8_tile", tile)
    tuning.set("fp8_split", split)
    n, k = 200, 4112
    q, ws = weight(k, n, k, dev)
    x = normal(m, m, k).to(BF16)
    want, spread = plain.product(plain.row_values(*plain.codes(x)).to(dev), plain.weight_values(q, ws), False)
    first = hip_fp8_linear(x.to(dev), q, ws)
    assert_within(first, want, 2 * spread)
    for _ in range(3):
        assert torch.equal(hip_fp8_linear(x.to(dev), q, ws), first)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("split", [None, 1, 3])
@pytest.mark.parametrize("m,k", [(1, 4096), (1, 16384), (2, 1032), (5, 72), (7, 2304), (16, 512), (16, 1096), (16, 4160)])
def test_few_rows(dev, tuning, m, k, split, dtype):
    """Rows quantized inside the product's launch, in a launch of their own (longer or unaligned rows), and as
    codes: the same bits."""
    from convrot_mlx_amd import hip_fp8_linear, hip_fp8_matmul, quantize_fp8_blockwise

    if split:
        tuning.set("fp8_split", split)
    n = 330
    q, ws = weight(k, n, k, dev)
    bias, x = normal(n, n).to(dev), normal(m, m, k).to(dtype)
    want, spread = plain.product(plain.row_values(*plain.codes(x)).to(dev), plain.weight_values(q, ws), dtype == F32)
    x = x.to(dev)
    got = hip_fp8_linear(x, q, ws, bias)
    # (the parts' sums are added in float32: up to `parts` more roundings)
    assert_within(got, want + bias.double(), 2 * spread + U * (bias.abs().double() + want.abs()))
    codes, scales = quantize_fp8_blockwise(x)
    assert torch.equal(hip_fp8_matmul(codes, q, scales, ws, bias, output_dtype=dtype), got)
    apart = torch.full((m, k + 9), float("nan"), dtype=dtype, device=dev)
    apart[:, 1:k + 1] = x
    assert torch.equal(hip_fp8_linear(apart[:, 1:k + 1], q, ws, bias), got)
    apart = torch.full((2 * m, k), float("nan"), dtype=dtype, device=dev)
    apart[::2] = x
    assert torch.equal(hip_fp8_linear(apart[::2], q, ws, bias), got)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,k", [(40, 72), (330, 1032), (200, 4160), (4096, 512)])
@pytest.mark.parametrize("m", [17, 32, 33, 48, 50, 65, 77, 96])
def test_17_to_96_rows(dev, m, n, k, dtype):
    from convrot_mlx_amd import hip_fp8_linear, hip_fp8_matmul, quantize_fp8_blockwise

    q, ws = weight(k, n, k, dev)
    bias, x, res, gate = normal(n, n).to(dev), normal(m, m, k).to(dtype), normal(2, m, n).to(dtype).to(dev), normal(3, 1, n).to(dtype).to(dev)
    want, spread = plain.product(plain.row_values(*plain.codes(x)).to(dev), plain.weight_values(q, ws), False)
    want, spread = want + bias.double(), spread + U * (bias.abs().double() + want.abs())
    x = x.to(dev)
    got = hip_fp8_linear(x, q, ws, bias)
    assert_within(got, want, spread)
    codes, scales = quantize_fp8_blockwise(x)
    assert torch.equal(hip_fp8_matmul(codes, q, scales.contiguous(), ws, bias, output_dtype=dtype), got)
    full = res.double() + gate.double() * want
    gated = hip_fp8_linear(x, q, ws, bias, residual=res, gate=gate)
    assert_within(gated, full, gate.double().abs() * spread + U * ((gate.double() * want).abs() + full.abs()))
    into = res.clone()
    assert hip_fp8_linear(x, q, ws, bias, residual=into, gate=gate, inplace=True) is into
    assert torch.equal(into, gated)


def test_few_rows_in_place_of_their_residual(dev):
    """A residual that is the input itself, written in place: no workgroup may read what another has written."""
    from convrot_mlx_amd import hip_fp8_linear

    for m in (1, 8):
        q, ws = weight(3, 2048, 2048, dev)
        x = normal(m, m, 2048).to(BF16).to(dev)
        want = hip_fp8_linear(x, q, ws, residual=x)
        for _ in range(3):
            got = x.clone()
            assert hip_fp8_linear(got, q, ws, residual=got, inplace=True) is got
            assert torch.equal(got, want)


@pytest.mark.parametrize("k", [50, 64, 200])
def test_strided_and_unaligned_operands(dev, k):
    from convrot_mlx_amd import hip_fp8_matmul

    m, n = 20, 40
    q, ws = weight(k, n, k, dev)
    a = (normal(1, m, k) * 60).clamp(-448, 448).to(FP8).to(dev)
    xs = (torch.rand((m, (k + 127) // 128), generator=torch.Generator().manual_seed(3)) + 0.1).to(dev)
    want = hip_fp8_matmul(a, q, xs, ws, output_dtype=F32)
    ref, spread = plain.product(plain.row_values(a, xs), plain.weight_values(q, ws), True)
    assert_within(want, ref, spread)
    wide = lambda t, by: torch.cat([t.view(torch.uint8), torch.full((t.shape[0], by), 0x7f, dtype=torch.uint8, device=dev)], 1).view(FP8)[:, :k]  # noqa: E731
    for by in (16, 7, 48 - k % 16):
        assert torch.equal(hip_fp8_matmul(wide(a, by), wide(q, by), xs, ws, output_dtype=F32), want)
    flip = lambda t: t.view(torch.uint8).t().contiguous().t().view(FP8)  # noqa: E731
    assert torch.equal(hip_fp8_matmul(flip(a), flip(q), xs.t().contiguous().t(), ws.t().contiguous().t(), output_dtype=F32), want)
    one = xs[:1].expand(m, -1)
    assert torch.equal(hip_fp8_matmul(a, q, one, ws, output_dtype=F32),
                       hip_fp8_matmul(a, q, one.contiguous(), ws, output_dtype=F32))


def test_not_finite(dev):
    """A NaN or an infinity reaches the rows of its block alone; a NaN code its row (or its output)."""
    from convrot_mlx_amd import hip_fp8_linear, hip_fp8_matmul, quantize_fp8_blockwise

    q, ws = weight(5, 70, 300, dev)
    x = normal(4, 40, 300).to(BF16).to(dev)
    clean = hip_fp8_linear(x, q, ws)
    x[3, 290], x[7, 0] = float("nan"), float("inf")
    for dtype in (BF16, F32):
        got = hip_fp8_linear(x.to(dtype), q, ws)
        rows = got.isnan().all(1)
        assert rows[[3, 7]].all() and rows.sum() == 2
        assert torch.isfinite(got[~rows]).all()
    keep = [r for r in range(40) if r not in (3, 7)]
    assert torch.equal(hip_fp8_linear(x, q, ws)[keep], clean[keep])
    codes, xs = quantize_fp8_blockwise(normal(4, 40, 300).to(BF16).to(dev))
    bad = q.view(torch.uint8).clone()
    bad[11, 17] = 0x7f
    for dtype in (BF16, F32):
        got = hip_fp8_matmul(codes, bad.view(FP8), xs, ws, output_dtype=dtype)
        assert got[:, 11].isnan().all() and got.isnan().sum() == 40


@pytest.mark.parametrize("m,n", [(0, 16), (4, 0), (0, 0)])
def test_nothing_to_do(dev, m, n):
    from convrot_mlx_amd import hip_fp8_linear, quantize_fp8_blockwise

    q, ws = torch.zeros((n, 32), device=dev).to(FP8), torch.zeros(((n + 127) // 128, 1), device=dev)
    assert hip_fp8_linear(torch.zeros((m, 32), device=dev, dtype=BF16), q, ws).shape == (m, n)
    codes, scales = quantize_fp8_blockwise(torch.zeros((m, 0), device=dev))
    assert codes.shape == (m, 0) and scales.shape == (m, 0)


def test_offsets_past_32_bits(dev):
    """Rows whose codes and outputs lie past 4 GiB."""
    from convrot_mlx_amd import hip_fp8_linear

    k, n, m = 4096, 32, (1 << 20) + 70
    q, ws = weight(1, n, k, dev)
    x = torch.zeros((m, k), dtype=BF16, device=dev)
    rows = [0, 1, 70, m // 2, (1 << 20) - 1, 1 << 20, m - 1]
    some = normal(2, len(rows), k).to(BF16)
    x[rows] = some.to(dev)
    got = hip_fp8_linear(x, q, ws)
    want, spread = plain.product(plain.row_values(*plain.codes(some)).to(dev), plain.weight_values(q, ws), False)
    assert_within(got[rows], want, spread)
    got[rows] = 0
    assert not got.any()


def test_graphs_and_streams(dev):
    """Captured calls hold their own codes, counters and partial sums: replays beside eager calls, other
    graphs and another stream give the eager bits."""
    from convrot_mlx_amd import hip_fp8_linear

    cases = []
    for m, n, k in ((1, 512, 8192), (24, 512, 8192), (300, 700, 2000)):
        q, ws = weight(m, n, k, dev)
        cases.append((normal(m, m, k).to(BF16).to(dev), q, ws))
    want = [hip_fp8_linear(*c) for c in cases]
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = hip_fp8_linear(*c)
        graphs.append((g, out))
    side = torch.cuda.Stream()
    for _ in range(4):
        for (g, out), c, w in zip(graphs, cases, want):
            out.zero_()
            g.replay()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                other = hip_fp8_linear(*c)
            assert torch.equal(hip_fp8_linear(*c), w)
            torch.cuda.synchronize()
            assert torch.equal(out, w) and torch.equal(other, w)


def test_layer(dev):
    from convrot_mlx_amd import Fp8Linear, hip_fp8_linear, hip_layer_norm, replace_fp8_linears

    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(300, 200), torch.nn.GELU(), torch.nn.Linear(200, 150, bias=False)).to(dev)
    dense = [m.weight.detach().clone() for m in (model[0], model[2])]
    assert replace_fp8_linears(model, select=lambda name, m: name == "0") == ["0"]
    assert replace_fp8_linears(model) == ["2"] and isinstance(model[2], Fp8Linear)
    layer = model[0]
    values = plain.weight_values(layer.qweight, layer.scales)
    assert ((values - dense[0].double()).abs() <= dense[0].abs().double() * 2.0 ** -4 + 2.0 ** -10 * layer.scales.max().double()).all()
    x = normal(9, 2, 7, 300).to(BF16).to(dev)
    y = layer(x)
    assert y.shape == (2, 7, 200) and torch.equal(y.reshape(14, 200), hip_fp8_linear(x.reshape(14, 300), layer.qweight, layer.scales, layer.bias))
    moved = torch.nn.Sequential(layer).to(BF16)[0]
    assert moved.qweight.dtype == FP8 and moved.scales.dtype == F32 and moved.bias.dtype == F32
    assert torch.equal(moved(x), y)
    other = Fp8Linear(300, 200, device=dev)
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), y)
    shift, scale = (normal(i, 2, 1, 300).to(BF16).to(dev) for i in (1, 2))
    res, gate = normal(3, 2, 7, 200).to(BF16).to(dev), normal(4, 2, 1, 200).to(BF16).to(dev)
    got = layer.forward_modulated(x, shift, scale, residual=res, gate=gate)
    assert torch.equal(got, layer(hip_layer_norm(x, scale=scale, shift=shift), residual=res, gate=gate))
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="has no gradient"):
        layer(x).sum().backward()
    with torch.inference_mode():
        assert torch.equal(model(x[0]), model(x)[0])
