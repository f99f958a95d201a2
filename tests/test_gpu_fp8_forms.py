"""GPU: the forms of the 8-bit floating point and grouped products' kernels that need many tiles, a forced split, or rows
that are copied: whole large tiles of every output type, shared K with every epilogue, gathered rows."""

from __future__ import annotations

import pytest
import torch

from tests import _plain_fp8 as plain
from tests._plain64 import U, assert_within
from tests.test_gpu_experts import check_products, choose, fp8_weight, normal, product16
from tests.test_gpu_fp8 import weight

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def wanted(x, q, ws, bias, dev):
    want, spread = plain.product(plain.row_values(*plain.codes(x)).to(dev), plain.weight_values(q, ws), x.dtype == F32)
    return want + bias.double(), spread + U * (bias.abs().double() + want.abs())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", [(2900, 2820, 272), (5004, 3900, 144)])
def test_whole_large_tiles(dev, tuning, m, n, k, dtype):
    """144 tiles of 256 x 256 in one round, and 320: a whole round and quarters.  Gates of one vector, and of vectors
    that change inside a tile."""
    from convrot_mlx_amd import hip_fp8_linear

    tuning.set("fp8_tile", "256x256")
    q, ws = weight(n + k, n, k, dev)
    bias, x = normal(n, n).to(dev), normal(1, m, k).to(dtype)
    want, spread = wanted(x, q, ws, bias, dev)
    x = x.to(dev)
    assert_within(hip_fp8_linear(x, q, ws, bias), want, spread)
    res = normal(2, m, n).to(dtype).to(dev)
    for vectors in (1, 4):
        gate = normal(3, vectors, 1, n).to(dtype).to(dev)
        rows = gate[:, 0].double().repeat_interleave(m // vectors, 0)
        full = res.double() + rows * want
        into = res.clone().view(vectors, -1, n)
        got = hip_fp8_linear(x.view(vectors, -1, k), q, ws, bias, residual=into, gate=gate, inplace=True)
        assert got is into
        assert_within(got.view(m, n), full, rows.abs() * spread + U * ((rows * want).abs() + full.abs()), f"{vectors} gates")


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_whole_large_tiles_of_experts(dev, tuning, dtype, gather):
    from convrot_mlx_amd import expert_plan, hip_fp8_grouped_linear

    tuning.set("fp8_tile", "256x256")
    tokens, experts, n, k = 2900, 2, 2820, 272
    plan = expert_plan(choose(1, tokens, 1, experts).to(dev), experts)
    q, ws = fp8_weight(n, experts, n, k, dev)
    x = normal(n, tokens, k).to(dtype)
    values = plain.row_values(*plain.codes(x)).to(dev)
    rows = values[plan.order.long()] if gather else values
    got = hip_fp8_grouped_linear(x.to(dev), q, ws, plan, gather=gather)
    at = plan.offsets.tolist()
    for e in range(experts):
        want, spread = plain.product(rows[at[e]: at[e + 1]], plain.weight_values(q[e], ws[e]), dtype == F32)
        assert_within(got[at[e]: at[e + 1]], want, spread, f"expert {e}")
    assert not got[at[-1]:].any()


@pytest.mark.parametrize("n,k", [(2820, 2100), (2100, 2820)])
def test_whole_large_tiles_in_float16(dev, tuning, n, k):
    """More than half of the CUs have a tile of 256 x 256: of outputs and weights' gradients, then of rows' gradients."""
    tuning.set("grouped_tile", "256x256")
    check_products(dev, 2900, 1, 2, n, k, F16, False)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tile,m", [("32x64", 33), ("64x64", 70), ("64x128", 65), ("128x128", 200)])
def test_shared_k_and_epilogues(dev, tuning, tile, m, dtype):
    """The last workgroup to arrive adds the parts and goes through every epilogue: up to 7 additions more than with K
    whole, of the 2 a block of 128 (33 of them) that the bound counts."""
    from convrot_mlx_amd import hip_fp8_linear

    tuning.set("fp8_tile", tile)
    n, k = 203, 4112
    q, ws = weight(k, n, k, dev)
    bias, x = normal(n, n).to(dev), normal(m, m, k).to(dtype)
    want, spread = wanted(x, q, ws, bias, dev)
    x, spread = x.to(dev), 2 * spread
    res, gate = normal(2, m, n).to(dtype).to(dev), normal(3, 1, n).to(dtype).to(dev)
    full = res.double() + gate.double() * want
    gated = gate.double().abs() * spread + U * ((gate.double() * want).abs() + full.abs())
    for split in (3, 7):
        tuning.set("fp8_split", split)
        for _ in range(2):
            assert_within(hip_fp8_linear(x, q, ws, bias), want, spread, f"{split} parts")
            got = hip_fp8_linear(x, q, ws, bias, residual=res, gate=gate)
            assert_within(got, full, gated, f"{split} parts, gated")
            into = res.clone()
            assert hip_fp8_linear(x, q, ws, bias, residual=into, gate=gate, inplace=True) is into
            assert torch.equal(into, got)


def test_large_tiles_do_not_share_k(dev, tuning):
    """A split asked for with tiles of 256 x 256 is not made: the same bits as without."""
    from convrot_mlx_amd import hip_fp8_linear

    tuning.set("fp8_tile", "256x256")
    q, ws = weight(1, 200, 4112, dev)
    x = normal(2, 300, 4112).to(BF16).to(dev)
    tuning.set("fp8_split", 1)
    want = hip_fp8_linear(x, q, ws)
    tuning.set("fp8_split", 7)
    assert torch.equal(hip_fp8_linear(x, q, ws), want)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,choices,n", [(1, 1, 8), (6, 2, 33), (40, 3, 264), (300, 4, 2056), (9, 5, 17)])
def test_gathered_rows(dev, rows, choices, n, dtype):
    """Row index[s] / choices of x, zeros for an index out of range: rows in 16-byte steps and one by one."""
    from convrot_mlx_amd import _native

    g = torch.Generator().manual_seed(rows)
    x = normal(n, rows, n).to(dtype)
    index = torch.randint(0, rows * choices, (rows * choices + 3,), generator=g)
    index[0], index[-1] = -1, rows * choices
    want = torch.where(((index < 0) | (index >= rows * choices))[:, None], torch.zeros((), dtype=dtype), x[(index // choices).clamp(0, rows - 1)])
    i = index.int().to(dev)
    for view in (x.to(dev), torch.cat([x, x, x], 1).to(dev)[:, n: 2 * n]):
        out = torch.full((len(index), n), float("nan"), dtype=dtype, device=dev)
        _native.check(_native.load().convrot_gather_rows(
            view.data_ptr(), _native.dtype_code(dtype), rows, view.stride(0), i.data_ptr(), choices, len(index), n, out.data_ptr(),
            _native.stream_handle(out.device)))
        assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k", [(1, 65536), (16, 65521), (40, 65536), (300, 65536)])
def test_longest_rows(dev, m, k, dtype):
    """512 blocks, whose scales lie in LDS together; few tiles share K (up to 64 additions more, of 1024 in the bound)."""
    from convrot_mlx_amd import hip_fp8_linear

    n = 70
    q, ws = weight(k, n, k, dev)
    bias, x = normal(n, n).to(dev), normal(m, m, k).to(dtype)
    want, spread = wanted(x, q, ws, bias, dev)
    assert_within(hip_fp8_linear(x.to(dev), q, ws, bias), want, 2 * spread)


def test_most_experts(dev):
    """65536 experts, rows of a few of them: the first, the last and some between."""
    from convrot_mlx_amd import ExpertPlan, hip_fp8_grouped_linear, hip_grouped_linear, hip_grouped_linear_backward

    experts, n, k, rows = 65536, 16, 24, 90
    at = torch.zeros(experts + 1, dtype=torch.int32)
    met = {0: 3, 63: 1, 64: 40, 4096: 7, 40000: 20, 65535: 19}
    for e, count in met.items():
        at[e + 1:] += count
    assert at[-1] == rows
    plan = ExpertPlan(at.to(dev))
    w, x, dy = (normal(i, *s).to(BF16).to(dev) for i, s in enumerate(((experts, n, k), (rows, k), (rows, n))))
    q, ws = fp8_weight(1, experts, n, k, dev)
    values = plain.row_values(*plain.codes(x.cpu())).to(dev)
    out, (dx, dw) = hip_grouped_linear(x, w, plan), hip_grouped_linear_backward(dy, x, w, plan)
    codes = hip_fp8_grouped_linear(x, q, ws, plan)
    for e in met:
        r = slice(int(at[e]), int(at[e + 1]))
        assert_within(out[r], *product16(x[r].double(), w[e].double(), k), f"forward {e}")
        assert_within(dx[r], *product16(dy[r].double(), w[e].double().t().contiguous(), n), f"rows {e}")
        assert_within(dw[e], *product16(dy[r].double().t().contiguous(), x[r].double().t().contiguous(), met[e]), f"weights {e}")
        assert_within(codes[r], *plain.product(values[r], plain.weight_values(q[e], ws[e]), False), f"8 bits {e}")
    assert int(dw.flatten(1).any(1).sum()) == len(met)
