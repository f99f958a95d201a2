"""GPU: row operators on more rows than one launch takes (a HIP grid has fewer than 2^32 threads an axis): the
rows on both sides of each seam have the bits that a call on them alone gives."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
ROWS = 2 ** 26 + 5  # of one wave each: 2^32 threads and more; a launch takes 67108860


@pytest.fixture(autouse=True)
def memory():
    if torch.cuda.mem_get_info()[0] < 64 * 2 ** 30:
        pytest.skip("needs 64 GiB of device memory")
    yield
    torch.cuda.empty_cache()


def many(rows, k, dev, seed=0):
    return torch.randn((rows, k), generator=torch.Generator(dev).manual_seed(seed), device=dev, dtype=BF16)


def seams(rows, *at):
    return [slice(max(0, a - 5), min(rows, a + 5)) for a in (0, *at, rows) if a <= rows]


@pytest.mark.parametrize("vectors", [0, 1, 3])
def test_layer_norm(dev, vectors):
    from convrot_mlx_amd import hip_layer_norm

    x, p = many(ROWS, 8, dev), many(8, 8, dev, 1)
    each = ROWS // max(1, vectors)
    kw = dict(scale=p[:vectors], shift=p[3: 3 + vectors]) if vectors else dict(weight=p[0], bias=p[1])
    y, mean, rstd = hip_layer_norm(x, return_stats=True, **kw)
    for part in seams(ROWS, 67108860, each, 2 * each):
        rows = torch.arange(part.start, part.stop, device=dev) // each
        own = dict(scale=p[:vectors][rows], shift=p[3: 3 + vectors][rows]) if vectors else kw
        want = hip_layer_norm(x[part], return_stats=True, **own)
        assert all(torch.equal(a, b) for a, b in zip((y[part], mean[part], rstd[part]), want))


def test_quantizer(dev):
    from convrot_mlx_amd import quantize_int8_rowwise

    x = many(ROWS, 8, dev)
    codes, scales = quantize_int8_rowwise(x)
    for part in seams(ROWS, 67108860):
        want = quantize_int8_rowwise(x[part])
        assert torch.equal(codes[part], want[0]) and torch.equal(scales[part], want[1])


@pytest.mark.parametrize("rows,k,seam", [(2 ** 23 + 9, 8, 2 ** 23 - 1), (140001, 1024, (2 ** 22 - 1) // 32)])
def test_layer_norm_gradient_of_a_vector_a_row(dev, rows, k, seam):
    from convrot_mlx_amd import hip_layer_norm, hip_layer_norm_backward

    x, dy, scale = (many(rows, k, dev, i) for i in range(3))
    _, mean, rstd = hip_layer_norm(x, scale=scale, return_stats=True)
    got = hip_layer_norm_backward(dy, x, mean, rstd, scale=scale)
    for part in seams(rows, (2 ** 22 - 1) // (k // 32 or 1), seam):
        want = hip_layer_norm_backward(dy[part], x[part], mean[part], rstd[part], scale=scale[part])
        assert all(torch.equal(a[part], b) for a, b in zip(got, want))


def test_rotary(dev):
    from convrot_mlx_amd import hip_qk_rotary

    q = many(ROWS, 16, dev).reshape(ROWS, 1, 1, 16)
    k = q[:, :0]
    ang = torch.arange(8, device=dev) * 0.3
    table = torch.stack([ang.cos(), ang.sin()], -1)[None]
    out, _ = hip_qk_rotary(q, k, table, q_weight=many(1, 16, dev, 1)[0])
    for part in seams(ROWS, 4 * (2 ** 24 - 1)):
        want, _ = hip_qk_rotary(q[part], k[part], table, q_weight=many(1, 16, dev, 1)[0])
        assert torch.equal(out[part], want)


def test_axes_table(dev):
    from convrot_mlx_amd import rotary_axes_table

    pos = torch.randint(0, 8192, (ROWS, 1), generator=torch.Generator(dev).manual_seed(0), device=dev, dtype=torch.int32)
    table = rotary_axes_table(pos, (128,))
    for part in seams(ROWS, (2 ** 24 - 1) * 4):
        assert torch.equal(table[part], rotary_axes_table(pos[part], (128,)))


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_product_of_2_30_rows(dev, dtype):
    """Rows whose scales lie past 4 GiB, and more tiles of 64 x 64 than a launch takes."""
    from convrot_mlx_amd import hip_w8a8_matmul

    rows = 2 ** 30 + 3000
    gen = torch.Generator(dev).manual_seed(0)
    act = torch.randint(-127, 128, (rows, 16), generator=gen, device=dev, dtype=torch.int8)
    w = torch.randint(-127, 128, (3, 16), generator=gen, device=dev, dtype=torch.int8)
    xs, ws = torch.rand((rows,), generator=gen, device=dev), torch.rand((3,), generator=gen, device=dev)
    out = hip_w8a8_matmul(act, w, xs, ws, ws, output_dtype=dtype)
    for part in seams(rows, 750, 3000, 2 ** 29, 2 ** 30):
        assert torch.equal(out[part], hip_w8a8_matmul(act[part], w, xs[part], ws, ws, output_dtype=dtype))
