"""GPU: the adaptive norm whose result goes to 8-bit codes from registers (convrot_layer_norm_int8), at the
widths of every kernel form: against the 64-bit formula, and bit for bit the quantizer's codes of the same
norm in float32."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from _plain64 import norm
from test_gpu_norm import BF16, EPS, F16, F32, inputs
from test_gpu_w8a8 import quantize_plain

pytestmark = pytest.mark.gpu


def norm_to_codes(x, scale, shift, eps=EPS, pad=16):
    """codes [rows, K rounded up to `pad`] and scales of (1 + scale) * u + shift, rows of x in even groups."""
    from convrot_mlx_amd import _native as nat

    rows, k = x.shape
    codes = torch.full((rows, -(-k // pad) * pad), 99, dtype=torch.int8, device=x.device)
    scales = torch.full((rows,), 7.0, device=x.device)
    nat.check(nat.load().convrot_layer_norm_int8(
        nat.ptr(x), nat.dtype_code(x.dtype), rows, k, x.stride(0), nat.ptr(scale), nat.ptr(shift),
        nat.dtype_code(scale.dtype), 1, rows // scale.shape[0], eps, nat.ptr(codes), codes.shape[1], nat.ptr(scales),
        nat.stream_of(x.device)))
    return codes, scales


def check(x, scale, shift, pad=16, x32=None):
    """x32: x in float32 in the same alignment, where x has one (rows of other alignments are summed in
    another order)."""
    from convrot_mlx_amd import hip_layer_norm

    rows, k = x.shape
    codes, scales = norm_to_codes(x, scale, shift, pad=pad)
    assert not codes[:, k:].any()
    # a code is at most half a step from the norm's value, whose float32 evaluation has its own bound
    each = rows // scale.shape[0]
    g64, b64 = (t.double().cpu().repeat_interleave(each, 0) for t in (scale, shift))
    want, _, _, _, _, off = norm(x.double().cpu(), 1 + g64, b64, EPS)
    step = scales.double().cpu()[:, None]
    assert ((codes[:, :k].double().cpu() * step - want).abs() <= 0.5001 * step + off).all()
    top = want.abs().amax(1, keepdim=True)
    assert ((step * 127 - top).abs() <= off.amax(1, keepdim=True) + 2.0 ** -22 * top).all()
    n32 = hip_layer_norm(x.float() if x32 is None else x32, scale=scale.float(), shift=shift.float(), eps=EPS)
    wc, ws = quantize_plain(n32)
    assert np.array_equal(codes[:, :k].cpu().numpy(), wc) and np.array_equal(scales.cpu().numpy(), ws)


WIDTHS = [(1, 1), (3, 7), (5, 64), (6, 500), (4, 512), (3, 1000), (2, 1024), (3, 1001), (2, 2048), (2, 2690), (4, 3072), (2, 4096),
          (4, 5120), (2, 6458), (2, 8192), (2, 10001), (2, 12288), (2, 15360), (1, 20001), (2, 32768), (1, 40000),
          (1, 65535), (1, 65536)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,k", WIDTHS)
def test_widths(dev, rows, k, dtype):
    x, scale, shift, _ = inputs(k, rows, k, dtype, dev)
    check(x, scale, shift)
    if k % 128 and k < 65000:
        check(x, scale, shift, pad=128)


@pytest.mark.parametrize("k", [96, 770, 3072, 5121])
def test_vectors_and_float32_parameters(dev, k):
    x, scale, shift, _ = inputs(k, 36, k, BF16, dev, 4)
    check(x, scale, shift)
    check(x, scale.float() + 0.001, shift.float())


def test_strided_rows(dev):
    base, scale, shift, _ = inputs(3, 11, 3200, BF16, dev)
    for at, k in ((0, 3072), (8, 3072), (1, 3072), (3, 1333), (5, 512)):
        check(base[:, at: at + k], scale[:, :k].contiguous(), shift[:, :k].contiguous(),
              x32=base.float()[:, at: at + k])


@pytest.mark.parametrize("k", [100, 512, 3072, 3075, 9000])
def test_non_finite_and_constant_rows(dev, k):
    """A row with a NaN or an infinity gets codes 0 and the scale NaN, a constant row its shift, and the rows
    beside them are as they are alone."""
    x, scale, shift, _ = inputs(5, 6, k, BF16, dev)
    x[1, 5], x[2, k - 1], x[3] = float("nan"), -float("inf"), 4.0
    codes, scales = norm_to_codes(x, scale, shift)
    assert not codes[1:3].any() and scales[1:3].isnan().all()
    wc, ws = quantize_plain(shift)
    assert np.array_equal(codes[3:4, :k].cpu().numpy(), wc) and np.array_equal(scales[3:4].cpu().numpy(), ws)
    keep = torch.tensor([0, 4, 5], device=dev)
    alone = norm_to_codes(x[keep].contiguous(), scale, shift)
    assert torch.equal(codes[keep], alone[0]) and torch.equal(scales[keep], alone[1])
    zero = norm_to_codes(x[3:4], torch.zeros_like(scale), torch.zeros_like(shift))
    assert not zero[0].any() and zero[1] == 0


@pytest.mark.parametrize("k", [3072, 5120, 1000])
def test_layer_at_wide_inputs(dev, k):
    """The whole layer: the product of those codes."""
    from convrot_mlx_amd import Int8Linear, hip_w8a8_matmul

    x, scale, shift, _ = inputs(7, 21, k, BF16, dev)
    weight = torch.randn((40, k), generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    layer = Int8Linear(k, 40, device=dev).load_weight(weight)
    codes, scales = norm_to_codes(x, scale, shift)
    want = hip_w8a8_matmul(codes[:, :k], layer.qweight, scales, layer.scales, layer.bias, output_dtype=BF16)
    assert torch.equal(layer.forward_modulated(x, shift, scale, eps=EPS), want)
