"""Plain 64-bit forms of the 8-bit floating point linears, with bounds on what the kernels may add
(elementwise, unit roundoff U)."""

from __future__ import annotations

import torch

from tests._plain64 import U

# The matrix units' FP8 form aligns the products of 16 neighbouring features to the largest and cuts what
# lies over 13 bits below its leading one: of each of 15 others, less than 2^-13 of the largest product.
CUT = 15 * 2.0 ** -13


def codes(x: torch.Tensor):
    """(values of the e4m3 codes [M, K], scales [M, K / 128]) in 64 bits: the smallest power of two with
    absmax / scale <= 448; four bits of mantissa, steps of 2^-9 at the least, ties to even."""
    m, k = x.shape
    pad = torch.zeros((m, (k + 127) // 128 * 128), dtype=torch.float64, device=x.device)
    pad[:, :k] = x.double()
    b = pad.view(m, -1, 128)
    a = b.abs().amax(2, keepdim=True)
    zero, bad = a < 2.0 ** -100, ~torch.isfinite(a)
    mantissa, exponent = torch.frexp(torch.where(zero | bad, 1.0, a))
    scale = torch.exp2((exponent - 9 + (mantissa > 0.875).int()).double())
    v = b / scale
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    q = torch.where(zero | bad, 0.0, torch.round(v / step) * step)
    scale = torch.where(zero, 0.0, torch.where(bad, float("nan"), scale))
    return q.view(m, -1)[:, :k], scale[..., 0]


def weight_values(q: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    n, k = q.shape[-2:]
    s = scales.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]
    return q.double() * s


def row_values(q: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return q.double() * scales.double().repeat_interleave(128, 1)[:, : q.shape[1]]


def product(x: torch.Tensor, w: torch.Tensor, wide: bool):
    """x [M, K] times w [N, K]^T (values with their scales), and its bound; wide: products added at float32."""
    mag = x.abs() @ w.abs().t().contiguous()
    k = x.shape[1]
    # float32 sums: 128 products of a block (in sixteens), then a multiplication and an addition a block
    spread = U * (32 + 2 * ((k + 127) // 128)) * mag + U * 2 * mag
    if wide:
        spread = spread + U * 128 * mag
    else:
        pad = lambda t: torch.nn.functional.pad(t, (0, -k % 16)).unflatten(1, (-1, 16)).abs().amax(2)  # noqa: E731
        spread = spread + CUT * (pad(x) @ pad(w).t().contiguous())
    return x @ w.t().contiguous(), spread
