"""Plain 64-bit forms of the layer norm and rotary operators, with first-order bounds on what
float32 evaluation and one rounding to the output type may add (elementwise, unit roundoff U)."""

from __future__ import annotations

import torch

U = 2.0 ** -24
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}


def assert_within(got: torch.Tensor, want: torch.Tensor, spread: torch.Tensor, what: str = "") -> None:
    """|got - want| <= half a unit of got's type + spread, all elements finite."""
    got64 = got.detach().double().cpu()
    want, spread = want.cpu(), spread.cpu()
    assert torch.isfinite(got64).all(), f"{what}: not finite"
    bound = ROUND[got.dtype] * (want.abs() + spread) + TINY[got.dtype] + spread
    over = (got64 - want).abs() / bound
    assert over.max().item() <= 1.0, f"{what}: {over.max().item():.2f} times its bound at {int(over.argmax())}"


# ------------------------------------------------------------------ layer norm
#
# Sums of K values in float32: a thread adds at most 64 in a row, then 10 lane and 16 wave steps,
# so a sum is off by at most 96 U times the sum of magnitudes.


def norm(x, gain, shift, eps):
    """x [R, K], gain and shift [R or 1, K] in 64 bits: y, the parts, and the bounds of u and y."""
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1.0 / (c.square().mean(1, keepdim=True) + eps).sqrt()
    u = c * rstd
    du = U * (96 * rstd * (x.abs().mean(1, keepdim=True) + x.abs()) + 128 * u.abs())
    y = u * gain + shift
    return y, mean, rstd, u, du, du * gain.abs() + 4 * U * ((u * gain).abs() + shift.abs())


def norm_grads(x, gain, dy, eps, vectors):
    """dx, dgain, dshift [V, K] with bounds."""
    rows, k = x.shape
    _, _, rstd, u, du, _ = norm(x, gain, torch.zeros_like(gain), eps)
    h = dy * gain
    hu = h * u
    dx = rstd * (h - h.mean(1, keepdim=True) - u * hu.mean(1, keepdim=True))
    mag = h.abs() + h.abs().mean(1, keepdim=True) + u.abs() * hu.abs().mean(1, keepdim=True)
    dx_off = rstd * (256 * U * mag + du * hu.abs().mean(1, keepdim=True)
                     + u.abs() * (h.abs() * du).mean(1, keepdim=True))
    each = rows // vectors
    group = lambda t: t.reshape(vectors, each, k).sum(1)  # noqa: E731
    order = (each + 64) * U
    return (dx, dx_off, group(dy * u), order * group((dy * u).abs()) + group(dy.abs() * du), group(dy),
            order * group(dy.abs()))


# ------------------------------------------------------------------ rotary


def turn(x, cos, sin, interleaved):
    """(turned, magnitudes) of the pairs of x [.., D]."""
    p = cos.shape[-1]
    y, mag = x.clone(), x.abs()
    ia = torch.arange(p) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else p)
    ia, ib = ia.to(x.device), ib.to(x.device)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * cos - b * sin, a * sin + b * cos
    mag[..., ia], mag[..., ib] = (a * cos).abs() + (b * sin).abs(), (a * sin).abs() + (b * cos).abs()
    return y, mag


def rotary(x, w, table, eps, interleaved):
    """x [B, H, L, D], w [D] or None, table [B or 1, L, P, 2]: (y, bound)."""
    cos, sin = table[:, None, :, :, 0], table[:, None, :, :, 1]
    n = x if w is None else x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    y, mag = turn(n, cos, sin, interleaved)
    return y, 48 * U * mag


def rotary_grads(x, w, table, dy, eps, interleaved):
    """(dx, bound, dw, bound); dw None without a weight."""
    cos, sin = table[:, None, :, :, 0], table[:, None, :, :, 1]
    g, mag = turn(dy, cos, -sin, interleaved)
    if w is None:
        return g, 4 * U * mag, None, None
    r = 1.0 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    u = x * r
    along = (g * w * u).mean(-1, keepdim=True)
    dx = r * (g * w - u * along)
    size = mag * w.abs()
    dx_off = 96 * U * r * (size + u.abs() * (size * u.abs()).mean(-1, keepdim=True))
    count = x.shape[0] * x.shape[1] * x.shape[2]
    return dx, dx_off, (g * u).sum((0, 1, 2)), (count + 96) * U * (mag * u.abs()).sum((0, 1, 2))
