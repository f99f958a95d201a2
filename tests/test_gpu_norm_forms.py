"""GPU: layer norm and its gradient at the forms of parameters, types and sizes beside those of
test_gpu_norm.py."""

from __future__ import annotations

import pytest
import torch

from _plain64 import assert_within, norm, norm_grads
from test_gpu_norm import BF16, EPS, F16, F32, inputs

pytestmark = pytest.mark.gpu


def test_vectors_that_broadcast_to_other_rows_are_refused(dev):
    from convrot_mlx_amd import Int8Linear, hip_layer_norm, hip_layer_norm_backward, layer_norm

    x, scale, shift, dy = (t.reshape(4, 5, 64) if t.shape[0] == 20 else t[None]
                           for t in inputs(1, 20, 64, BF16, dev, 5))
    _, mean, rstd = hip_layer_norm(x, return_stats=True)
    leaf = scale.clone().requires_grad_()
    for call in (lambda: hip_layer_norm(x, scale=scale, shift=shift), lambda: layer_norm(x, scale=leaf),
                 lambda: hip_layer_norm_backward(dy, x, mean, rstd, scale=scale),
                 lambda: Int8Linear(64, 8, device=dev).forward_modulated(x, shift, scale)):
        with pytest.raises(ValueError, match="no even groups of rows"):
            call()
    # of a batch of one, and written out, these are groups in order
    y = hip_layer_norm(x, scale=scale.expand(4, 5, 64), shift=shift.expand(4, 5, 64))
    for b in range(4):
        assert torch.equal(hip_layer_norm(x[b: b + 1], scale=scale, shift=shift)[0], y[b])
    want = norm(x.reshape(20, 64).double().cpu(), 1 + scale[0].double().cpu().repeat(4, 1),
                shift[0].double().cpu().repeat(4, 1), EPS)
    assert_within(y.reshape(20, 64), want[0], want[5])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,k", [(1, 7), (3, 100), (5, 456), (3, 520), (4, 1000), (2, 2050), (2, 3080), (2, 4104), (2, 6152),
                                    (2, 8193), (2, 8200), (2, 16392), (1, 20001)])
def test_gradient_of_constant_rows_of_large_values(dev, rows, k, dtype):
    """A constant row has u = 0 and dx = rstd (h - mean(h)), however large its values: 2^110 with eps 1e-12,
    where mean times rstd passes float32's range.  Other rows share their sums with it."""
    from convrot_mlx_amd import hip_layer_norm, hip_layer_norm_backward

    eps = 1e-12
    x, w, b, dy = inputs(k, rows, k, dtype, dev)
    w = w[0] + 1
    x[0] = 2.0 ** 110
    y, mean, rstd = hip_layer_norm(x, w, b[0], eps=eps, return_stats=True)
    assert torch.equal(y[0], b[0]) and mean[0] == 2.0 ** 110
    dx, dw, db = hip_layer_norm_backward(dy, x, mean, rstd, weight=w)
    x64 = x.double().cpu()
    x64[0] = 0.0  # the same u, rstd and gradients
    wdx, odx, wdw, odw, wdb, odb = norm_grads(x64, w.double().cpu()[None], dy.double().cpu(), eps, 1)
    assert_within(dx, wdx, odx, "dx")
    assert_within(dw, wdw[0], odw[0], "dw")
    assert_within(db, wdb[0], odb[0], "db")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("form", ["bias", "weight16", "shift", "scale16", "weight32", "f64"])
def test_each_gradient_is_rounded_to_its_own_type(dev, dtype, form):
    """A float32 bias or shift beside 16-bit activations, alone or beside a 16-bit weight or scale: its
    gradient is the float32 sum, and the weight's that sum in 16 bits."""
    from convrot_mlx_amd import layer_norm

    x, w, b, dy = inputs(23, 300, 640, dtype, dev, 2)
    adaptive = form in ("shift", "scale16")
    other = torch.float64 if form == "f64" else F32
    gain = None if form in ("bias", "shift") else w if adaptive else (w[0] + 1).to(F32 if form == "weight32" else dtype)
    add = (b if adaptive else b[0]).to(dtype if form == "weight32" else other)
    leaves = [t.detach().clone().requires_grad_() for t in (gain, add) if t is not None]
    names = ("scale", "shift") if adaptive else ("weight", "bias")
    y = layer_norm(x, eps=EPS, **dict(zip(names[2 - len(leaves):], leaves)))
    y.backward(dy)
    vectors = 2 if adaptive else 1
    g64 = torch.ones(1, 640, dtype=torch.float64) if gain is None else gain.double().cpu().reshape(vectors, 640) + adaptive
    _, _, wdg, odg, wdb, odb = norm_grads(x.double().cpu(), g64.repeat_interleave(300 // vectors, 0)
                                          if adaptive and gain is not None else g64, dy.double().cpu(), EPS, vectors)
    assert leaves[-1].grad.dtype == leaves[-1].dtype
    sums = leaves[-1].grad.reshape(vectors, 640)
    assert_within(sums.float(), wdb, odb, "dshift") if form != "weight32" else assert_within(sums, wdb, odb, "dshift")
    if gain is not None:
        assert leaves[0].grad.dtype == gain.dtype
        assert_within(leaves[0].grad.reshape(vectors, 640), wdg, odg, "dgain")


def test_float32_shift_beyond_the_range_of_float16(dev):
    from convrot_mlx_amd import hip_layer_norm, hip_layer_norm_backward, layer_norm

    x, w, _, _ = inputs(29, 400, 64, F16, dev)
    dy = torch.full((400, 64), 1000.0, dtype=F16, device=dev)
    for kw in ({}, dict(weight=w[0] + 1)):
        bias = torch.zeros(64, device=dev, requires_grad=True)
        layer_norm(x, bias=bias, eps=EPS, **kw).backward(dy)
        assert torch.equal(bias.grad, torch.full((64,), 400e3, device=dev))
        _, mean, rstd = hip_layer_norm(x, eps=EPS, return_stats=True, **kw)
        _, dgain, dshift = hip_layer_norm_backward(dy, x, mean, rstd, shift_dtype=F32, **kw)
        assert dgain.dtype == F16 and torch.equal(dshift, bias.grad)
        assert hip_layer_norm_backward(dy, x, mean, rstd, **kw)[2].isinf().all()  # without it, x's type


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,k", [(1, 64), (70, 8), (33, 320), (40, 1024), (20, 1500), (12, 2690), (10, 3072), (6, 5120),
                                    (4, 6458), (3, 8200), (2, 12289), (2, 20000)])
def test_gradient_with_a_vector_a_row(dev, rows, k, dtype):
    """Modulation a token: every row's parameter gradients are that row's alone."""
    from convrot_mlx_amd import hip_layer_norm, hip_layer_norm_backward

    x, scale, shift, dy = inputs(rows + k, rows, k, dtype, dev, rows)
    y, mean, rstd = hip_layer_norm(x, scale=scale, shift=shift, eps=EPS, return_stats=True)
    g64 = 1 + scale.double().cpu()
    want, _, _, _, _, off = norm(x.double().cpu(), g64, shift.double().cpu(), EPS)
    assert_within(y, want, off, "y")
    dx, ds, dh = hip_layer_norm_backward(dy, x, mean, rstd, scale=scale)
    wdx, odx, wds, ods, wdh, odh = norm_grads(x.double().cpu(), g64, dy.double().cpu(), EPS, rows)
    assert_within(dx, wdx, odx, "dx")
    assert_within(ds, wds, ods, "dscale")
    assert torch.equal(dh, dy)
    only, none, _ = hip_layer_norm_backward(dy, x, mean, rstd, scale=scale, param_grads=False)
    assert none is None and torch.equal(only, dx)
