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
