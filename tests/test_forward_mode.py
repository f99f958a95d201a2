"""CPU: the differentiable operators refuse dual tensors of forward mode, whose tangents their kernels would
drop (the kernels' calls are stood in for by torch operations)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from convrot_mlx_amd import norm, rotary


def stand_in_norm(x, weight=None, bias=None, *, return_stats=False, **kw):
    y = x.detach().clone()
    return (y, y.mean(-1), y.mean(-1)) if return_stats else y


def stand_in_rotary(q, k, table, **kw):
    return q.detach().clone(), k.detach().clone()


@pytest.mark.parametrize("grad", [True, False])
def test_dual_tensors(monkeypatch, grad):
    monkeypatch.setattr(norm, "hip_layer_norm", stand_in_norm)
    monkeypatch.setattr(rotary, "hip_qk_rotary", stand_in_rotary)
    x, w, heads, table = torch.randn(4, 8), torch.ones(8), torch.randn(1, 2, 3, 8), torch.randn(3, 4, 2)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: norm.layer_norm(dual(x), w), lambda: norm.layer_norm(x, dual(w)),
                     lambda: norm.layer_norm(x, scale=w, shift=dual(w)), lambda: rotary.qk_rotary(dual(heads), heads, table),
                     lambda: rotary.qk_rotary(heads, dual(heads), table),
                     lambda: rotary.qk_rotary(heads, heads, table, q_weight=dual(w))):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()
        assert torch.equal(norm.layer_norm(x, w), x) and torch.equal(rotary.qk_rotary(heads, heads, table)[0], heads)
    assert torch.equal(norm.layer_norm(x, w), x)
