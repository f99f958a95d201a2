"""CPU: a call without a gradient keeps its forward result and refuses the backward pass (the kernels'
calls are stood in for by torch operations)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from convrot_mlx_amd import Int8Linear, int8
from convrot_mlx_amd import _native as nat


def doubled(x):
    return lambda: torch.stack([x.detach()[0] * 2, x.detach()[1] * 2]).reshape(-1, 3)


def test_plain_calls_are_not_touched():
    x = torch.randn(2, 3)
    out = torch.zeros(2, 3)
    assert nat.without_gradient(lambda: out, "it", x, None) is out
    with torch.no_grad():
        assert nat.without_gradient(lambda: out, "it", x.clone().requires_grad_()) is out


def test_backward_is_refused_and_the_result_may_be_changed():
    x = torch.randn(2, 3, requires_grad=True)
    y = nat.without_gradient(doubled(x), "it", x, None)
    assert torch.equal(y, 2 * x) and y.requires_grad
    y += 1
    y[0] *= 2
    with pytest.raises(RuntimeError, match="it has no gradient"):
        y.sum().backward()
    assert x.grad is None


@pytest.mark.parametrize("needs", [(True, False), (False, True), (True, True)])
def test_in_place(needs):
    x, r = (torch.randn(2, 3, requires_grad=n) for n in needs)
    r = r * 1.0

    def run():
        r.data.add_(1)
        return r

    want = r.detach() + 1
    saved = r.exp() if r.requires_grad else None
    y = nat.without_gradient(run, "it", x, r, target=r)
    assert y is r and torch.equal(y.detach(), want)
    with pytest.raises(RuntimeError, match="it has no gradient"):
        (y.sum() + (0 if saved is None else saved.detach().sum())).backward()


def test_leaf_in_place_is_refused_before_the_call():
    r = torch.zeros(2, 3, requires_grad=True)

    def run():
        raise AssertionError("called")

    with pytest.raises(RuntimeError, match="leaf tensor"):
        nat.without_gradient(run, "it", r, target=r)


def test_forward_mode_is_refused():
    x = torch.randn(2, 3)
    with forward_ad.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="jvp"):
                nat.without_gradient(doubled(x), "it", forward_ad.make_dual(x, torch.ones_like(x)))
        assert torch.equal(nat.without_gradient(doubled(x), "it", x), 2 * x)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("call", ["layer", "modulated", "linear", "matmul"])
def test_every_8_bit_call(monkeypatch, call, inplace):
    """Each entry point, its launch replaced by a sum over features."""
    monkeypatch.setattr(nat, "on_device", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(int8, "_gated_residual", lambda res, gate, shape, dtype, inplace: int8.GatedResidual(res, None, 0, 1,
                                                                                                         inplace))

    def linear(x, weight, ws, bias, k, residual, gate, inplace):
        out = x.detach().sum(-1, keepdim=True).expand(*x.shape[:-1], weight.shape[0])
        if inplace:
            residual.data.copy_(out)
        return residual if inplace else out.clone()

    monkeypatch.setattr(int8, "_linear", linear)
    monkeypatch.setattr(int8, "_w8a8", lambda a, w, xs, ws, b, k, dtype, gr: linear(a.float() * xs.detach()[:, None], w, ws, b, k,
                                                                                    gr and gr.residual, None, inplace))
    monkeypatch.setattr(Int8Linear, "_modulated",
                        lambda self, x, sh, sc, eps, res, gate, inplace: linear(x, self.qweight, None, None, 0, res, gate, inplace))
    x, layer = torch.randn(5, 32, requires_grad=True), Int8Linear(32, 4)
    residual = torch.zeros(5, 4) if inplace else None
    kw = dict(residual=residual, inplace=inplace)
    codes, xs = torch.ones(5, 32, dtype=torch.int8), torch.ones(5, requires_grad=True)
    calls = {"layer": lambda: layer(x, **kw), "modulated": lambda: layer.forward_modulated(x, x[0, :32], x[1, :32], **kw),
             "linear": lambda: int8.hip_w8a8_linear(x, layer.qweight, layer.scales, **kw),
             "matmul": lambda: int8.hip_w8a8_matmul(codes, layer.qweight, xs, layer.scales, output_dtype=torch.float32, **kw)}
    with torch.no_grad():
        want = calls[call]().clone()
        assert not want.requires_grad
    got = calls[call]()
    assert got.requires_grad and torch.equal(got, want)
    with pytest.raises(RuntimeError, match="has no gradient"):
        got.sum().backward()


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("call", ["forward", "forward_modulated", "forward_gelu"])
def test_every_4_bit_layer_call(monkeypatch, call, inplace):
    from convrot_mlx_amd import ConvRotLinear, core

    def project(self, prep, lead, dtype, residual, gate, inplace):
        out = torch.ones(*lead, self.out_features)
        if inplace:
            residual.data.copy_(out)
        return residual if inplace else out

    monkeypatch.setattr(ConvRotLinear, "_project", project)
    monkeypatch.setattr(core, "_linear_rows_eligible", lambda *args: False)
    layer, x = ConvRotLinear(64, 4, group_size=64), torch.randn(5, 64, requires_grad=True)
    args = (x.detach()[0], x.detach()[1]) if call == "forward_modulated" else ()
    kw = dict(residual=torch.zeros(5, 4), inplace=True) if inplace else {}
    with torch.no_grad():
        assert not getattr(layer, call)(x, *args, **kw).requires_grad
    got = getattr(layer, call)(x, *args, **kw)
    assert got.requires_grad and (got == 1).all()
    with pytest.raises(RuntimeError, match="ConvRotLinear has no gradient"):
        got.sum().backward()
