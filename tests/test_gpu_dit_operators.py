"""GPU: the operators together in the example's diffusion transformer, small: 8-bit linears with the
norm in front and the gated residual behind, head norms and rotary positions in one kernel, and a
training step through layer_norm and qk_rotary, against the same model in torch operations."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def model_and_inputs(dev):
    from examples.flux1_dev import dit

    p = dit.FluxParams(in_channels=32, vec_in_dim=48, context_in_dim=64, hidden_size=256, num_heads=2, depth=2,
                       depth_single_blocks=2)
    return dit, p, dit.build(p, dev), dit.make_inputs(p, 64, 19, dev)


def rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


def test_fused_rotary_and_norm_in_the_dense_model(dev):
    """The same numbers up to bf16 rounding: the torch ops round q and k after the norm and
    normalized inputs after every operation, the operators once (2^-8 an element and block)."""
    dit, _, model, inputs = model_and_inputs(dev)
    with torch.no_grad():
        plain = model(**inputs)
        dit.set_fused_rotary(model, True)
        assert rel(model(**inputs), plain) < 0.02
        dit.set_fused_norm(model, True)
        fused = model(**inputs)
        assert rel(fused, plain) < 0.02
        assert torch.equal(model(**inputs), fused)
        dit.set_fused_rotary(model, False), dit.set_fused_norm(model, False)
        assert torch.equal(model(**inputs), plain)


def test_int8_and_mixed_models(dev):
    """8-bit rows are off by 2^-8 of their largest value a product: near bf16's own rounding; the
    mixed model's 4-bit layers by 2^-4."""
    from convrot_mlx_amd import ConvRotLinear, Int8Linear, replace_convrot_linears, replace_int8_linears

    dit, p, model, inputs = model_and_inputs(dev)
    with torch.no_grad():
        dense = model(**inputs)
        names = replace_int8_linears(model)
        assert len(names) == sum(isinstance(m, Int8Linear) for m in model.modules()) > 20
        assert rel(model(**inputs), dense) < 0.1
        for setter in (dit.set_fused_modulation, dit.set_fused_residual, dit.set_fused_rotary):
            setter(model, True)
        fused = model(**inputs)
        assert rel(fused, dense) < 0.1
        mixed = dit.build(p, dev)
        eight = replace_int8_linears(mixed, select=dit.keep_at_8_bits)
        four = replace_convrot_linears(mixed, backend="hip-w4a4", group_size=64)
        assert eight and four and not any(isinstance(m, torch.nn.Linear) for m in mixed.modules())
        for setter in (dit.set_fused_modulation, dit.set_fused_gelu, dit.set_fused_residual, dit.set_fused_rotary):
            setter(mixed, True)
        assert any(isinstance(m, ConvRotLinear) for m in mixed.modules())
        assert rel(mixed(**inputs), dense) < 0.8


def test_training_step_of_a_block(dev):
    from convrot_mlx_amd import rotary_axes_table

    dit, p, model, inputs = model_and_inputs(dev)
    vec = torch.randn((1, 256), device=dev).bfloat16()
    ids = torch.cat([inputs["txt_ids"], inputs["img_ids"]], 1)
    pes = {False: model.pe_embedder(ids), True: rotary_axes_table(ids, p.axes_dim, p.theta)}
    for block in (model.single_blocks[0], model.double_blocks[0]):
        x = torch.randn((1, 83, 256), device=dev).bfloat16().requires_grad_()
        grads = {}
        for on in (False, True):
            dit.set_fused_rotary(block, on), dit.set_fused_norm(block, on)
            if block is model.single_blocks[0]:
                y = block(x, vec, pes[on])
            else:
                y = torch.cat(block(x[:, 19:], x[:, :19], vec, pes[on]), 1)
            grads[on] = torch.autograd.grad(y.float().square().sum(), [x, *block.parameters()])
        for a, b in zip(grads[True], grads[False]):
            assert a.shape == b.shape and a.isfinite().all()
            assert rel(a, b) < 0.05
