"""GPU: training a part of the example's blocks through the fused operators."""

from __future__ import annotations

import pytest
import torch

from test_gpu_dit_operators import model_and_inputs, rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("double", [True, False])
def test_head_norm_scales_behind_frozen_projections(dev, double):
    """Only the head norms' scales are trained: inputs and projections need no gradient, and the fused operator
    gives the scales the gradients that the torch operations give."""
    from convrot_mlx_amd import rotary_axes_table

    dit, p, model, inputs = model_and_inputs(dev)
    block = model.double_blocks[0] if double else model.single_blocks[0]
    scales = [t for name, t in block.named_parameters() if "norm" in name]
    assert len(scales) == (4 if double else 2)
    for t in block.parameters():
        t.requires_grad_(False)
    for t in scales:
        t.requires_grad_(True)
    ids = torch.cat([inputs["txt_ids"], inputs["img_ids"]], 1)
    pes = {False: model.pe_embedder(ids), True: rotary_axes_table(ids, p.axes_dim, p.theta)}
    gen = torch.Generator(dev).manual_seed(3)
    x = torch.randn((1, 83, 256), device=dev, generator=gen).bfloat16()
    vec = torch.randn((1, 256), device=dev, generator=gen).bfloat16()
    grads = {}
    for on in (False, True):
        dit.set_fused_rotary(block, on)
        y = torch.cat(block(x[:, 19:], x[:, :19], vec, pes[on]), 1) if double else block(x, vec, pes[on])
        grads[on] = torch.autograd.grad(y.float().square().sum(), scales)
    for a, b in zip(grads[True], grads[False]):
        assert a.isfinite().all() and b.any() and rel(a, b) < 0.05  # bf16 roundings of q and k, as in the step's test
