"""CPU: which shapes of modulation vectors the norms take: the grouping of rows in order that the kernels
do must be what broadcasting over x means."""

from __future__ import annotations

import pytest
import torch

from convrot_mlx_amd import norm

K = 3
SHAPES = [  # x, vectors
    ((4, 5), (1,)), ((4, 5), (4,)), ((4, 5), (2,)), ((4, 5), (20,)), ((4, 5), (4, 1)), ((4, 5), (1, 1)), ((4, 5), (4, 5)),
    ((4, 5), (10, 1)), ((2, 3, 4), (2, 1, 1)), ((2, 3, 4), (2, 3, 1)), ((2, 3, 4), (2, 3, 4)), ((2, 3, 4), (6, 1)),
    ((2, 3, 4), (1, 1, 1)), ((2, 3, 4), (2, 1, 1, 1)), ((1, 5), (1, 5)), ((1, 3, 4), (3, 1)), ((6,), (2, 3)), ((6,), (3, 1)),
    ((1, 1, 5), (1, 1, 5)), ((0, 5), (1, 1)),
]
REFUSED = [((4, 5), (1, 5)), ((2, 3, 4), (1, 3, 1)), ((2, 3, 4), (3, 1)), ((2, 3, 4), (3, 4)), ((2, 3, 4), (2, 1, 4)),
           ((2, 2, 4), (2, 1)), ((4, 5), (2, 2)), ((4, 5), (2, 10)), ((2, 3, 4), (1, 1, 4))]


@pytest.mark.parametrize("lead,vectors", SHAPES)
def test_taken(lead, vectors):
    x, t = torch.zeros(*lead, K), torch.arange(torch.Size(vectors).numel()).float()[:, None].expand(-1, K)
    t = t.reshape(*vectors, K)
    _, _, each, _ = norm.norm_operands(x.reshape(-1, K), None, None, t, None, x.shape)
    rows = x.numel() // K
    grouped = torch.arange(rows) // each
    if len(vectors) > 1 and t.ndim <= x.ndim and all(d in (1, n) for d, n in zip(t.shape[::-1], x.shape[::-1])):
        assert torch.equal(t.expand(x.shape).reshape(-1, K)[:, 0].long(), grouped)


@pytest.mark.parametrize("lead,vectors", REFUSED)
@pytest.mark.parametrize("name", ["scale", "shift"])
def test_refused(lead, vectors, name):
    x, t = torch.zeros(*lead, K), torch.zeros(*vectors, K)
    kw = dict(scale=None, shift=None) | {name: t}
    with pytest.raises(ValueError, match="no even groups of rows"):
        norm.norm_operands(x.reshape(-1, K), None, None, kw["scale"], kw["shift"], x.shape)


def test_refused_by_the_fused_preparation():
    from convrot_mlx_amd import ConvRotLinear, hip_fused_modulated_prepare

    x, t = torch.zeros(4, 5, 64), torch.zeros(1, 5, 64)
    with pytest.raises(ValueError, match="no even groups of rows"):
        hip_fused_modulated_prepare(x, t, t, 64)
    with pytest.raises(ValueError, match="no even groups of rows"):
        ConvRotLinear(64, 16, group_size=64).forward_modulated(x, t, t)
    with pytest.raises(RuntimeError, match="ROCm device"):
        hip_fused_modulated_prepare(x, t.transpose(0, 1), t.transpose(0, 1), 64)
