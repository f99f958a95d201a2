"""GPU: the rows summed back, and their gradient, on plans of any content."""

from __future__ import annotations

import pytest
import torch

from tests._plain64 import U, assert_within

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def plans(tokens, choices):
    """(order, slots) of a permutation, and of ones whose places are out of range, named for no choice or for another."""
    count = tokens * choices
    g = torch.Generator().manual_seed(count)
    order = torch.randperm(count, generator=g)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(count)
    yield order, slots
    out = slots.clone()
    out[torch.rand(count, generator=g) < 0.3] = count + 5
    out[0] = -1
    yield order, out
    names = order.clone()
    names[torch.rand(count, generator=g) < 0.3] = -7
    names[0] = 2 ** 31 - 1
    yield names, slots
    yield order, torch.full_like(slots, -1)
    yield torch.randint(0, count, (count,), generator=g), torch.randint(0, count, (count,), generator=g)


def rows_gradient(order, slots, weights, dout, choices):
    """weights[i] * dout[i // choices] for the row s that names choice i = order[s] and is its place, else 0."""
    count = order.numel()
    want = torch.zeros((count, dout.shape[1]), dtype=torch.float64)
    for s, i in enumerate(order.tolist()):
        if 0 <= i < count and int(slots[i]) == s:
            want[s] = weights[i].double() * dout[i // choices].double()
    return want


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,choices,n", [(2, 2, 40), (1, 1, 33), (7, 5, 264), (33, 8, 17), (20, 3, 2056), (300, 2, 64)])
def test_gradient_of_rows_that_no_choice_has(dev, tokens, choices, n, dtype):
    """Every row of the gradient is written, whatever its memory held: zeros where no choice's place is the row."""
    from convrot_mlx_amd import ExpertPlan, _native, combine_rows, hip_combine_rows_backward

    code = {F32: 0, F16: 1, BF16: 2}[dtype]
    assert code == _native.dtype_code(dtype)
    count = tokens * choices
    y, dout, w = normal(1, count, n).to(dtype), normal(2, tokens, n).to(dtype), normal(3, tokens, choices)
    dev_y, dev_dout, dev_w = y.to(dev), dout.to(dev), w.to(dev)
    offsets = torch.tensor([0, count], dtype=torch.int32, device=dev)
    for order, slots in plans(tokens, choices):
        o, s = order.int().to(dev), slots.int().to(dev).view(tokens, choices)
        want = rows_gradient(order, slots, w.flatten(), dout, choices)
        dy = torch.full((count, n), float("nan"), dtype=dtype, device=dev)
        dw = torch.full((tokens, choices), float("nan"), dtype=F32, device=dev)
        _native.check(_native.load().convrot_combine_rows_backward(
            dev_dout.data_ptr(), n, dev_y.data_ptr(), n, code, count, o.data_ptr(), s.data_ptr(), dev_w.data_ptr(), tokens,
            choices, n, dy.data_ptr(), dw.data_ptr(), _native.stream_handle(dev_y.device)))
        assert_within(dy, want, U * want.abs())
        assert not dw.isnan().any()
        plan = ExpertPlan(offsets, o, s)
        junk = torch.full((count, n), float("nan"), dtype=dtype, device=dev)
        del junk
        assert torch.equal(hip_combine_rows_backward(dev_dout, dev_y, plan, dev_w)[0], dy)
        rows = dev_y.clone().requires_grad_()
        (got,) = torch.autograd.grad(combine_rows(rows, plan, dev_w), rows, dev_dout)
        assert torch.equal(got, dy)
        plain = rows_gradient(order, slots, torch.ones(count), dout, choices)
        assert torch.equal(hip_combine_rows_backward(dev_dout, None, plan)[0].cpu().double(), plain)
