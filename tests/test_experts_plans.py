"""CPU: what the experts' calls make of a plan that does not fit their rows, before any launch."""

from __future__ import annotations

import pytest
import torch

from convrot_mlx_amd import (ExpertPlan, grouped_linear, hip_combine_rows_backward, hip_fp8_grouped_linear, hip_grouped_linear,
                             hip_grouped_linear_backward)

P = 4096  # stands for any aligned device address: never read
MOST = 2 ** 31 - 2048  # features of a row that is walked in 32 bits, up to 2048 a step
FP8 = torch.float8_e4m3fn
BF16 = torch.bfloat16


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


PLAN = ExpertPlan(ints(0, 2, 4), ints(0, 2, 1, 3), ints(0, 2, 1, 3).view(2, 2))  # 2 tokens of 2 choices


@pytest.mark.parametrize("plan,rows", [(PLAN, 4), (PLAN, 1), (PLAN._replace(slots=PLAN.slots.view(4, 1)), 2),
                                       (PLAN._replace(slots=PLAN.slots.view(1, 4)), 2),
                                       (PLAN._replace(slots=ints(0, 1).view(2, 1)), 2)])
def test_rows_of_another_number_of_tokens(plan, rows):
    """Sorted rows are a whole number of choices of any divisor's tokens: the plan's slots say which it is."""
    x, w = torch.zeros(rows, 16, dtype=BF16), torch.zeros(2, 8, 16, dtype=BF16)
    codes = torch.zeros(2, 8, 16, dtype=torch.uint8).view(FP8)
    for call in (lambda: hip_grouped_linear(x, w, plan, gather=True), lambda: grouped_linear(x, w, plan, gather=True),
                 lambda: hip_fp8_grouped_linear(x, codes, torch.ones(2, 1, 1), plan, gather=True),
                 lambda: hip_grouped_linear_backward(torch.zeros(4, 8, dtype=BF16), x, w, plan, gather=True)):
        with pytest.raises(ValueError, match="the plan orders"):
            call()


def test_rows_that_fit_reach_the_device_check():
    w = torch.zeros(2, 8, 16, dtype=BF16)
    for rows, plan, gather in ((2, PLAN, True), (4, PLAN, False), (2, PLAN._replace(slots=None), True), (4, PLAN._replace(slots=None), True)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            hip_grouped_linear(torch.zeros(rows, 16, dtype=BF16), w, plan, gather=gather)


def test_gradient_of_gathered_rows_without_slots():
    """Refused by the forward pass: the backward pass could not sum a token's choices."""
    w, plan = torch.zeros(2, 8, 16, dtype=BF16), PLAN._replace(slots=None)
    x = torch.zeros(2, 16, dtype=BF16, requires_grad=True)
    with pytest.raises(ValueError, match="needs the plan's slots"):
        grouped_linear(x, w, plan, gather=True)
    # the weight's gradient alone, sorted rows, and no gradient at all do without
    for call in (lambda: grouped_linear(x.detach(), w.requires_grad_(), plan, gather=True),
                 lambda: grouped_linear(torch.zeros(4, 16, dtype=BF16, requires_grad=True), w, plan),
                 lambda: torch.no_grad()(grouped_linear)(x, w, plan, gather=True)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_gradient_of_weights_without_rows():
    with pytest.raises(ValueError, match="needs the rows"):
        hip_combine_rows_backward(torch.zeros(2, 6), None, PLAN, torch.ones(2, 2))


@pytest.mark.parametrize("features", [MOST + 1, 2 ** 31 - 1])
def test_rows_too_long_to_walk(features):
    from convrot_mlx_amd import _native

    lib = _native.load()
    for status in (lib.convrot_gather_rows(P, 2, 4, features, P, 2, 8, features, P, None),
                   lib.convrot_combine_rows(P, 2, 8, features, P, P, 4, 2, features, P, None),
                   lib.convrot_combine_rows_backward(P, features, P, features, 2, 8, P, P, P, 4, 2, features, P, P, None),
                   lib.convrot_combine_rows_backward(P, features, None, 0, 2, 8, P, P, None, 4, 2, features, P, None, None)):
        assert status == 2 and f"at most {MOST} features" in lib.convrot_last_error().decode()
