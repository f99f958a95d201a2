"""GPU: the linears of a mixture of experts and what lies around them, against plain forms in 64 bits."""

from __future__ import annotations

import pytest
import torch

from tests import _plain_fp8 as plain
from tests._plain64 import U, assert_within

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
FP8 = torch.float8_e4m3fn


def normal(seed, *shape, std=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std


def choose(seed, tokens, choices, experts, dropped=True):
    """Random experts (any, the same one twice too), some choices of none."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, experts, (tokens, choices), generator=g)
    if dropped:
        at = torch.rand((tokens, choices), generator=g)
        ids = torch.where(at < 0.06, -1, torch.where(at > 0.96, experts + 3, ids))
    return ids


def order_plain(ids, experts):
    flat = ids.flatten()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.sort(key, stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel())
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(key, minlength=experts + 1)[:experts].cumsum(0)])
    return offsets, order, slots.view(ids.shape)


# ------------------------------------------------------------------ the order by expert


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,choices,experts", [
    (0, 2, 4), (1, 1, 1), (1, 8, 8), (3, 2, 5), (16, 4, 64), (63, 1, 2), (64, 1, 1024), (65, 2, 7), (1000, 3, 60),
    (4096, 2, 16), (4097, 2, 1023), (8191, 1, 31), (9216, 4, 64), (3000, 8, 1024), (50001, 3, 33)])
def test_plan(dev, tokens, choices, experts, kind):
    from convrot_mlx_amd import expert_plan

    ids = choose(tokens + experts, tokens, choices, experts).to(kind)
    want = order_plain(ids.long(), experts)
    for _ in range(2):
        for t in (ids.to(dev), ids.to(dev).t().contiguous().t()):
            plan = expert_plan(t, experts)
            for name, got, w in zip(("offsets", "order", "slots"), plan, want):
                assert got.dtype == torch.int32 and got.shape == w.shape, name
                assert torch.equal(got.cpu().long(), w), name


@pytest.mark.parametrize("value", [0, 3, 4, -1, 2 ** 31, -2 ** 40])
def test_plan_of_one_expert(dev, value):
    from convrot_mlx_amd import expert_plan

    ids = torch.full((9000, 1), value)
    plan = expert_plan(ids.to(dev), 4)
    assert torch.equal(plan.order.cpu(), torch.arange(9000, dtype=torch.int32))
    start = [0] + [9000 if 0 <= value <= e else 0 for e in range(4)]
    assert plan.offsets.tolist() == start


def test_plan_of_one_choice_a_token(dev):
    from convrot_mlx_amd import expert_plan

    ids = choose(1, 100, 1, 8)
    a, b = expert_plan(ids.to(dev), 8), expert_plan(ids[:, 0].to(dev), 8)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and b.slots.shape == (100, 1)


# ------------------------------------------------------------------ the rows summed back


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,choices,n", [(1, 1, 8), (1, 5, 1), (7, 2, 33), (16, 4, 2048), (33, 8, 264), (100, 3, 72),
                                              (9, 9, 4096), (300, 2, 520), (5, 1, 8200), (40, 4, 1000)])
def test_combine(dev, tokens, choices, n, dtype):
    from convrot_mlx_amd import expert_plan, hip_combine_rows, hip_combine_rows_backward

    ids = choose(n, tokens, choices, 6)
    y, dout = normal(n, tokens * choices, n).to(dtype), normal(n + 1, tokens, n).to(dtype)
    w = normal(n + 2, tokens, choices)
    plan = expert_plan(ids.to(dev), 6)
    slots = plan.slots.cpu().long()
    rows = y.double()[slots]
    views = [lambda t: t.to(dev), lambda t: torch.cat([t, t, t], 1).to(dev)[:, n: 2 * n], lambda t: t.to(dev).t().contiguous().t()]
    for view in views:
        out = hip_combine_rows(view(y), plan, w.to(dev))
        want, mag = (rows * w.double()[..., None]).sum(1), (rows * w.double()[..., None]).abs().sum(1)
        assert_within(out, want, U * choices * mag)
        dy, dw = hip_combine_rows_backward(view(dout), view(y), plan, w.to(dev))
        want = torch.empty((tokens * choices, n), dtype=torch.float64)
        want[slots.flatten()] = (w.double()[..., None] * dout.double()[:, None]).flatten(0, 1)
        assert dw.dtype == F32
        assert_within(dy, want, U * want.abs())
        prod = rows * dout.double()[:, None]
        # a thread adds at most n / 32 products (of one feature each, or of 8), then 8 steps over threads
        assert_within(dw, prod.sum(2), U * (n / 32 + 16) * prod.abs().sum(2))
        out = hip_combine_rows(view(y), plan)
        assert_within(out, rows.sum(1), U * choices * rows.abs().sum(1))
        dy, dw = hip_combine_rows_backward(view(dout), None, plan)
        assert dw is None
        want[slots.flatten()] = dout.double().repeat_interleave(choices, 0)
        assert torch.equal(dy.cpu().double(), want)


def test_combine_differentiates(dev):
    from convrot_mlx_amd import combine_rows, expert_plan, hip_combine_rows_backward

    plan = expert_plan(choose(3, 40, 2, 5).to(dev), 5)
    y = normal(1, 80, 48).to(dev).requires_grad_()
    w = normal(2, 40, 2).to(BF16).to(dev).requires_grad_()
    dout = normal(3, 40, 48).to(dev)
    out = combine_rows(y, plan, w)
    dy, dw = torch.autograd.grad(out, (y, w), dout)
    want = hip_combine_rows_backward(dout, y.detach(), plan, w.detach())
    assert torch.equal(dy, want[0]) and torch.equal(dw, want[1]) and dw.dtype == BF16
    # against differences along a direction (the operator is bilinear: central differences are exact but for rounding)
    v, u = normal(4, 80, 48).to(dev), normal(5, 40, 2).to(dev)
    f = lambda s: (combine_rows(y.detach().double().float() + s * v, plan, w.detach().float() + s * u).double() * dout.double()).sum().item()  # noqa: E731
    slope, steps = (f(0.5) - f(-0.5)), (dy.double() * v.double()).sum().item() + (dw.double() * u.double()).sum().item()
    size = (dy.double() * v.double()).abs().sum().item() + (dw.double() * u.double()).abs().sum().item()
    # dw is rounded to bfloat16 (2^-8), the two sums are of float32 outputs of a few times `size`
    assert abs(slope - steps) <= 2.0 ** -8 * (dw.double() * u.double()).abs().sum().item() + 2.0 ** -20 * 40 * size
    (only,) = torch.autograd.grad(combine_rows(y, plan), y, dout)
    assert torch.equal(only, hip_combine_rows_backward(dout, None, plan)[0])


def test_plans_of_any_content(dev):
    """Places out of range add nothing and are not written; no call reads or writes past its rows."""
    from convrot_mlx_amd import ExpertPlan, hip_combine_rows, hip_combine_rows_backward

    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    plan = ExpertPlan(i32(0, 4), i32(0, 1, 2, 3), i32(0, 7, -3, 3).view(2, 2))
    y, w = normal(1, 4, 40).to(dev), normal(2, 2, 2).to(dev)
    out = hip_combine_rows(y, plan, w)
    assert torch.allclose(out[0], w[0, 0] * y[0]) and torch.allclose(out[1], w[1, 1] * y[3])
    _, dw = hip_combine_rows_backward(out, y, plan, w)
    assert dw[0, 1] == 0 and dw[1, 0] == 0


# ------------------------------------------------------------------ the products in 8-bit floating point


def fp8_weight(seed, experts, n, k, dev):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn((experts, n, k), generator=g) * 60).clamp(-448, 448).to(FP8)
    ws = torch.rand((experts, (n + 127) // 128, (k + 127) // 128), generator=g) * 1e-3 + 1e-5
    return q.to(dev), ws.to(dev)


GROUPS = [(1, 1, 1, 16, 16), (3, 2, 5, 70, 144), (8, 2, 16, 256, 512), (40, 1, 3, 130, 128), (64, 4, 70, 96, 256),
          (129, 2, 4, 300, 400), (700, 1, 2, 264, 272), (300, 3, 9, 515, 1040), (16, 2, 300, 64, 128)]


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,choices,experts,n,k", GROUPS)
def test_fp8_products(dev, tokens, choices, experts, n, k, dtype, gather):
    from convrot_mlx_amd import expert_plan, hip_fp8_grouped_linear

    ids = choose(n, tokens, choices, experts)
    plan = expert_plan(ids.to(dev), experts)
    q, ws = fp8_weight(n, experts, n, k, dev)
    x = normal(k, tokens if gather else tokens * choices, k).to(dtype)
    got = hip_fp8_grouped_linear(x.to(dev), q, ws, plan, gather=gather)
    assert got.dtype == dtype and got.shape == (tokens * choices, n)
    values = plain.row_values(*plain.codes(x)).to(dev)
    if gather:
        values = values[plan.order.long() // choices]
    at = plan.offsets.tolist()
    for e in range(experts):
        rows = slice(at[e], at[e + 1])
        if at[e] == at[e + 1]:
            continue
        want, spread = plain.product(values[rows], plain.weight_values(q[e], ws[e]), dtype == F32)
        assert_within(got[rows], want, spread, f"expert {e}")
    assert not got[at[-1]:].any()


@pytest.mark.parametrize("tile", ["256x256", "256x128", "128x128", "64x128", "32x64"])
def test_fp8_every_tile(dev, tuning, tile):
    from convrot_mlx_amd import expert_plan, hip_fp8_grouped_linear

    tuning.set("fp8_tile", tile)
    for gather in (False, True):
        tokens, choices, experts, n, k = 500, 2, 5, 270, 400
        plan = expert_plan(choose(7, tokens, choices, experts).to(dev), experts)
        q, ws = fp8_weight(n, experts, n, k, dev)
        x = normal(k, tokens if gather else tokens * choices, k).to(BF16)
        got = hip_fp8_grouped_linear(x.to(dev), q, ws, plan, gather=gather)
        values = plain.row_values(*plain.codes(x)).to(dev)
        values = values[plan.order.long() // choices] if gather else values
        at = plan.offsets.tolist()
        for e in range(experts):
            want, spread = plain.product(values[at[e]: at[e + 1]], plain.weight_values(q[e], ws[e]), False)
            assert_within(got[at[e]: at[e + 1]], want, spread, f"{tile} expert {e}")
        assert not got[at[-1]:].any()


def test_fp8_operands_of_other_layouts(dev):
    from convrot_mlx_amd import ExpertPlan, expert_plan, hip_fp8_grouped_linear

    plan = expert_plan(choose(3, 30, 2, 4).to(dev), 4)
    for k in (128, 40):
        q, ws = fp8_weight(1, 4, 72, k, dev)
        x = normal(2, 60, k).to(BF16).to(dev)
        want = hip_fp8_grouped_linear(x, q, ws, plan)
        bits = q.view(torch.uint8)
        for other in (torch.cat([bits, bits], 2)[..., :k], torch.cat([bits, bits], 1)[:, :72], bits.transpose(0, 1).contiguous().transpose(0, 1),
                      bits.transpose(1, 2).contiguous().transpose(1, 2)):
            assert torch.equal(hip_fp8_grouped_linear(x, other.view(FP8), ws, plan), want)
        assert torch.equal(hip_fp8_grouped_linear(x, q, ws.transpose(1, 2).contiguous().transpose(1, 2), plan), want)
        assert torch.equal(hip_fp8_grouped_linear(torch.cat([x, x], 1)[:, k:], q, ws, ExpertPlan(plan.offsets)), want)
        one = hip_fp8_grouped_linear(x, q[2:3], ws[2:3], ExpertPlan(torch.tensor([0, 60], dtype=torch.int32, device=dev)))
        at = plan.offsets.tolist()
        assert torch.equal(one[at[2]: at[3]], want[at[2]: at[3]])


def test_fp8_offsets_and_indices_of_any_content(dev):
    """Offsets out of range or order, and indices out of range, stay within the call's memory."""
    from convrot_mlx_amd import ExpertPlan, hip_fp8_grouped_linear

    q, ws = fp8_weight(1, 3, 40, 128, dev)
    x = normal(2, 50, 128).to(BF16).to(dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    for offsets in (i32(-5, 10, 2 ** 31 - 1, 60), i32(0, 50, 10, 20), i32(7, -1, -1, 50), i32(0, 0, 0, 0)):
        assert hip_fp8_grouped_linear(x, q, ws, ExpertPlan(offsets)).shape == (50, 40)
    assert not hip_fp8_grouped_linear(x, q, ws, ExpertPlan(i32(0, 0, 0, 0))).any()
    order = torch.arange(100, dtype=torch.int32, device=dev)
    order[3], order[40], order[99] = -1, 2 ** 31 - 1, 100
    got = hip_fp8_grouped_linear(x, q, ws, ExpertPlan(i32(0, 30, 60, 100), order), gather=True)
    good = torch.arange(100, dtype=torch.int32, device=dev)
    want = hip_fp8_grouped_linear(x, q, ws, ExpertPlan(i32(0, 30, 60, 100), good), gather=True)
    bad = [3, 40, 99]
    assert not got[bad].any()
    keep = [i for i in range(100) if i not in bad]
    assert torch.equal(got[keep], want[keep])


def test_no_rows(dev):
    from convrot_mlx_amd import expert_plan, hip_combine_rows, hip_combine_rows_backward, hip_fp8_grouped_linear

    q, ws = fp8_weight(1, 3, 40, 128, dev)
    plan = expert_plan(torch.zeros((0, 2), dtype=torch.int64, device=dev), 3)
    assert plan.offsets.tolist() == [0, 0, 0, 0]
    x = torch.zeros((0, 128), dtype=BF16, device=dev)
    for gather in (False, True):
        assert hip_fp8_grouped_linear(x, q, ws, plan, gather=gather).shape == (0, 40)
    assert hip_combine_rows(x, plan).shape == (0, 128)
    assert hip_combine_rows_backward(x, None, plan)[0].shape == (0, 128)


def test_fp8_rows_past_32_bits(dev):
    """Tokens whose codes pass 4 GiB: gathered rows are copied first."""
    from convrot_mlx_amd import ExpertPlan, hip_fp8_grouped_linear

    k, tokens = 8192, (1 << 19) + 100
    q, ws = fp8_weight(1, 2, 32, k, dev)
    x = torch.zeros((tokens, k), dtype=BF16, device=dev)
    rows = [0, 5, tokens // 2, 1 << 19, tokens - 1]
    some = normal(2, len(rows), k).to(BF16)
    x[rows] = some.to(dev)
    order = torch.arange(tokens - 1, -1, -1, dtype=torch.int32, device=dev)
    offsets = torch.tensor([0, tokens // 3, tokens], dtype=torch.int32, device=dev)
    values = plain.row_values(*plain.codes(some)).to(dev)
    for gather in (True, False):
        got = hip_fp8_grouped_linear(x, q, ws, ExpertPlan(offsets, order), gather=gather)
        for row, v in zip(rows, values):
            at = tokens - 1 - row if gather else row
            e = int(at >= tokens // 3)
            want, spread = plain.product(v[None], plain.weight_values(q[e], ws[e]), False)
            assert_within(got[at][None], want, spread)
        assert int(got.any(1).sum()) == len(rows)
