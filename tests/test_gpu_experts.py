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


@pytest.mark.parametrize("tile", ["256x256", "128x128", "64x128", "64x64", "32x64"])
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


@pytest.mark.parametrize("tokens,n", [(2500, 2000), (2500, 7690), (300, 1000)])
def test_fp8_last_round_in_parts(dev, tuning, tokens, n):
    """Large tiles whose last round runs as halves (80 of 256 CUs; 341, 85 past a round) and as quarters."""
    from convrot_mlx_amd import expert_plan, hip_fp8_grouped_linear, hip_fp8_linear

    tuning.set("fp8_tile", "256x256")
    experts, k = 2, 272
    plan = expert_plan(choose(n, tokens, 1, experts).to(dev), experts)
    q, ws = fp8_weight(n, experts, n, k, dev)
    x = normal(n, tokens, k).to(BF16)
    values = plain.row_values(*plain.codes(x)).to(dev)
    assert_within(hip_fp8_linear(x.to(dev), q[1], ws[1]), *plain.product(values, plain.weight_values(q[1], ws[1]), False))
    for gather in (False, True):
        got = hip_fp8_grouped_linear(x.to(dev), q, ws, plan, gather=gather)
        rows = values[plan.order.long()] if gather else values
        at = plan.offsets.tolist()
        for e in range(experts):
            want, spread = plain.product(rows[at[e]: at[e + 1]], plain.weight_values(q[e], ws[e]), False)
            assert_within(got[at[e]: at[e + 1]], want, spread, f"expert {e}")
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


# ------------------------------------------------------------------ the products in 16 bits


def product16(a, b, length):
    """a [M, C] b [N, C]^T in 64 bits, and what float32 sums may add: a chain of at most `length` additions."""
    return a @ b.t().contiguous(), U * (length + 8) * (a.abs() @ b.abs().t().contiguous())


GROUPS16 = [(1, 1, 1, 8, 8), (3, 2, 5, 70, 144), (8, 2, 16, 256, 512), (40, 1, 3, 130, 61), (64, 4, 70, 96, 256),
            (129, 2, 4, 300, 400), (700, 1, 2, 264, 72), (300, 3, 9, 515, 333), (16, 2, 300, 64, 136), (600, 2, 2, 520, 264)]


def check_products(dev, tokens, choices, experts, n, k, dtype, gather, seed=0):
    from convrot_mlx_amd import expert_plan, hip_grouped_linear, hip_grouped_linear_backward

    ids = choose(n + seed, tokens, choices, experts)
    plan = expert_plan(ids.to(dev), experts)
    w = normal(n, experts, n, k).to(dtype).to(dev)
    x = normal(k, tokens if gather else tokens * choices, k).to(dtype).to(dev)
    dy = normal(k + 1, tokens * choices, n).to(dtype).to(dev)
    at = plan.offsets.tolist()
    dy[at[-1]:] = float("nan")  # rows of no expert reach nothing but themselves
    got = hip_grouped_linear(x, w, plan, gather=gather)
    dx, dw = hip_grouped_linear_backward(dy, x, w, plan, gather=gather)
    assert got.dtype == dtype and got.shape == (tokens * choices, n) and dx.shape == x.shape and dw.shape == w.shape
    rows = (x[plan.order.long() // choices] if gather else x).double()
    want_dx, off_dx = torch.zeros((tokens * choices, k), dtype=torch.float64, device=dev), torch.zeros((tokens * choices, k), dtype=torch.float64, device=dev)
    for e in range(experts):
        r = slice(at[e], at[e + 1])
        we, g = w[e].double(), dy[r].double()
        if at[e + 1] == at[e]:
            assert not dw[e].any()
            continue
        assert_within(got[r], *product16(rows[r], we, k), f"forward {e}")
        want_dx[r], off_dx[r] = product16(g, we.t().contiguous(), n)
        count = at[e + 1] - at[e]
        assert_within(dw[e], *product16(g.t().contiguous(), rows[r].t().contiguous(), count), f"weights {e}")
    assert not got[at[-1]:].any()
    if gather:  # each choice's gradient is rounded, then they are added at float32
        slots = plan.slots.long()
        each, off = want_dx[slots], off_dx[slots]
        half = {BF16: 2.0 ** -8, F16: 2.0 ** -11}[dtype]
        tiny = {BF16: 2.0 ** -133, F16: 2.0 ** -25}[dtype]
        assert_within(dx, each.sum(1), (half * (each.abs() + off) + off + tiny).sum(1) + U * choices * each.abs().sum(1), "rows")
    else:
        assert_within(dx, want_dx, off_dx, "rows")
        assert not dx[at[-1]:].any()


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,choices,experts,n,k", GROUPS16)
def test_products(dev, tokens, choices, experts, n, k, dtype, gather):
    check_products(dev, tokens, choices, experts, n, k, dtype, gather)


@pytest.mark.parametrize("tile", ["256x256", "128x128", "64x128", "64x64", "32x128", "32x64"])
@pytest.mark.parametrize("tokens,choices,experts,n,k", [(500, 2, 5, 270, 400), (600, 1, 2, 520, 264), (30, 1, 4, 64, 64)])
def test_every_tile(dev, tuning, tile, tokens, choices, experts, n, k):
    tuning.set("grouped_tile", tile)
    for gather in (False, True):
        check_products(dev, tokens, choices, experts, n, k, BF16, gather, seed=1)


@pytest.mark.parametrize("tile", [None, "256x256", "128x128"])
@pytest.mark.parametrize("tokens,choices", [(200, 5), (150, 7), (20, 64), (333, 3), (1, 1)])
def test_rows_read_through_the_index(dev, tuning, tile, tokens, choices):
    """Every number of choices a token: the rows of a block of the weights' gradient come through the index."""
    if tile:
        tuning.set("grouped_tile", tile)
    check_products(dev, tokens, choices, 4, 136, 264, BF16, True, seed=3)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("n,k", [(2000, 1960), (264, 7690), (7690, 264)])
def test_last_round_in_parts(dev, tuning, n, k, gather):
    """Large tiles whose last round runs as halves (80 to 128 of 256 CUs, behind a whole round of 256 too) or as
    quarters, of outputs and of both gradients."""
    tuning.set("grouped_tile", "256x256")
    check_products(dev, 1250, 2, 2, n, k, BF16, gather)


def test_operands_of_other_layouts(dev):
    from convrot_mlx_amd import ExpertPlan, expert_plan, hip_grouped_linear, hip_grouped_linear_backward

    plan = expert_plan(choose(3, 30, 2, 4).to(dev), 4)
    for n, k in ((72, 128), (33, 41)):
        w, x, dy = (normal(i, *s).to(F16).to(dev) for i, s in enumerate(((4, n, k), (60, k), (60, n))))
        want = hip_grouped_linear(x, w, plan)
        dx, dw = hip_grouped_linear_backward(dy, x, w, plan)
        for other in (torch.cat([w, w], 2)[..., :k], torch.cat([w, w], 1)[:, :n], w.transpose(0, 1).contiguous().transpose(0, 1),
                      w.transpose(1, 2).contiguous().transpose(1, 2)):
            assert torch.equal(hip_grouped_linear(x, other, plan), want)
            got = hip_grouped_linear_backward(dy, x, other, plan)
            assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
        for view in (lambda t: torch.cat([t, t], 1)[:, t.shape[1]:], lambda t: t.t().contiguous().t(),
                     lambda t: torch.cat([t.flatten(), t.flatten()])[t.numel():].view(t.shape)):
            assert torch.equal(hip_grouped_linear(view(x), w, ExpertPlan(plan.offsets)), want)
            got = hip_grouped_linear_backward(view(dy), view(x), w, plan)
            assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
        one = hip_grouped_linear_backward(dy, x, w, plan, rows_grad=False)
        assert one[0] is None and torch.equal(one[1], dw)
        one = hip_grouped_linear_backward(dy, x, w, plan, weight_grad=False)
        assert one[1] is None and torch.equal(one[0], dx)
        same = w[:1].expand(4, -1, -1)  # one weight for all: experts 0 elements apart
        assert torch.equal(hip_grouped_linear(x, same, plan), hip_grouped_linear(x, same.contiguous(), plan))


def test_not_finite_rows(dev):
    """A row's NaN or infinity reaches its own outputs, its own gradient and its expert's weight gradient alone."""
    from convrot_mlx_amd import ExpertPlan, hip_grouped_linear, hip_grouped_linear_backward

    offsets = torch.tensor([0, 37, 37, 100], dtype=torch.int32, device=dev)
    plan = ExpertPlan(offsets)
    w, x, dy = (normal(i, *s).to(BF16).to(dev) for i, s in enumerate(((3, 72, 136), (120, 136), (120, 72))))
    want = hip_grouped_linear(x, w, plan), *hip_grouped_linear_backward(dy, x, w, plan)
    x[36, 5], x[110], dy[36, 3], dy[119] = float("nan"), float("inf"), float("inf"), float("nan")
    got = hip_grouped_linear(x, w, plan), *hip_grouped_linear_backward(dy, x, w, plan)
    keep = [i for i in range(120) if i != 36]
    for a, b in zip(got[:2], want[:2]):
        assert torch.equal(a[keep], b[keep]) and not torch.isfinite(a[36]).any()
    assert torch.equal(got[2][1:], want[2][1:]) and got[2][0].isnan().any()


def test_offsets_and_indices_of_any_content(dev):
    from convrot_mlx_amd import ExpertPlan, hip_grouped_linear, hip_grouped_linear_backward

    w, x, dy = (normal(i, *s).to(BF16).to(dev) for i, s in enumerate(((3, 40, 128), (50, 128), (50, 40))))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    for offsets in (i32(-5, 10, 2 ** 31 - 1, 60), i32(0, 50, 10, 20), i32(7, -1, -1, 50), i32(0, 0, 0, 0)):
        plan = ExpertPlan(offsets)
        assert hip_grouped_linear(x, w, plan).shape == (50, 40)
        dx, dw = hip_grouped_linear_backward(dy, x, w, plan)
        assert dx.shape == x.shape and dw.shape == w.shape
    assert not hip_grouped_linear(x, w, plan).any() and not dx.any() and not dw.any()
    order = torch.arange(100, dtype=torch.int32, device=dev)
    order[3], order[40], order[99] = -1, 2 ** 31 - 1, 100
    got = hip_grouped_linear(x, w, ExpertPlan(i32(0, 30, 60, 100), order), gather=True)
    want = hip_grouped_linear(x, w, ExpertPlan(i32(0, 30, 60, 100), torch.arange(100, dtype=torch.int32, device=dev)), gather=True)
    keep = [i for i in range(100) if i not in (3, 40, 99)]
    assert torch.equal(got[keep], want[keep]) and not got[[3, 40, 99]].any()


def test_gradient_of_weights_with_indices_out_of_range(dev):
    from convrot_mlx_amd import ExpertPlan, hip_grouped_linear_backward

    w, x, dy = (normal(i, *s).to(BF16).to(dev) for i, s in enumerate(((3, 40, 128), (50, 128), (100, 40))))
    offsets = torch.tensor((0, 30, 60, 100), dtype=torch.int32, device=dev)
    order = torch.randperm(100, generator=torch.Generator().manual_seed(5)).int().to(dev)
    without = dy.clone()
    without[[3, 40, 99]] = 0
    _, want = hip_grouped_linear_backward(without, x, w, ExpertPlan(offsets, order), gather=True, rows_grad=False)
    order[3], order[40], order[99] = -1, 2 ** 31 - 1, 100
    _, got = hip_grouped_linear_backward(dy, x, w, ExpertPlan(offsets, order), gather=True, rows_grad=False)
    assert torch.equal(got, want)


def test_no_rows_in_16_bits(dev):
    from convrot_mlx_amd import expert_plan, hip_grouped_linear, hip_grouped_linear_backward

    plan = expert_plan(torch.zeros((0, 2), dtype=torch.int32, device=dev), 3)
    w, x = torch.ones((3, 40, 24), dtype=BF16, device=dev), torch.zeros((0, 24), dtype=BF16, device=dev)
    for gather in (False, True):
        assert hip_grouped_linear(x, w, plan, gather=gather).shape == (0, 40)
        dx, dw = hip_grouped_linear_backward(torch.zeros((0, 40), dtype=BF16, device=dev), x, w, plan, gather=gather)
        assert dx.shape == (0, 24) and dw.shape == w.shape and not dw.any()


def test_rows_past_32_bits(dev):
    """Tokens, sorted rows and gradients past 4 GiB."""
    from convrot_mlx_amd import ExpertPlan, hip_grouped_linear, hip_grouped_linear_backward

    k, tokens = 4096, (1 << 19) + 100
    w = normal(1, 2, 32, k, std=0.05).to(BF16).to(dev)
    x = torch.zeros((tokens, k), dtype=BF16, device=dev)
    dy = torch.zeros((tokens, 32), dtype=BF16, device=dev)
    rows = [0, 5, tokens // 2, 1 << 19, tokens - 1]
    some, g = normal(2, len(rows), k).to(BF16).to(dev), normal(3, len(rows), 32).to(BF16).to(dev)
    x[rows], dy[rows] = some, g
    order = torch.arange(tokens - 1, -1, -1, dtype=torch.int32, device=dev)
    third = tokens // 3
    plan = ExpertPlan(torch.tensor([0, third, tokens], dtype=torch.int32, device=dev), order)
    for gather in (True, False):
        got = hip_grouped_linear(x, w, plan, gather=gather)
        for row, v in zip(rows, some):
            at = tokens - 1 - row if gather else row
            assert_within(got[at][None], *product16(v[None].double(), w[int(at >= third)].double(), k))
        assert int(got.any(1).sum()) == len(rows)
    dx, dw = hip_grouped_linear_backward(dy, x, w, plan)
    for e in range(2):
        mine = [i for i, r in enumerate(rows) if int(r >= third) == e]
        assert_within(dw[e], *product16(g[mine].double().t().contiguous(), some[mine].double().t().contiguous(), len(rows)))
        assert_within(dx[[rows[i] for i in mine]], *product16(g[mine].double(), w[e].double().t().contiguous(), 32))
    assert int(dx.any(1).sum()) == len(rows)


# ------------------------------------------------------------------ together


def mixture(x, ids, weights, up, down):
    """A mixture's feed-forward layer on rows x [T, K]: up and down are called on sorted rows."""
    from convrot_mlx_amd import combine_rows, expert_plan

    plan = expert_plan(ids, up.experts)
    h = up(x, plan, gather=True)
    return combine_rows(down(torch.nn.functional.silu(h), plan), plan, weights)


def layers(dev, experts, k, hidden, dtype=BF16):
    from convrot_mlx_amd import ExpertLinear

    torch.manual_seed(0)
    up, down = ExpertLinear(experts, k, hidden, device=dev, dtype=dtype), ExpertLinear(experts, hidden, k, device=dev, dtype=dtype)
    up.experts = experts
    return up, down


@pytest.mark.parametrize("tokens", [1, 37, 300])
def test_a_mixture_and_its_gradients(dev, tokens):
    """The layer as a user builds it, against the same in 64 bits, and its gradients against the formula's there.
    Every 16-bit tensor between the products is off by at most half a unit (2^-9 of its value, bf16): the
    relative errors of h, silu(h), the rows, and (backward) three more roundings add up."""
    k, hidden, experts, choices = 136, 264, 6, 2
    up, down = layers(dev, experts, k, hidden)
    ids = choose(tokens, tokens, choices, experts).to(dev)
    x = normal(1, tokens, k).to(BF16).to(dev).requires_grad_()
    wts = torch.rand((tokens, choices), generator=torch.Generator().manual_seed(2)).to(dev).requires_grad_()
    out = mixture(x, ids, wts, up, down)
    dout = normal(3, tokens, k).to(BF16).to(dev)
    leaves = (x, wts, up.weight, down.weight)
    grads = torch.autograd.grad(out, leaves, dout)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    xd, wd, ud, dd = wide
    ref = torch.zeros((tokens, k), dtype=torch.float64, device=dev)
    for e in range(experts):
        for c in range(choices):
            at = (ids[:, c] == e).nonzero()[:, 0]
            if len(at):
                h = torch.nn.functional.silu(xd[at] @ ud[e].t().contiguous())
                ref = ref.index_add(0, at, wd[at, c, None] * (h @ dd[e].t().contiguous()))
    want = torch.autograd.grad(ref, wide, dout.double(), allow_unused=True)
    for got, w in zip((out, *grads), (ref.detach(), *want)):
        w = torch.zeros_like(got, dtype=torch.float64) if w is None else w
        off = (got.detach().double() - w).norm() / w.norm().clamp_min(1e-30)
        assert off <= 8 * 2.0 ** -8, off  # at most eight roundings of half a unit each, in any of these tensors


def test_a_mixture_at_8_bits(dev):
    """The same layer with its experts quantized: the layer's own calls, and near the 16-bit one."""
    from convrot_mlx_amd import Fp8ExpertLinear, combine_rows, expert_plan, hip_fp8_grouped_linear

    k, hidden, experts, tokens = 256, 384, 5, 70
    up, down = layers(dev, experts, k, hidden)
    ids = choose(5, tokens, 2, experts).to(dev)
    x, wts = normal(1, tokens, k).to(BF16).to(dev), torch.rand((tokens, 2), device=dev)
    q_up = Fp8ExpertLinear(experts, k, hidden, device=dev).load_weight(up.weight.detach())
    q_down = Fp8ExpertLinear(experts, hidden, k, device=dev).load_weight(down.weight.detach())
    q_up.experts = experts
    got = mixture(x, ids, wts, q_up, q_down)
    plan = expert_plan(ids, experts)
    h = hip_fp8_grouped_linear(x, q_up.qweight, q_up.scales, plan, gather=True)
    y = hip_fp8_grouped_linear(torch.nn.functional.silu(h), q_down.qweight, q_down.scales, plan)
    assert torch.equal(got, combine_rows(y, plan, wts))
    near = mixture(x, ids, wts, up, down).detach().double()
    # codes are off by 2^-4 of a value at most: two operands of each of two products
    assert (got.double() - near).norm() <= 4 * 2.0 ** -4 * near.norm()
    moved = torch.nn.ModuleList([q_up]).half()[0]
    assert moved.qweight.dtype == FP8 and moved.scales.dtype == F32
    with pytest.raises(RuntimeError, match="has no gradient"):
        q_up(x.requires_grad_(), plan, gather=True).sum().backward()


def test_a_mixture_in_graphs(dev):
    """Forward and backward captured and replayed, on new inputs in the same memory, beside eager calls and on
    another stream."""
    from convrot_mlx_amd import Fp8ExpertLinear

    k, hidden, experts, tokens = 136, 264, 6, 4200
    up, down = layers(dev, experts, k, hidden)
    q_up = Fp8ExpertLinear(experts, k, hidden, device=dev).load_weight(up.weight.detach())
    q_down = Fp8ExpertLinear(experts, hidden, k, device=dev).load_weight(down.weight.detach())
    q_up.experts = experts
    x, ids = normal(1, tokens, k).to(BF16).to(dev).requires_grad_(), choose(2, tokens, 2, experts).to(dev)
    wts, dout = torch.rand((tokens, 2), device=dev).requires_grad_(), normal(3, tokens, k).to(BF16).to(dev)

    def train():
        out = mixture(x, ids, wts, up, down)
        return [out.detach(), *torch.autograd.grad(out, (x, wts, up.weight, down.weight), dout)]

    def serve():
        with torch.no_grad():
            return [mixture(x, ids, wts, q_up, q_down)]

    side = torch.cuda.Stream()
    for step in (train, serve):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
        for i in range(4):
            with torch.no_grad():
                x.copy_(normal(10 + i, tokens, k))
                ids.copy_(choose(10 + i, tokens, 2, experts))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(held, step()):
                assert torch.equal(a, b)


def test_gradients_against_differences(dev):
    """The product is linear in the rows and in the weights: a difference along a direction is the gradient's
    product with it, up to the roundings of the outputs."""
    from convrot_mlx_amd import expert_plan, grouped_linear

    plan = expert_plan(choose(4, 50, 2, 3).to(dev), 3)
    w, x, dy = (normal(i, *s).to(F16).to(dev) for i, s in enumerate(((3, 40, 72), (50, 72), (100, 40))))
    dy[int(plan.offsets[-1]):] = 0
    wg, xg = w.clone().requires_grad_(), x.clone().requires_grad_()
    dx, dw = torch.autograd.grad(grouped_linear(xg, wg, plan, gather=True), (xg, wg), dy)
    for t, grad, call in ((x, dx, lambda v: grouped_linear(v, w, plan, gather=True)), (w, dw, lambda v: grouped_linear(x, v, plan, gather=True))):
        v = torch.randint(-1, 2, t.shape, generator=torch.Generator().manual_seed(9)).to(F16).to(dev)
        a, b = call(t + v).double(), call(t - v).double()  # t and v: sums within half a unit of float16
        slope = ((a - b) / 2 * dy.double()).sum()
        want = (grad.double() * v.double()).sum()
        size = ((a.abs() + b.abs()) * dy.double().abs()).sum()
        # the outputs' roundings; the gradient's; and those of t + v and t - v, through the gradient
        bound = size + (grad.double() * v.double()).abs().sum() + 2 * (grad.double().abs() * (t.double().abs() + 1)).sum()
        assert abs(slope - want) <= 2.0 ** -11 * bound
