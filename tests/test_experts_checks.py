"""CPU: what the linears of a mixture of experts and what lies around them refuse before any launch."""

from __future__ import annotations

import pytest
import torch

from convrot_mlx_amd import (ExpertLinear, ExpertPlan, Fp8ExpertLinear, combine_rows, expert_plan, grouped_linear,
                             hip_combine_rows, hip_combine_rows_backward, hip_fp8_grouped_linear, hip_grouped_linear,
                             hip_grouped_linear_backward)

P = 4096  # stands for any 16-byte aligned device address: never read
F16, BF16, F32 = 1, 2, 0
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    from convrot_mlx_amd import _native

    return _native.load()


def refused(lib, status, code, text):
    assert status == code, lib.convrot_last_error()
    assert text in lib.convrot_last_error().decode()


GROUPS = [
    (dict(experts=0), 2, "1 to 65536 experts"), (dict(experts=65537), 2, "1 to 65536 experts"), (dict(offsets=None), 1, "null"),
    (dict(offsets=P + 2), 1, "aligned"), (dict(index=P + 1), 1, "aligned"), (dict(choices=0), 1, "invalid groups"),
    (dict(index=None), 1, "sorted rows, but"), (dict(weight=None), 1, "null"), (dict(weight=P + 8), 1, "aligned"),
    (dict(ldw=56), 1, "rows that cover"), (dict(expert=-64), 1, "16-byte aligned"), (dict(expert=516), 1, "16-byte aligned"),
    (dict(out=P + 8), 1, "aligned"), (dict(k=0), 1, "invalid"), (dict(rows=-1), 1, "invalid"), (dict(k=65544, ldx=65544), 2, ""),
]


def grouped(lib, **kw):
    a = dict(x=P, dtype=BF16, xrows=4, ldx=64, weight=P, ldw=64, expert=512, offsets=P, experts=3, index=P, choices=2, rows=8,
             n=8, k=64, out=P) | kw
    return lib.convrot_grouped_linear(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", GROUPS + [
    (dict(dtype=F32), 1, "float16 or bfloat16"), (dict(dtype=5), 1, "float16 or bfloat16"), (dict(n=0), 1, "invalid"),
    (dict(n=65537), 2, "up to 65536 features"), (dict(x=None), 1, "null"), (dict(x=P + 2), 1, "16-byte aligned rows"),
    (dict(ldx=60), 1, "16-byte aligned rows"), (dict(ldx=1 << 22), 2, "limited"), (dict(out=None), 1, "aligned"),
    (dict(xrows=0), 2, "through an index"), (dict(xrows=1 << 26, rows=1 << 27), 2, "through an index"),
    (dict(rows=0x7fffff00), 2, "too large"),
])
def test_products_in_16_bits(lib, kw, code, text):
    refused(lib, grouped(lib, **kw), code, text)


def fp8(lib, **kw):
    a = dict(x=P, dtype=BF16, xrows=4, ldx=64, weight=P, ldw=64, expert=512, ws=P, wr=1, wse=1, offsets=P, experts=3, index=P,
             choices=2, rows=8, n=8, k=64, scratch=P, nbytes=1 << 20, out=P) | kw
    return lib.convrot_fp8_grouped_linear(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", GROUPS + [
    (dict(dtype=9), 1, "dtype code"), (dict(x=None), 1, "null"), (dict(ws=None), 1, "null"), (dict(wr=0), 1, "weight scales"),
    (dict(wse=-1), 1, "16-byte aligned"), (dict(scratch=None), 1, "scratch buffer"), (dict(nbytes=500), 1, "scratch buffer"),
    (dict(xrows=0), 2, "through an index"), (dict(xrows=1 << 26, rows=1 << 27, nbytes=1 << 40), 2, "through an index"),
])
def test_products_at_8_bits(lib, kw, code, text):
    refused(lib, fp8(lib, **kw), code, text)


def rows_grad(lib, **kw):
    a = dict(dy=P, dtype=BF16, ldy=8, weight=P, ldw=64, expert=512, offsets=P, experts=3, rows=8, n=8, k=64, out=P) | kw
    return lib.convrot_grouped_linear_rows_grad(*a.values(), None)


def weight_grad(lib, **kw):
    a = dict(dy=P, dtype=BF16, ldy=8, x=P, xrows=4, ldx=64, offsets=P, experts=3, index=P, choices=2, rows=8, n=8, k=64, out=P) | kw
    return lib.convrot_grouped_linear_weight_grad(*a.values(), None)


@pytest.mark.parametrize("call,kw,code,text", [
    (rows_grad, dict(dtype=F32), 1, "float16 or bfloat16"), (rows_grad, dict(dy=None), 1, "null"),
    (rows_grad, dict(ldy=4), 1, "dy needs"), (rows_grad, dict(weight=P + 4), 1, "weight needs"),
    (rows_grad, dict(expert=-8), 1, "16-byte aligned"), (rows_grad, dict(out=None), 1, "aligned"),
    (rows_grad, dict(offsets=None), 1, "null"), (rows_grad, dict(experts=0), 2, "experts"), (rows_grad, dict(n=0), 1, "invalid"),
    (weight_grad, dict(dtype=F32), 1, "float16 or bfloat16"), (weight_grad, dict(x=None), 1, "null"),
    (weight_grad, dict(ldx=56), 1, "x needs"), (weight_grad, dict(out=P + 2), 1, "dw must"), (weight_grad, dict(out=None), 1, "dw must"),
    (weight_grad, dict(rows=0, offsets=None), 1, "null"), (weight_grad, dict(index=None), 1, "sorted rows, but"),
    (weight_grad, dict(choices=0), 1, "invalid groups"), (weight_grad, dict(xrows=0), 2, "through an index"),
    (weight_grad, dict(xrows=1 << 26, rows=1 << 27), 2, "through an index"), (weight_grad, dict(k=70000), 2, "features"),
])
def test_gradients(lib, call, kw, code, text):
    refused(lib, call(lib, **kw), code, text)


def plan(lib, **kw):
    a = dict(ids=P, bits=64, count=64, experts=8, offsets=P, order=P, slots=P, work=None, nbytes=0) | kw
    return lib.convrot_expert_plan(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(bits=16), 1, "32 or 64 bits"), (dict(experts=0), 2, "1 to 1024 experts"), (dict(experts=1025), 2, "1 to 1024 experts"),
    (dict(count=-1), 2, "at most 2^31-1"), (dict(count=1 << 31), 2, "at most 2^31-1"), (dict(offsets=None), 1, "null"),
    (dict(ids=None), 1, "null"), (dict(order=None), 1, "null"), (dict(slots=None), 1, "null"), (dict(ids=P + 4), 1, "aligned"),
    (dict(slots=P + 2), 1, "aligned"), (dict(count=100000), 1, "workspace"), (dict(count=100000, work=P, nbytes=8), 1, "workspace"),
    (dict(count=100000, work=P + 2, nbytes=1 << 20), 1, "workspace"),
])
def test_order(lib, kw, code, text):
    refused(lib, plan(lib, **kw), code, text)


def test_workspace_of_the_order(lib):
    size = lib.convrot_expert_plan_workspace_bytes
    assert size(64, 8) == 0 and size(-1, 8) == 0 and size(1 << 20, 2000) == 0
    assert 0 < size(100000, 8) <= 64 * 9 * 4 and 0 < size((1 << 31) - 1, 1024) <= 64 * 1025 * 4


def gather(lib, **kw):
    a = dict(x=P, dtype=BF16, xrows=4, stride=64, index=P, choices=2, rows=8, k=64, out=P) | kw
    return lib.convrot_gather_rows(*a.values(), None)


def combine(lib, **kw):
    a = dict(y=P, dtype=BF16, yrows=8, stride=64, slots=P, weights=P, tokens=4, choices=2, k=64, out=P) | kw
    return lib.convrot_combine_rows(*a.values(), None)


def combine_backward(lib, **kw):
    a = dict(dout=P, stride=64, y=P, ystride=64, dtype=BF16, yrows=8, order=P, slots=P, weights=P, tokens=4, choices=2, k=64,
             dy=P, dw=P) | kw
    return lib.convrot_combine_rows_backward(*a.values(), None)


@pytest.mark.parametrize("call,kw,code,text", [
    (gather, dict(dtype=8), 1, "dtype code"), (gather, dict(rows=-1), 1, "invalid shape"), (gather, dict(choices=0), 1, "invalid shape"),
    (gather, dict(index=None), 1, "null"), (gather, dict(out=None), 1, "null"), (gather, dict(index=P + 2), 1, "aligned"),
    (gather, dict(out=P + 1), 1, "aligned"), (gather, dict(x=None), 1, "null"), (gather, dict(stride=-8), 1, "negative"),
    (combine, dict(dtype=8), 1, "dtype code"), (combine, dict(choices=0), 1, "invalid shape"), (combine, dict(tokens=-1), 1, "invalid shape"),
    (combine, dict(tokens=1 << 20, choices=1 << 20), 1, "invalid shape"), (combine, dict(slots=None), 1, "null"),
    (combine, dict(out=None), 1, "null"), (combine, dict(weights=P + 2), 1, "aligned"), (combine, dict(y=None), 1, "null"),
    (combine_backward, dict(dtype=8), 1, "dtype code"), (combine_backward, dict(yrows=7), 1, "7 rows for 8 choices"),
    (combine_backward, dict(y=None), 1, "null"), (combine_backward, dict(dout=None), 1, "null"), (combine_backward, dict(slots=None), 1, "null"),
    (combine_backward, dict(order=None), 1, "null"), (combine_backward, dict(dw=P + 2), 1, "aligned"),
    (combine_backward, dict(dy=P + 1), 1, "aligned"),
])
def test_rows(lib, call, kw, code, text):
    refused(lib, call(lib, **kw), code, text)


def test_nothing_to_do_is_no_error(lib):
    assert grouped(lib, rows=0, index=None, xrows=0, x=None) == 0 and rows_grad(lib, rows=0, dy=None) == 0
    assert fp8(lib, rows=0, index=None, xrows=0, x=None, scratch=None, nbytes=0) == 0 and fp8(lib, n=0) == 0
    assert gather(lib, rows=0, index=None) == 0 and gather(lib, k=0) == 0
    assert combine(lib, tokens=0, slots=None) == 0 and combine(lib, k=0, slots=None) == 0
    assert combine_backward(lib, tokens=0, yrows=0, slots=None) == 0 and combine_backward(lib, dy=None, dw=None, slots=None) == 0


def test_tuning_names(lib):
    assert lib.convrot_set_tuning(b"grouped_tile", b"32x128") == 0 and lib.convrot_set_tuning(b"grouped_tile", None) == 0
    refused(lib, lib.convrot_set_tuning(b"grouped_tile", b"16x16"), 1, "invalid value")


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


PLAN = ExpertPlan(ints(0, 2, 4), ints(0, 2, 1, 3), ints(0, 2, 1, 3).view(2, 2))


def f8(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(FP8)


@pytest.mark.parametrize("ids,experts", [(torch.zeros(2, 2), 2), (ints(0, 1).view(1, 1, 2), 2), (ints(0, 1).short(), 2),
                                         (ints(0, 1), 0), (ints(0, 1), 1025)])
def test_expert_numbers(ids, experts):
    with pytest.raises(ValueError):
        expert_plan(ids, experts)


@pytest.mark.parametrize("x,plan,gather,text", [
    (torch.zeros(4), PLAN, False, r"rows \[R, K\]|K="), (torch.zeros(1, 4, 16), PLAN, False, r"rows \[R, K\]"),
    (torch.zeros(5, 16), PLAN, False, "sorts 4 rows"), (torch.zeros(3, 16), PLAN, True, "no whole number"),
    (torch.zeros(0, 16), PLAN, True, "no whole number"), (torch.zeros(4, 16), ExpertPlan(ints(0, 4)), False, "orders rows by 1"),
    (torch.zeros(4, 16), ExpertPlan(ints(0, 2, 4).long()), False, "contiguous int32"),
    (torch.zeros(2, 16), ExpertPlan(ints(0, 2, 4)), True, "needs the plan's order"),
    (torch.zeros(4, 16), ExpertPlan(ints(0, 9, 2, 9, 4, 9)[::2]), False, "contiguous int32"),
])
def test_groups(x, plan, gather, text):
    w = torch.zeros(2, 8, 16, dtype=torch.bfloat16)
    for call in (hip_grouped_linear, grouped_linear):
        with pytest.raises(ValueError, match=text):
            call(x.bfloat16(), w, plan, gather=gather)
    with pytest.raises(ValueError, match=text):
        hip_fp8_grouped_linear(x, f8(2, 8, 16), torch.ones(2, 1, 1), plan, gather=gather)


def test_weights_of_products():
    x, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(2, 8, 16, dtype=torch.bfloat16)
    for bad, text in ((w.half(), "must be torch.bfloat16"), (w[0], "must be torch.bfloat16"), (w[:, :, :8], "take K=8"),
                      (w[:, :0], "1 to 65536 features")):
        with pytest.raises(ValueError, match=text):
            hip_grouped_linear(x, bad, PLAN)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        hip_grouped_linear(x.float(), w.float(), PLAN)
    for dy in (torch.zeros(4, 7, dtype=torch.bfloat16), torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(4, 8)):
        with pytest.raises(ValueError, match="dy must be"):
            hip_grouped_linear_backward(dy, x, w, PLAN)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hip_grouped_linear(x, w, PLAN)
    for q, ws, text in ((w, torch.ones(2, 1, 1), "3D float8_e4m3fn"), (f8(8, 16), torch.ones(1, 1), "3D float8_e4m3fn"),
                        (f8(2, 8, 8), torch.ones(2, 1, 1), "K=16"), (f8(2, 8, 16), torch.ones(1, 1), "scales must have shape")):
        with pytest.raises(ValueError, match=text):
            hip_fp8_grouped_linear(x, q, ws, PLAN)
    with pytest.raises(ValueError, match="unsupported dtype"):
        hip_fp8_grouped_linear(x.double(), f8(2, 8, 16), torch.ones(2, 1, 1), PLAN)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hip_fp8_grouped_linear(x, f8(2, 8, 16), torch.ones(2, 1, 1), PLAN)


def test_rows_summed_back():
    y = torch.zeros(4, 6)
    for rows, plan, weights, text in (
            (y, ExpertPlan(PLAN.offsets), None, "needs the plan's slots"), (y[:3], PLAN, None, "the 4 sorted rows"),
            (torch.zeros(4), PLAN, None, "the 4 sorted rows"), (y, PLAN, torch.ones(4), "weights must be floating point"),
            (y, PLAN, torch.ones(2, 2, dtype=torch.int32), "weights must be floating point"), (y.double(), PLAN, None, "unsupported dtype"),
            (y, PLAN._replace(order=ints(0, 1)), None, "sorted rows"), (y, PLAN._replace(slots=PLAN.slots.view(4)), None, "with 2 axes")):
        for call in (hip_combine_rows, combine_rows):
            with pytest.raises(ValueError, match=text):
                call(rows, plan, weights)
    for dout, rows, weights, text in ((torch.zeros(3, 6), y, None, "a row for each of 2 tokens"), (torch.zeros(2, 5), y, torch.ones(2, 2), "must match rows"),
                                      (torch.zeros(2, 6).half(), y, torch.ones(2, 2), "must match rows")):
        with pytest.raises(ValueError, match=text):
            hip_combine_rows_backward(dout, rows, PLAN, weights)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hip_combine_rows(y, PLAN)


def test_layers():
    layer = Fp8ExpertLinear(2, 16, 8)
    with pytest.raises(ValueError, match="weight must have shape"):
        layer.load_weight(torch.zeros(2, 8, 15))
    with pytest.raises(ValueError, match="K=15"):
        layer(torch.zeros(4, 15), PLAN)
    layer.half()
    assert layer.qweight.dtype == FP8 and layer.scales.dtype == torch.float32 and "experts=2" in repr(layer)
    dense = ExpertLinear(2, 16, 8, dtype=torch.float16)
    assert dense.weight.shape == (2, 8, 16) and dense.weight.dtype == torch.float16 and 0 < dense.weight.abs().max() <= 0.25
    with pytest.raises(ValueError, match="take K=16"):
        dense(torch.zeros(4, 15, dtype=torch.float16), PLAN)
