"""The linears of a mixture of experts: the order of the tokens' choices by expert, the products of each
expert's rows with its weight (16 bits with gradients, or 8-bit floating point), and the rows summed back.

    plan = expert_plan(ids, experts)                        # ids [T, C]: each token's experts
    h = grouped_linear(x, w_up, plan, gather=True)           # [T C, N]: rows sorted by expert, read from x [T, K]
    y = grouped_linear(activation(h), w_down, plan)          # [T C, K]
    out = combine_rows(y, plan, weights)                     # [T, K] = sum over c of weights[t, c] * row

Choices outside 0 .. experts - 1 (dropped ones) go behind the last expert's rows; their products are zeros.
No counterpart in the reference, whose model is dense.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from .fp8 import _check_weight, _operand, _row_stride, _weight_scales
from .norm import rows_of

MAX_PLAN_EXPERTS = 1024
MAX_EXPERTS = 65536
MAX_GATHERED_BYTES = (1 << 32) - 4096


class ExpertPlan(NamedTuple):
    """Sorted rows by expert, int32 on the device: expert e has rows offsets[e] .. offsets[e + 1] - 1
    (offsets [E + 1], from 0), row s is choice order[s] (token order[s] // C, order [T C]), and choice
    (t, c) is row slots[t, c].  order and slots may be None for rows that a caller sorted itself."""

    offsets: torch.Tensor
    order: torch.Tensor | None = None
    slots: torch.Tensor | None = None


def expert_plan(ids: torch.Tensor, experts: int) -> ExpertPlan:
    """The stable order of choices ids [T, C] or [T] (int32 or int64) by expert."""
    if ids.ndim not in (1, 2) or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"expert numbers must be int32 or int64 [tokens, choices], got {ids.dtype} {tuple(ids.shape)}")
    if not 1 <= experts <= MAX_PLAN_EXPERTS:
        raise ValueError(f"expert_plan supports 1 to {MAX_PLAN_EXPERTS} experts, got {experts}")
    device = nat.require_device(ids)
    ids = ids.contiguous()
    count = ids.numel()
    lib = nat.load()
    offsets = torch.empty((experts + 1,), dtype=torch.int32, device=device)
    places = torch.empty((2, count), dtype=torch.int32, device=device)
    order, slots = places[0], places[1].view(ids.shape if ids.ndim == 2 else (count, 1))
    with nat.on(device):
        need = lib.convrot_expert_plan_workspace_bytes(count, experts)
        work = torch.empty((need,), dtype=torch.uint8, device=device) if need else None
        nat.check(lib.convrot_expert_plan(ids.data_ptr(), 64 if ids.dtype == torch.int64 else 32, count, experts,
                                          offsets.data_ptr(), order.data_ptr(), slots.data_ptr(), nat.address(work), need,
                                          nat.stream_handle(device)))
    return ExpertPlan(offsets, order, slots)


def _plan_tensor(name: str, t: torch.Tensor | None, ndim: int) -> torch.Tensor:
    if t is None:
        raise ValueError(f"this call needs the plan's {name}")
    if t.dtype != torch.int32 or t.ndim != ndim or not t.is_contiguous():
        raise ValueError(f"the plan's {name} must be contiguous int32 with {ndim} axes, got {t.dtype} {tuple(t.shape)}")
    return t


class _Rows(NamedTuple):
    offsets: torch.Tensor
    index: torch.Tensor | None  # choice of each sorted row, where rows are read through it
    choices: int
    rows: int


def _grouped_rows(x: torch.Tensor, experts: int, plan: ExpertPlan, gather: bool) -> _Rows:
    """The sorted rows of a call on x, checked against the plan and the weight's experts."""
    if x.ndim != 2:
        raise ValueError(f"experts' linears take rows [R, K], got {tuple(x.shape)}")
    offsets = _plan_tensor("offsets", plan.offsets, 1)
    if experts < 1 or experts > MAX_EXPERTS:
        raise ValueError(f"experts' linears support 1 to {MAX_EXPERTS} experts, got {experts}")
    if offsets.shape[0] != experts + 1:
        raise ValueError(f"the plan orders rows by {offsets.shape[0] - 1} experts, the weight has {experts}")
    tokens = x.shape[0]
    if not gather:
        if plan.order is not None and plan.order.numel() != tokens:
            raise ValueError(f"the plan sorts {plan.order.numel()} rows, got {tokens} (gather=True reads tokens' rows)")
        return _Rows(offsets, None, 1, tokens)
    index = _plan_tensor("order", plan.order, 1)
    rows = index.shape[0]
    if rows % max(1, tokens) or (tokens == 0 and rows):
        raise ValueError(f"{rows} sorted rows are no whole number of choices of {tokens} tokens")
    return _Rows(offsets, index, max(1, rows // max(1, tokens)), rows)


def _gather_rows(x: torch.Tensor, index: torch.Tensor, choices: int) -> torch.Tensor:
    """Row index[s] // choices of x for each s."""
    x = rows_of(x)
    out = torch.empty((index.shape[0], x.shape[1]), dtype=x.dtype, device=x.device)
    with nat.on(x.device):
        nat.check(nat.load().convrot_gather_rows(x.data_ptr(), nat.dtype_code(x.dtype), x.shape[0], x.stride(0),
                                                 index.data_ptr(), choices, index.shape[0], x.shape[1], out.data_ptr(),
                                                 nat.stream_handle(x.device)))
    return out


# ------------------------------------------------------------------ 8-bit floating point


def _fp8_grouped(x, qweight, wscales, k: int, r: _Rows) -> torch.Tensor:
    x, w, ws = rows_of(x), _operand(qweight), _weight_scales(wscales)
    experts, n, _ = qweight.shape
    padded = (k + 127) // 128 * 128
    if r.index is not None and x.shape[0] * padded > MAX_GATHERED_BYTES:
        x, r = _gather_rows(x, r.index, r.choices), r._replace(index=None, choices=1)
    out = torch.empty((r.rows, n), dtype=x.dtype, device=x.device)
    lib = nat.load()
    with nat.on(x.device):
        need = lib.convrot_fp8_scratch_bytes(x.shape[0], k)
        scratch = torch.empty((need,), dtype=torch.uint8, device=x.device)
        nat.check(lib.convrot_fp8_grouped_linear(
            x.data_ptr(), nat.dtype_code(x.dtype), x.shape[0], x.stride(0), w.data_ptr(), _row_stride(w),
            w.stride(0) if experts > 1 else 0, ws.data_ptr(), ws.shape[2], ws.stride(0) if experts > 1 else 0,
            r.offsets.data_ptr(), experts, nat.address(r.index), r.choices, r.rows, n, k, scratch.data_ptr(), need,
            out.data_ptr(), nat.stream_handle(x.device)))
    return out


def hip_fp8_grouped_linear(x: torch.Tensor, qweight: torch.Tensor, wscales: torch.Tensor, plan: ExpertPlan, *,
                           gather: bool = False) -> torch.Tensor:
    """Sorted rows x [R, K] (or with `gather` tokens' rows x [T, K], read in the plan's order; float32, float16
    or bfloat16), quantized in blocks of 128, each times its expert's weight: float8_e4m3fn qweight [E, N, K] with
    scales [E, ceil(N / 128), ceil(K / 128)] -> [R, N] of x's type.  Rows of no expert give zeros."""
    k = x.shape[-1] if x.ndim else 0
    _check_weight(k, qweight, wscales, 3)
    r = _grouped_rows(x, qweight.shape[0], plan, gather)
    nat.dtype_code(x.dtype)
    nat.on_device(x, qweight, wscales, plan.offsets, r.index)
    return nat.without_gradient(lambda: _fp8_grouped(x, qweight, wscales, k, r), "hip_fp8_grouped_linear", x, wscales)


# ------------------------------------------------------------------ the rows summed back


def _combine_checks(rows: torch.Tensor, plan: ExpertPlan, weights: torch.Tensor | None) -> tuple:
    slots, order = _plan_tensor("slots", plan.slots, 2), _plan_tensor("order", plan.order, 1)
    if rows.ndim != 2 or rows.shape[0] != slots.numel() or order.shape[0] != slots.numel():
        raise ValueError(f"rows {tuple(rows.shape)} must be the {slots.numel()} sorted rows of the plan")
    if slots.shape[1] < 1:
        raise ValueError("combine_rows needs at least one choice a token")
    if weights is not None and (weights.shape != slots.shape or not weights.is_floating_point()):
        raise ValueError(f"weights must be floating point {tuple(slots.shape)}, got {weights.dtype} {tuple(weights.shape)}")
    nat.dtype_code(rows.dtype)
    nat.on_device(rows, slots, order, weights)
    return slots, order


def _as_float(weights: torch.Tensor | None) -> torch.Tensor | None:
    return None if weights is None else weights.to(torch.float32).contiguous()


def hip_combine_rows(rows: torch.Tensor, plan: ExpertPlan, weights: torch.Tensor | None = None) -> torch.Tensor:
    """[T, N] = sum over c of weights[t, c] * rows[slots[t, c]] (weights [T, C], 1 without), in float32 in the
    choices' order, rounded once to the rows' type."""
    slots, _ = _combine_checks(rows, plan, weights)
    rows, w = rows_of(rows), _as_float(weights)
    tokens, choices = slots.shape
    out = torch.empty((tokens, rows.shape[1]), dtype=rows.dtype, device=rows.device)
    with nat.on(rows.device):
        nat.check(nat.load().convrot_combine_rows(rows.data_ptr(), nat.dtype_code(rows.dtype), rows.shape[0],
                                                  rows.stride(0), slots.data_ptr(), nat.address(w), tokens, choices,
                                                  rows.shape[1], out.data_ptr(), nat.stream_handle(rows.device)))
    return out


def hip_combine_rows_backward(dout: torch.Tensor, rows: torch.Tensor | None, plan: ExpertPlan,
                              weights: torch.Tensor | None = None):
    """Gradients of hip_combine_rows from dout [T, N]: (drows [T C, N] = weights[t, c] * dout[t], dweights [T, C] =
    <dout[t], rows[slots[t, c]]> of the weights' type); without weights dweights is None and rows are not read."""
    slots, order = _plan_tensor("slots", plan.slots, 2), _plan_tensor("order", plan.order, 1)
    tokens, choices = slots.shape
    if dout.ndim != 2 or dout.shape[0] != tokens:
        raise ValueError(f"dout {tuple(dout.shape)} must have a row for each of {tokens} tokens")
    if weights is not None:
        _combine_checks(rows, plan, weights)
        if rows.dtype != dout.dtype or rows.shape[1] != dout.shape[1]:
            raise ValueError(f"dout {dout.dtype} {tuple(dout.shape)} must match rows {rows.dtype} {tuple(rows.shape)}")
    elif order.shape[0] != slots.numel():
        raise ValueError(f"the plan's order has {order.shape[0]} rows, its slots {slots.numel()}")
    nat.dtype_code(dout.dtype)
    device = nat.on_device(dout, slots, order, weights, rows if weights is not None else None)
    dout, w = rows_of(dout), _as_float(weights)
    n = dout.shape[1]
    y = None if w is None else rows_of(rows)
    drows = torch.empty((slots.numel(), n), dtype=dout.dtype, device=device)
    dw = None if w is None else torch.empty((tokens, choices), dtype=torch.float32, device=device)
    if n == 0:
        return drows, None if dw is None else dw.zero_().to(weights.dtype)
    with nat.on(device):
        nat.check(nat.load().convrot_combine_rows_backward(
            dout.data_ptr(), dout.stride(0), nat.address(y), 0 if y is None else y.stride(0), nat.dtype_code(dout.dtype),
            slots.numel(), order.data_ptr(), slots.data_ptr(), nat.address(w), tokens, max(1, choices), n, drows.data_ptr(),
            nat.address(dw), nat.stream_handle(device)))
    return drows, None if dw is None else dw.to(weights.dtype)


class _CombineRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, plan):
        ctx.save_for_backward(rows if weights is not None else None, weights, *plan)
        return hip_combine_rows(rows, plan, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        rows, weights, *plan = ctx.saved_tensors
        drows, dw = hip_combine_rows_backward(dout, rows, ExpertPlan(*plan), weights)
        needs = ctx.needs_input_grad
        return drows if needs[0] else None, dw if needs[1] else None, None


def combine_rows(rows: torch.Tensor, plan: ExpertPlan, weights: torch.Tensor | None = None) -> torch.Tensor:
    """hip_combine_rows, with gradients for the rows and the weights (reverse mode; dual tensors of forward
    mode are refused)."""
    if nat.differentiated(rows, weights):
        return _CombineRows.apply(rows, weights, plan)
    return hip_combine_rows(rows, plan, weights)
