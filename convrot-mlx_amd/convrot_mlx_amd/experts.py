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
from torch import nn
from torch.autograd.function import once_differentiable

from . import _native as nat
from .fp8 import CODES, MAX_FEATURES, Fp8Buffers, _check_weight, _operand, _row_stride, _weight_scales, quantize_fp8_weight
from .norm import rows_of

MAX_PLAN_EXPERTS = 1024
MAX_EXPERTS = 65536
MAX_GATHERED_BYTES = (1 << 32) - 4096
MAX_STRIDE = 1 << 21


class ExpertPlan(NamedTuple):
    """Sorted rows by expert, int32 on the device: expert e has rows offsets[e] .. offsets[e + 1] - 1
    (offsets [E + 1], from 0), row s is choice order[s] (token order[s] // C, order [T C]), and choice
    (t, c) is row slots[t, c].  order and slots may be None for rows that a caller sorted itself.  A caller's own
    may hold places out of range (a row of no choice, a choice without a row); else they are each other's
    inverse, and no two choices share a row: gradients follow order and slots where they agree."""

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
    order = torch.empty((count,), dtype=torch.int32, device=device)
    slots = torch.empty(ids.shape if ids.ndim == 2 else (count, 1), dtype=torch.int32, device=device)
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
    if plan.slots is not None:  # says how many choices a token has: x of another number of tokens is no input of this plan
        slots = _plan_tensor("slots", plan.slots, 2)
        if slots.shape[0] != tokens or slots.numel() != rows:
            raise ValueError(f"the plan orders {tuple(slots.shape)} choices, {slots.shape[0]} tokens' ({rows} rows), got x of "
                             f"{tokens} rows (sorted rows are taken without gather)")
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
    """Gradients of hip_combine_rows from dout [T, N]: (drows [T C, N] = weights[t, c] * dout[t], zeros in rows
    that are no choice's, dweights [T, C] = <dout[t], rows[slots[t, c]]> of the weights' type); without weights
    dweights is None and rows are not read."""
    slots, order = _plan_tensor("slots", plan.slots, 2), _plan_tensor("order", plan.order, 1)
    tokens, choices = slots.shape
    if dout.ndim != 2 or dout.shape[0] != tokens:
        raise ValueError(f"dout {tuple(dout.shape)} must have a row for each of {tokens} tokens")
    if weights is not None:
        if rows is None:
            raise ValueError("the gradient of weights needs the rows they weighted")
        if rows.dtype != dout.dtype or rows.ndim != 2 or rows.shape[1] != dout.shape[1]:
            raise ValueError(f"dout {dout.dtype} {tuple(dout.shape)} must match rows {rows.dtype} {tuple(rows.shape)}")
        _combine_checks(rows, plan, weights)
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


# ------------------------------------------------------------------ 16 bits, with gradients


def _operand16(t: torch.Tensor) -> torch.Tensor:
    """[.., K] in 16 bits as the products read it, itself or a copy: adjacent features, rows (and experts) 16-byte
    aligned, zeros from K to the next multiple of 8."""
    k = t.shape[-1]
    if k % 8 == 0 and t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        stride = _stride16(t)
        if (t.stride(-1) == 1 and stride % 8 == 0 and k <= stride <= MAX_STRIDE
                and (t.ndim == 2 or t.shape[0] == 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= 0))):
            return t
    padded = t.new_zeros((*t.shape[:-1], (k + 7) // 8 * 8))
    padded[..., :k] = t
    return padded


def _stride16(t: torch.Tensor) -> int:
    """Elements between rows (the stride of a single row says nothing)."""
    return t.stride(-2) if t.shape[-2] > 1 else (t.shape[-1] + 7) // 8 * 8


def _expert_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else 0


def _check_grouped(x: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan, gather: bool) -> _Rows:
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"experts' linears take float16 or bfloat16, got {x.dtype}")
    if weight.ndim != 3 or weight.dtype != x.dtype:
        raise ValueError(f"experts' weights must be {x.dtype} [E, N, K], got {weight.dtype} {tuple(weight.shape)}")
    _, n, k = weight.shape
    if not (1 <= n <= MAX_FEATURES and 1 <= k <= MAX_FEATURES):
        raise ValueError(f"experts' linears support 1 to {MAX_FEATURES} features, got N={n} K={k}")
    r = _grouped_rows(x, weight.shape[0], plan, gather)
    if x.shape[1] != k:
        raise ValueError(f"experts' weights take K={k} features, got {x.shape[1]}")
    return r


def hip_grouped_linear(x: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan, *, gather: bool = False) -> torch.Tensor:
    """Sorted rows x [R, K] (or with `gather` tokens' rows x [T, K], read in the plan's order), float16 or
    bfloat16, each times its expert's weight of [E, N, K] -> [R, N]; float32 sums, rounded once.  Rows of no
    expert give zeros.  Features no multiple of 8 copy operands into padded rows."""
    r = _check_grouped(x, weight, plan, gather)
    nat.on_device(x, weight, r.offsets, r.index)
    experts, n, k = weight.shape
    x, w = _operand16(x), _operand16(weight)
    if r.index is not None and x.shape[0] * _stride16(x) * 2 > MAX_GATHERED_BYTES:
        x, r = _operand16(_gather_rows(x[:, :k], r.index, r.choices)), r._replace(index=None, choices=1)
    out = torch.empty((r.rows, n), dtype=x.dtype, device=x.device)
    with nat.on(x.device):
        nat.check(nat.load().convrot_grouped_linear(
            x.data_ptr(), nat.dtype_code(x.dtype), x.shape[0], _stride16(x), w.data_ptr(), _stride16(w), _expert_stride(w),
            r.offsets.data_ptr(), experts, nat.address(r.index), r.choices, r.rows, n, k, out.data_ptr(),
            nat.stream_handle(x.device)))
    return out


def hip_grouped_linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan, *,
                                gather: bool = False, rows_grad: bool = True, weight_grad: bool = True):
    """Gradients of hip_grouped_linear from dy [R, N]: (dx of x's shape, dweight [E, N, K]), either None where not
    wanted; float32 sums in a fixed order, rounded once (with `gather` a token's dx is the float32 sum of its
    choices' gradients, each rounded)."""
    r = _check_grouped(x, weight, plan, gather)
    experts, n, k = weight.shape
    if tuple(dy.shape) != (r.rows, n) or dy.dtype != x.dtype:
        raise ValueError(f"dy must be {x.dtype} {(r.rows, n)}, got {dy.dtype} {tuple(dy.shape)}")
    nat.on_device(dy, x, weight, r.offsets, r.index)
    if gather and rows_grad:
        _combine_checks(dy, plan, None)
    lib, code, device = nat.load(), nat.dtype_code(x.dtype), x.device
    g = _operand16(dy)
    dx = dw = None
    if rows_grad:
        w = _operand16(weight)
        dx = torch.empty((r.rows, k), dtype=x.dtype, device=device)
        with nat.on(device):
            nat.check(lib.convrot_grouped_linear_rows_grad(
                g.data_ptr(), code, _stride16(g), w.data_ptr(), _stride16(w), _expert_stride(w), r.offsets.data_ptr(),
                experts, r.rows, n, k, dx.data_ptr(), nat.stream_handle(device)))
        if gather:
            dx = hip_combine_rows(dx, plan)
    if weight_grad:
        rows = _operand16(x)
        if r.index is not None and rows.shape[0] * _stride16(rows) * 2 > MAX_GATHERED_BYTES:
            rows, r = _operand16(_gather_rows(x, r.index, r.choices)), r._replace(index=None, choices=1)
        dw = torch.empty((experts, n, k), dtype=x.dtype, device=device)
        with nat.on(device):
            nat.check(lib.convrot_grouped_linear_weight_grad(
                g.data_ptr(), code, _stride16(g), rows.data_ptr(), rows.shape[0], _stride16(rows), r.offsets.data_ptr(),
                experts, nat.address(r.index), r.choices, r.rows, n, k, dw.data_ptr(), nat.stream_handle(device)))
    return dx, dw


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, plan, gather):
        ctx.save_for_backward(x, weight, *plan)
        ctx.gather = gather
        return hip_grouped_linear(x, weight, plan, gather=gather)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, *plan = ctx.saved_tensors
        needs = ctx.needs_input_grad
        dx, dw = hip_grouped_linear_backward(dy, x, weight, ExpertPlan(*plan), gather=ctx.gather, rows_grad=needs[0],
                                             weight_grad=needs[1])
        return dx, dw, None, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan, *, gather: bool = False) -> torch.Tensor:
    """hip_grouped_linear, with gradients for the rows and the weights (reverse mode; dual tensors of forward
    mode are refused).  With `gather` the rows' gradient needs the plan's slots."""
    if nat.differentiated(x, weight):
        if gather and x.requires_grad:
            _plan_tensor("slots", plan.slots, 2)
        return _GroupedLinear.apply(x, weight, plan, gather)
    return hip_grouped_linear(x, weight, plan, gather=gather)


class ExpertLinear(nn.Module):
    """The dense linears of E experts: `weight` [E, N, K] (no bias), called on rows sorted by an ExpertPlan, or
    with gather=True on the tokens' rows.  Parameters start as torch's Linear starts its weight."""

    def __init__(self, experts: int, in_features: int, out_features: int, *, device=None, dtype=torch.bfloat16):
        super().__init__()
        self.weight = nn.Parameter(torch.empty((experts, out_features, in_features), device=device, dtype=dtype))
        nn.init.uniform_(self.weight, -in_features ** -0.5, in_features ** -0.5)

    def forward(self, x: torch.Tensor, plan: ExpertPlan, *, gather: bool = False) -> torch.Tensor:
        return grouped_linear(x, self.weight, plan, gather=gather)

    def extra_repr(self) -> str:
        experts, n, k = self.weight.shape
        return f"experts={experts}, in_features={k}, out_features={n}"


class Fp8ExpertLinear(Fp8Buffers):
    """The linears of E experts stored and executed in 8-bit floating point: `qweight` float8_e4m3fn [E, N, K],
    `scales` float32 [E, ceil(N / 128), ceil(K / 128)] (ones); no bias and no gradient: a backward pass that reaches
    it raises an error."""

    def __init__(self, experts: int, in_features: int, out_features: int, *, device=None):
        super().__init__()
        blocks = (out_features + 127) // 128, (in_features + 127) // 128
        self.register_buffer("qweight", torch.zeros((experts, out_features, in_features), dtype=torch.uint8,
                                                    device=device).view(CODES))
        self.register_buffer("scales", torch.ones((experts, *blocks), dtype=torch.float32, device=device))

    def load_weight(self, weight: torch.Tensor) -> Fp8ExpertLinear:
        """Quantize dense weights [E, N, K] into this layer."""
        if weight.shape != self.qweight.shape:
            raise ValueError(f"weight must have shape {tuple(self.qweight.shape)}, got {tuple(weight.shape)}")
        self.qweight, self.scales = quantize_fp8_weight(weight)
        return self

    def forward(self, x: torch.Tensor, plan: ExpertPlan, *, gather: bool = False) -> torch.Tensor:
        return hip_fp8_grouped_linear(x, self.qweight, self.scales, plan, gather=gather)

    def extra_repr(self) -> str:
        experts, n, k = self.qweight.shape
        return f"experts={experts}, in_features={k}, out_features={n}"
