"""Layer norm with a weight and bias, or with the shift and scale of adaptive layer norm (adaLN),
and its gradient.

    y = u * g + b,  u = (x - mean) / sqrt(var + eps),  g = weight or 1 + scale, b = bias or shift

in float32, rounded once.  hip_layer_norm and hip_layer_norm_backward are the two kernels;
layer_norm is the operator that torch differentiates through.  No counterpart in the reference,
whose example model runs the norm as array operations (examples/flux1_dev/adapter.py:45-70).
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from .core import check_vectors

MAX_BACKWARD_FEATURES = 32768


def rows_of(x: torch.Tensor) -> torch.Tensor:
    """A 2-D tensor with adjacent features and rows at one stride (else a contiguous copy)."""
    if (x.shape[1] > 1 and x.stride(1) != 1) or x.stride(0) < 0:
        return x.contiguous()
    return x


def flat_rows(x: torch.Tensor) -> torch.Tensor:
    """x [..., K] as rows_of's two dimensions."""
    if x.ndim < 1:
        raise ValueError("rows of features need at least one dimension")
    if x.ndim != 2:
        x = x.reshape(-1, x.shape[-1]) if x.shape[-1] else x.new_empty((0, 0))
    return rows_of(x)


def norm_operands(x2d, weight, bias, scale, shift, shape):
    """(gain or None, shift or None, rows a vector, plus one?) of a norm's parameters beside x of `shape`:
    contiguous rows of K, both of one type that the kernels take beside x's."""
    rows, k = x2d.shape
    check_vectors(shape, scale, shift)
    if (weight is not None or bias is not None) and (scale is not None or shift is not None):
        raise ValueError("layer norm takes weight and bias, or scale and shift")
    plus_one = scale is not None or shift is not None
    gain, add = (scale, shift) if plus_one else (weight, bias)
    given = [t for t in (gain, add) if t is not None]
    if not given:
        return None, None, max(1, rows), plus_one
    for t in given:
        if t.ndim < 1 or t.shape[-1] != k or t.numel() == 0 or (not plus_one and t.ndim != 1):
            what = "scale and shift must end in" if plus_one else "weight and bias must have"
            raise ValueError(f"layer norm {what} {k} features, got {tuple(t.shape)}")
    vectors = given[0].numel() // k
    if given[-1].numel() // k != vectors:
        raise ValueError(f"shift has {given[-1].numel() // k} rows but scale has {vectors}")
    if rows % vectors:
        raise ValueError(f"{rows} activation rows do not split evenly over {vectors} modulation vectors")
    kind = x2d.dtype
    for t in given:
        if t.dtype != kind:
            kind = torch.float32
    if gain is not None and not (gain.dtype == kind and gain.is_contiguous()):
        gain = gain.to(kind).contiguous()
    if add is not None and not (add.dtype == kind and add.is_contiguous()):
        add = add.to(kind).contiguous()
    return gain, add, max(1, rows // vectors), plus_one


def hip_layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
                   scale: torch.Tensor | None = None, shift: torch.Tensor | None = None, eps: float = 1e-6,
                   return_stats: bool = False):
    """Layer norm over the last axis of x [..., K] (rows at any one stride), of x's type.

    weight, bias: [K].  Or scale, shift: [V, K] or [V, 1, K], the rows split evenly over the V
    vectors in order, as x [B, L, K] beside scale [B, 1, K] does: (1 + scale) * u + shift (shapes that
    broadcast to other rows, [1, L, K], are refused).  Either of a pair may be None.  With
    return_stats also the rows' float32 mean and 1 / sqrt(var + eps)."""
    device = nat.on_device(x, weight, bias, scale, shift)
    x2d = flat_rows(x)
    rows, k = x2d.shape
    gain, add, each, plus_one = norm_operands(x2d, weight, bias, scale, shift, x.shape)
    out = x.new_empty(x.shape)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if return_stats else None
    mean, rstd = (None, None) if stats is None else stats.unbind(0)
    kind = gain if gain is not None else add
    nat.check(nat.load().convrot_layer_norm(
        x2d.data_ptr(), nat.dtype_code(x.dtype), rows, k, x2d.stride(0), nat.address(gain), nat.address(add),
        nat.dtype_code(x.dtype if kind is None else kind.dtype), plus_one, each, eps, out.data_ptr(),
        nat.address(mean), nat.address(rstd), nat.stream_handle(device)))
    return out if stats is None else (out, mean, rstd)


def hip_layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, *,
                            weight: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                            vectors: int | None = None, param_grads: bool = True,
                            shift_dtype: torch.dtype | None = None):
    """Gradients of hip_layer_norm from dy, its input and its stats: (dx, dgain, dshift).

    dgain is the gradient of weight (or scale), dshift that of bias (or shift), [K] beside a
    weight, else of scale's shape ([vectors, K] where the norm had a shift alone: pass `vectors`);
    both are of the weight's or scale's type (x's without one), None without param_grads.  A bias or
    shift of another type: pass it as `shift_dtype`, and dshift is rounded to that one alone.  Sums
    over rows are float32 in a fixed order: results repeat bit for bit."""
    nat.require_device(dy, x, mean, rstd, weight, scale)
    if dy.shape != x.shape:
        raise ValueError(f"dy {tuple(dy.shape)} must have the shape of x {tuple(x.shape)}")
    if dy.dtype != x.dtype:
        raise ValueError(f"dy dtype {dy.dtype} differs from x dtype {x.dtype}")
    x2d, dy2d = flat_rows(x), flat_rows(dy)
    rows, k = x2d.shape
    if k > MAX_BACKWARD_FEATURES:
        raise ValueError(f"the layer norm's gradient supports at most {MAX_BACKWARD_FEATURES} features, got {k}")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if tuple(t.shape) != (rows,) or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 {(rows,)}, got {t.dtype} {tuple(t.shape)}")
    gain, _, each, plus_one = norm_operands(x2d, weight, None, scale, None, x.shape)
    if gain is None and vectors is not None:
        if vectors < 1 or rows % vectors:
            raise ValueError(f"{rows} activation rows do not split evenly over {vectors} modulation vectors")
        each = max(1, rows // vectors)
    if gain is not None:
        vectors = gain.numel() // k
    given = scale if scale is not None else weight
    kind = x.dtype if gain is None else gain.dtype
    gain_dtype = x.dtype if given is None else given.dtype
    if shift_dtype is None:
        shift_dtype = gain_dtype
    if param_grads and kind != torch.float32 and shift_dtype != kind:
        kind = torch.float32  # the sums as they are, each rounded once to its parameter's type
        gain = None if gain is None else gain.to(kind)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    grads = work = None
    lib = nat.load()
    if param_grads:
        grads = torch.empty((2, vectors or 1, k), dtype=kind, device=x.device)
        work = torch.empty((lib.convrot_layer_norm_workspace_bytes(rows, k, each),), dtype=torch.uint8,
                           device=x.device)
    nat.check(lib.convrot_layer_norm_backward(
        dy2d.data_ptr(), dy2d.stride(0), x2d.data_ptr(), x2d.stride(0), mean.data_ptr(), rstd.data_ptr(),
        nat.dtype_code(x.dtype), rows, k, nat.address(gain), nat.dtype_code(kind), plus_one, each, dx.data_ptr(),
        None if grads is None else grads[0].data_ptr(), None if grads is None else grads[1].data_ptr(),
        nat.address(work), 0 if work is None else work.numel(), nat.stream_handle(x.device)))
    if grads is None:
        return dx, None, None
    if rows == 0:
        grads.zero_()
    shape = given.shape if given is not None else (k,) if vectors is None else (vectors, k)
    return dx, grads[0].reshape(shape).to(gain_dtype), grads[1].reshape(shape).to(shift_dtype)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, scale, shift, eps):
        y, mean, rstd = hip_layer_norm(x, weight, bias, scale=scale, shift=shift, eps=eps, return_stats=True)
        ctx.save_for_backward(x, mean, rstd, weight, scale)
        add = bias if bias is not None else shift
        ctx.adaptive = scale is not None or shift is not None
        ctx.add = None if add is None else (add.shape, add.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, mean, rstd, weight, scale = ctx.saved_tensors
        needs = ctx.needs_input_grad
        vectors = None
        if ctx.adaptive and scale is None:
            vectors = ctx.add[0].numel() // max(1, x.shape[-1])
        dx, dgain, dadd = hip_layer_norm_backward(dy, x, mean, rstd, weight=weight, scale=scale, vectors=vectors,
                                                  param_grads=any(needs[1:5]),
                                                  shift_dtype=None if ctx.add is None else ctx.add[1])
        if dadd is not None and ctx.add is not None:
            dadd = dadd.reshape(ctx.add[0])
        a = ctx.adaptive
        return (dx if needs[0] else None, dgain if needs[1] and not a else None, dadd if needs[2] and not a else None,
                dgain if needs[3] and a else None, dadd if needs[4] and a else None, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
               scale: torch.Tensor | None = None, shift: torch.Tensor | None = None,
               eps: float = 1e-6) -> torch.Tensor:
    """hip_layer_norm, with gradients for x and for the parameters that need them (reverse mode; dual
    tensors of forward mode are refused)."""
    if nat.differentiated(x, weight, bias, scale, shift):
        return _LayerNorm.apply(x, weight, bias, scale, shift, eps)
    return hip_layer_norm(x, weight, bias, scale=scale, shift=shift, eps=eps)
