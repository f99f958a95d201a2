"""Rotary positions with several axes (time, height, width) and the per-head RMS norm in front of
them, for queries and keys, and their gradients.

A head's features x become n = x / sqrt(mean(x^2) + eps) * weight (with weights), and the pairs
(a, b) of its first 2 P features (a cos - b sin, a sin + b cos): features (2 p, 2 p + 1) when
interleaved, else (p, P + p).  All in float32, rounded once.  hip_qk_rotary and
hip_qk_rotary_backward are the kernels; qk_rotary is the operator that torch differentiates
through.  No counterpart in the reference, which leaves rotary positions to its model runtime.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat

MAX_HEAD_DIM = 512
_POSITIONS = {torch.float32: nat.POS_F32, torch.float64: nat.POS_F64, torch.int32: nat.POS_I32,
              torch.int64: nat.POS_I64}


def rotary_axes_table(positions: torch.Tensor, axes_dim, theta: float = 10000.0) -> torch.Tensor:
    """Cosines and sines of positions [..., A] (float32, float64, int32 or int64) -> float32
    [..., P, 2], P = sum(axes_dim) / 2: axis a turns axes_dim[a] features, its i-th pair by
    position * theta^(-2 i / axes_dim[a]).  Made once for all heads and layers of a step."""
    dims = [int(d) for d in axes_dim]
    if positions.ndim < 1 or positions.shape[-1] != len(dims):
        raise ValueError(f"positions {tuple(positions.shape)} must end in {len(dims)} axes")
    if positions.dtype not in _POSITIONS:
        raise ValueError(f"positions must be float32, float64, int32 or int64, got {positions.dtype}")
    if not 1 <= len(dims) <= 8 or any(d < 0 or d % 2 for d in dims):
        raise ValueError(f"axes_dim must be 1 to 8 even numbers of features, got {dims}")
    nat.require_device(positions)
    pos = positions.contiguous()
    out = torch.empty((*pos.shape[:-1], sum(dims) // 2, 2), dtype=torch.float32, device=pos.device)
    rows = pos.numel() // len(dims)
    nat.check(nat.load().convrot_axes_table(nat.ptr(pos), _POSITIONS[pos.dtype], rows, len(dims),
                                            (ctypes.c_int * len(dims))(*dims), float(theta), nat.ptr(out),
                                            nat.stream_of(pos.device)))
    return out


def _heads(name: str, t: torch.Tensor) -> torch.Tensor:
    """[B, H, L, D] with adjacent features (else a contiguous copy)."""
    if t.ndim != 4:
        raise ValueError(f"{name} must be [batch, heads, length, dim], got {tuple(t.shape)}")
    return t.contiguous() if t.shape[3] > 1 and t.stride(3) != 1 else t


def _check(q, k, table, q_weight, k_weight):
    b, _, length, d = q.shape
    kb, _, klength, kd = k.shape
    if kb != b or klength != length or kd != d:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must agree in batch, length and dim")
    if k.dtype != q.dtype:
        raise ValueError(f"k dtype {k.dtype} differs from q dtype {q.dtype}")
    if d > MAX_HEAD_DIM:
        raise ValueError(f"rotary positions support heads of up to {MAX_HEAD_DIM} features, got {d}")
    size = table.shape
    if len(size) not in (3, 4) or size[-1] != 2 or size[-3] != length or table.dtype != torch.float32:
        raise ValueError(f"table must be float32 [batch or 1, {length}, pairs, 2], got {table.dtype} "
                         f"{tuple(table.shape)}")
    if len(size) == 4 and size[0] not in (1, b):
        raise ValueError(f"table has {size[0]} batch entries for a batch of {b}")
    if 2 * size[-2] > d:
        raise ValueError(f"{size[-2]} pairs do not fit a head of {d} features")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and tuple(w.shape) != (d,):
            raise ValueError(f"{name} must have shape {(d,)}, got {tuple(w.shape)}")
    nat.on_device(q, k, table, q_weight, k_weight)


def _weights(q_weight, k_weight, dtype):
    """The norm weights in one type that the kernel takes (x's or float32)."""
    if q_weight is None and k_weight is None:
        return None, None, dtype
    given = [w for w in (q_weight, k_weight) if w is not None]
    kind = dtype if all(w.dtype == dtype for w in given) else torch.float32
    qw, kw = (None if w is None else w.to(kind).contiguous() for w in (q_weight, k_weight))
    return qw, kw, kind


def _table_args(table: torch.Tensor):
    """(table, floats between batch entries): its last three axes dense."""
    if table.is_contiguous():
        return table, table.stride(0) if table.ndim == 4 and table.shape[0] > 1 else 0
    dense = (2 * table.shape[-2], 2, 1)
    if any(n > 1 and s != want for n, s, want in zip(table.shape[-3:], table.stride()[-3:], dense)):
        table = table.contiguous()
    stride = table.stride(0) if table.ndim == 4 and table.shape[0] > 1 else 0
    return table, stride


_Int64x12, _Int64x18 = ctypes.c_int64 * 12, ctypes.c_int64 * 18


def _strides(*tensors):
    flat = []
    for t in tensors:
        flat += t.stride()[:3]
    return (_Int64x12 if len(flat) == 12 else _Int64x18)(*flat)


def _out(name: str, out, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return like.new_empty(like.shape)
    if out.shape != like.shape or out.dtype != like.dtype or (out.shape[3] > 1 and out.stride(3) != 1):
        raise ValueError(f"{name} must be {like.dtype} {tuple(like.shape)} with adjacent features, got {out.dtype} "
                         f"{tuple(out.shape)}")
    if any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError(f"{name} must not be an expanded tensor")
    return out


def hip_qk_rotary(q: torch.Tensor, k: torch.Tensor, table: torch.Tensor, *, q_weight: torch.Tensor | None = None,
                  k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = True,
                  q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """(q, k) [B, H, L, D] with the head norm (where a weight [D] is given) and rotary positions.

    q and k are read in place with any strides of batch, head and token (views of a fused
    projection's output); k may have fewer heads.  table: rotary_axes_table's [L, P, 2] or
    [B or 1, L, P, 2].  Without q_out / k_out the results are contiguous [B, H, L, D], what
    attention reads; with them they go there, e.g. into one stream's part of a joint sequence."""
    q, k = _heads("q", q), _heads("k", k)
    _check(q, k, table, q_weight, k_weight)
    qw, kw, kind = _weights(q_weight, k_weight, q.dtype)
    table, table_stride = _table_args(table)
    if q_out is not None or k_out is not None:
        nat.on_device(q, q_out, k_out)
    q_out, k_out = _out("q_out", q_out, q), _out("k_out", k_out, k)
    b, hq, length, d = q.shape
    nat.check(nat.load().convrot_qk_rotary(
        q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), _strides(q, k, q_out, k_out),
        nat.dtype_code(q.dtype), b, hq, k.shape[1], length, d, table.data_ptr(), table.shape[-2], table_stride,
        nat.address(qw), nat.address(kw), nat.dtype_code(kind), eps, interleaved, nat.stream_handle(q.device)))
    return q_out, k_out


def hip_qk_rotary_backward(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                           table: torch.Tensor, *, q_weight: torch.Tensor | None = None,
                           k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = True):
    """Gradients of hip_qk_rotary: (dq_in, dk_in, dq_weight, dk_weight), the last two None without
    the weight.  dq_in and dk_in are [B, H, L, D] over memory in [B, L, H, D] order, as a fused
    projection's output holds heads.  Weight gradients are float32 sums over tokens and heads in
    a fixed order (results repeat bit for bit), of the weight's type."""
    q, k, dq, dk = _heads("q", q), _heads("k", k), _heads("dq", dq), _heads("dk", dk)
    _check(q, k, table, q_weight, k_weight)
    if dq.shape != q.shape or dk.shape != k.shape or dq.dtype != q.dtype or dk.dtype != q.dtype:
        raise ValueError(f"dq {dq.dtype} {tuple(dq.shape)} and dk {dk.dtype} {tuple(dk.shape)} must match q "
                         f"{q.dtype} {tuple(q.shape)} and k {tuple(k.shape)}")
    nat.on_device(q, dq, dk)
    qw, kw, kind = _weights(q_weight, k_weight, q.dtype)
    table, table_stride = _table_args(table)
    b, hq, length, d = q.shape

    def like(t):
        return torch.empty((t.shape[0], t.shape[2], t.shape[1], t.shape[3]), dtype=t.dtype,
                           device=t.device).transpose(1, 2)

    lib = nat.load()
    gq, gk = like(q), like(k)
    work = gw = None
    if qw is not None or kw is not None:
        gw = torch.empty((2, d), dtype=kind, device=q.device)
        work = torch.empty((lib.convrot_qk_rotary_workspace_bytes(d),), dtype=torch.uint8, device=q.device)
    nat.check(lib.convrot_qk_rotary_backward(
        dq.data_ptr(), dk.data_ptr(), q.data_ptr(), k.data_ptr(), gq.data_ptr(), gk.data_ptr(),
        None if qw is None else gw[0].data_ptr(), None if kw is None else gw[1].data_ptr(),
        _strides(dq, dk, q, k, gq, gk), nat.dtype_code(q.dtype), b, hq, k.shape[1], length, d, table.data_ptr(),
        table.shape[-2], table_stride, nat.address(qw), nat.address(kw), nat.dtype_code(kind), eps, interleaved,
        nat.address(work), 0 if work is None else work.numel(), nat.stream_handle(q.device)))
    if gw is not None and b * length * (hq + k.shape[1]) == 0:
        gw.zero_()
    return (gq, gk, None if qw is None else gw[0].to(q_weight.dtype), None if kw is None else gw[1].to(k_weight.dtype))


class _QkRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, table, q_weight, k_weight, eps, interleaved):
        ctx.save_for_backward(q, k, table, q_weight, k_weight)
        ctx.eps, ctx.interleaved = eps, interleaved
        return hip_qk_rotary(q, k, table, q_weight=q_weight, k_weight=k_weight, eps=eps, interleaved=interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, table, q_weight, k_weight = ctx.saved_tensors
        gq, gk, gqw, gkw = hip_qk_rotary_backward(dq, dk, q, k, table, q_weight=q_weight, k_weight=k_weight,
                                                  eps=ctx.eps, interleaved=ctx.interleaved)
        return gq, gk, None, gqw, gkw, None, None


def qk_rotary(q: torch.Tensor, k: torch.Tensor, table: torch.Tensor, *, q_weight: torch.Tensor | None = None,
              k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = True):
    """hip_qk_rotary, with gradients for q, k and the norm weights (none for the table; reverse mode, dual
    tensors of forward mode are refused)."""
    if nat.differentiated(q, k, q_weight, k_weight):
        return _QkRotary.apply(q, k, table, q_weight, k_weight, eps, interleaved)
    return hip_qk_rotary(q, k, table, q_weight=q_weight, k_weight=k_weight, eps=eps, interleaved=interleaved)
