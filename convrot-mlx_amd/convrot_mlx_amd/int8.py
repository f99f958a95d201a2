"""Linears of 8-bit integers (W8A8): one scale a token, one an output channel.

For the layers that 4 bits hurt, or whose features no rotation group divides: rows are
quantized symmetrically to [-127, 127] (codes = round(x * (127 / absmax)), scale = absmax / 127),
the integer product is exact and the epilogue is that of the 4-bit linears,
((dot * xscale) * wscale) + bias in float32.  A gated residual, residual + gate * linear, is taken
in float32 too and rounded once (the 4-bit linears round each operation).  Weights stay
row-major int8 [N, K], as 8-bit checkpoints hold them.  No counterpart in the reference, which
quantizes to 4 bits only.
"""

from __future__ import annotations

import torch
from torch import nn

from . import _native as nat
from .core import GatedResidual, _f32, _gated_residual, _workspace
from .norm import flat_rows, norm_operands, rows_of

MAX_FEATURES = 65536
MAX_ROW_STRIDE = 1 << 22


def _round16(k: int) -> int:
    return (k + 15) // 16 * 16


def quantize_int8_rowwise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of x [M, K] (any strides) as (int8 codes [M, K], float32 scales [M]).

    A row that holds a NaN or an infinity gets the scale NaN (its products are NaN); a row whose
    largest magnitude is below 2^-100 counts as zero.  Where K is no multiple of 16 the codes are a
    view of rows padded to one, as the matrix product reads them."""
    if x.ndim != 2:
        raise ValueError(f"rowwise int8 quantization expects 2D input, got {tuple(x.shape)}")
    nat.require_device(x)
    x = rows_of(x)
    m, k = x.shape
    codes = torch.empty((m, _round16(k)), dtype=torch.int8, device=x.device)
    scales = torch.empty((m,), dtype=torch.float32, device=x.device)
    nat.check(nat.load().convrot_quantize_int8(nat.ptr(x), nat.dtype_code(x.dtype), m, k, x.stride(0), nat.ptr(codes),
                                               codes.shape[1], nat.ptr(scales), nat.stream_of(x.device)))
    if k == 0:
        scales.zero_()
    return codes if codes.shape[1] == k else codes[:, :k], scales


def _row_stride(t: torch.Tensor) -> int:
    """Bytes between an operand's rows (the stride of a single row says nothing)."""
    return t.stride(0) if t.shape[0] > 1 else _round16(t.shape[1])


def _readable(t: torch.Tensor, zero_tail: bool) -> bool:
    """Whether the product can read an int8 matrix where it lies: adjacent features, 16-byte aligned rows
    that cover the features rounded up to 16 (past them zeros, with `zero_tail`)."""
    rows, k = t.shape
    if k % 16 == 0 and t.is_contiguous() and t.data_ptr() % 16 == 0:
        return True
    stride = _row_stride(t)
    return (t.stride(1) == 1 and stride % 16 == 0 and _round16(k) <= stride <= MAX_ROW_STRIDE
            and t.data_ptr() % 16 == 0
            and (k % 16 == 0 or (not zero_tail and (rows - 1) * stride + _round16(k) + t.storage_offset()
                                 <= t.untyped_storage().nbytes())))


def _padded(t: torch.Tensor) -> torch.Tensor:
    """A copy of an int8 matrix that the product can read."""
    k = t.shape[1]
    return torch.nn.functional.pad(t, (0, -k % 16)) if k % 16 else t.clone(memory_format=torch.contiguous_format)


def _operand(t: torch.Tensor, zero_tail: bool) -> torch.Tensor:
    """An int8 matrix as rows the product can read: itself, else a padded copy."""
    return t if _readable(t, zero_tail) else _padded(t)


def _scales(t: torch.Tensor | None) -> torch.Tensor | None:
    return t if t is None or (t.dtype == torch.float32 and t.is_contiguous()) else _f32(t)


def _check_scales(name: str, t: torch.Tensor, n: int) -> None:
    if t.ndim != 1 or t.shape[0] != n:
        raise ValueError(f"W8A8 {name} must have shape {(n,)}, got {tuple(t.shape)}")


def _residual_args(gr: GatedResidual | None) -> tuple:
    """(residual, gate, gate stride, rows per gate) of a library call."""
    if gr is None:
        return None, None, 0, 1
    return gr.residual.data_ptr(), None if gr.gate is None else gr.gate.data_ptr(), gr.stride, gr.rows_per_gate


def _output(gr: GatedResidual | None, m: int, n: int, dtype: torch.dtype, device) -> torch.Tensor:
    if gr is not None and gr.inplace:
        return gr.residual.view(m, n)
    return torch.empty((m, n), dtype=dtype, device=device)


_CONTROL_BYTES = 32768  # of a workspace: zero before a launch


def _product_workspace(device, stream: int, capturing: bool, m: int, n: int, k: int) -> torch.Tensor | None:
    """Counters and partial sums of a product whose workgroups share K: the stream's, or, as a graph may be
    replayed beside that stream and beside other graphs, memory of the graph's own."""
    if not capturing:
        return _workspace(device, stream)
    need = nat.load().convrot_w8a8_workspace_bytes(m, n, k)
    if need == 0:
        return None
    work = torch.empty((need,), dtype=torch.uint8, device=device)
    work[:_CONTROL_BYTES].zero_()
    return work


def _w8a8(act, weight, xscales, wscales, bias, k: int, dtype: torch.dtype, gr: GatedResidual | None) -> torch.Tensor:
    """The product of operands as the kernel reads them (see _operand)."""
    m, n = act.shape[0], weight.shape[0]
    out = _output(gr, m, n, dtype, act.device)
    stream = nat.stream_handle(act.device)
    work = _product_workspace(act.device, stream, torch.cuda.is_current_stream_capturing(), m, n, k)
    nat.check(nat.load().convrot_w8a8_gemm(
        act.data_ptr(), _row_stride(act), xscales.data_ptr(), weight.data_ptr(), _row_stride(weight), wscales.data_ptr(),
        None if bias is None else bias.data_ptr(), m, n, k, *_residual_args(gr),
        None if work is None else work.data_ptr(), 0 if work is None else work.numel(), out.data_ptr(),
        nat.dtype_code(dtype), stream))
    return out


def _linear(x: torch.Tensor, weight: torch.Tensor, wscales, bias, k: int, residual, gate, inplace: bool) -> torch.Tensor:
    """x [..., k] times a weight as the kernel reads it, one library call."""
    n, device = weight.shape[0], x.device
    x2d = flat_rows(x)
    m = x2d.shape[0]
    gr = _residual(residual, gate, inplace, m, n, x.dtype)
    out = _output(gr, m, n, x.dtype, device)
    lib, dtype, stride = nat.load(), nat.dtype_code(x.dtype), x2d.stride(0)
    stream = nat.stream_handle(device)
    capturing = torch.cuda.is_current_stream_capturing()
    work = _product_workspace(device, stream, capturing, m, n, k)
    work_bytes = 0 if work is None else work.numel()
    # codes and scales between the two launches: the end of the stream's workspace holds up to a
    # quarter of it; a graph holds its own
    need, scratch = m * ((k + 127) // 128 * 128 + 4), None
    if need * 4 > work_bytes or capturing:
        scratch = torch.empty((need,), dtype=torch.uint8, device=device)
    nat.check(lib.convrot_w8a8_linear(
        x2d.data_ptr(), dtype, stride, weight.data_ptr(), _row_stride(weight), wscales.data_ptr(),
        None if bias is None else bias.data_ptr(), m, n, k, *_residual_args(gr),
        None if scratch is None else scratch.data_ptr(), need, None if work is None else work.data_ptr(), work_bytes,
        out.data_ptr(), stream))
    if inplace:
        return residual
    return out if x.ndim == 2 else out.reshape(*x.shape[:-1], n)


def _check_product(k: int, weight: torch.Tensor, wscales, bias) -> int:
    if weight.ndim != 2 or weight.dtype != torch.int8:
        raise ValueError(f"W8A8 weight must be 2D int8, got {tuple(weight.shape)} {weight.dtype}")
    n = weight.shape[0]
    if weight.shape[1] != k:
        raise ValueError(f"W8A8 weight must be N x K with K={k}, got {tuple(weight.shape)}")
    if not 0 < k <= MAX_FEATURES:
        raise ValueError(f"W8A8 product needs 1 to {MAX_FEATURES} features, got {k}")
    _check_scales("weight scales", wscales, n)
    if bias is not None:
        _check_scales("bias", bias, n)
    return n


def _residual(residual, gate, inplace: bool, m: int, n: int, dtype: torch.dtype) -> GatedResidual | None:
    if residual is None:
        if gate is not None or inplace:
            raise ValueError("gate and inplace need a residual")
        return None
    if residual.ndim < 1 or residual.shape[-1] != n or residual.numel() != m * n:
        raise ValueError(f"residual {tuple(residual.shape)} must hold the [{m}, {n}] output as [..., {n}]")
    return _gated_residual(residual, gate, tuple(residual.shape), dtype, inplace)


def hip_w8a8_matmul(qact: torch.Tensor, qweight: torch.Tensor, xscales: torch.Tensor, wscales: torch.Tensor,
                    bias: torch.Tensor | None = None, *, output_dtype: torch.dtype, residual=None, gate=None,
                    inplace: bool = False) -> torch.Tensor:
    """int8 activations [M, K] x int8 weight [N, K] -> output_dtype [M, N]:
    ((dot * xscales[m]) * wscales[n]) + bias[n]; residual, gate and inplace as in hip_w4a4_matmul, with one rounding at the end."""
    if qact.ndim != 2 or qact.dtype != torch.int8:
        raise ValueError(f"W8A8 activation must be 2D int8, got {tuple(qact.shape)} {qact.dtype}")
    m, k = qact.shape
    n = _check_product(k, qweight, wscales, bias)
    _check_scales("activation scales", xscales, m)
    nat.dtype_code(output_dtype)
    nat.on_device(qact, qweight, xscales, wscales, bias, residual, gate)
    gr = _residual(residual, gate, inplace, m, n, output_dtype)

    def run():
        out = _w8a8(_operand(qact, False), _operand(qweight, True), _scales(xscales), _scales(wscales), _scales(bias), k,
                    output_dtype, gr)
        return residual if inplace else out

    out = nat.without_gradient(run, "hip_w8a8_matmul", xscales, wscales, bias, residual, gate,
                               target=residual if inplace else None)
    return out.view(m, n) if inplace else out


def hip_w8a8_linear(x: torch.Tensor, qweight: torch.Tensor, wscales: torch.Tensor, bias: torch.Tensor | None = None,
                    *, residual=None, gate=None, inplace: bool = False) -> torch.Tensor:
    """x [..., K] (float32, float16 or bfloat16), quantized row by row, times the int8 weight
    [N, K] -> [..., N] of x's type; residual, gate and inplace as in ConvRotLinear.forward, with one
    rounding at the end."""
    k = x.shape[-1]
    _check_product(k, qweight, wscales, bias)
    nat.on_device(x, qweight, wscales, bias, residual, gate)
    return nat.without_gradient(
        lambda: _linear(x, _operand(qweight, True), _scales(wscales), _scales(bias), k, residual, gate, inplace),
        "hip_w8a8_linear", x, wscales, bias, residual, gate, target=residual if inplace else None)


class Int8Linear(nn.Module):
    """A linear layer stored and executed in 8 bits: `qweight` int8 [N, K], `scales` float32 [N]
    (ones), `bias` float32 [N] (zeros); the output type is the input type.  Of ConvRotLinear's calls it
    has forward and forward_modulated, each with residual=, gate= and inplace=.  It has no gradient: a
    backward pass that reaches it raises an error."""

    def __init__(self, in_features: int, out_features: int, *, bias: bool = True, device=None):
        super().__init__()
        if not 0 < in_features <= MAX_FEATURES:
            raise ValueError(f"W8A8 product needs 1 to {MAX_FEATURES} features, got {in_features}")
        self.in_features, self.out_features = in_features, out_features
        self.register_buffer("qweight", torch.zeros((out_features, in_features), dtype=torch.int8, device=device))
        self.register_buffer("scales", torch.ones((out_features,), dtype=torch.float32, device=device))
        self.register_buffer("bias", torch.zeros((out_features,), dtype=torch.float32, device=device))
        self.source_has_bias = bias
        self._kept_copy: tuple | None = None

    def load_weight(self, weight: torch.Tensor, bias: torch.Tensor | None = None) -> Int8Linear:
        """Quantize a dense (out, in) weight into this layer."""
        if tuple(weight.shape) != (self.out_features, self.in_features):
            raise ValueError(f"weight must have shape {(self.out_features, self.in_features)}, got "
                             f"{tuple(weight.shape)}")
        if bias is not None:
            _check_scales("bias", bias, self.out_features)
        codes, self.scales = quantize_int8_rowwise(weight)
        self.qweight = codes.contiguous()
        if bias is not None:
            self.bias = bias.to(weight.device, torch.float32)
        return self

    def _checked(self, x: torch.Tensor, residual: torch.Tensor | None, *others: torch.Tensor | None) -> tuple:
        """The layer's weight, scales and bias (which may have been assigned anew), after a look whether
        they, x and the residual fit each other and lie on one device: the kernels read as far as these
        shapes say."""
        if x.shape[-1] != self.in_features:
            raise ValueError(f"Int8Linear expected K={self.in_features}, got {x.shape[-1]}")
        if residual is not None and tuple(residual.shape) != (*x.shape[:-1], self.out_features):
            raise ValueError(f"residual {tuple(residual.shape)} must have the output shape "
                             f"{(*x.shape[:-1], self.out_features)}")
        q, scales, bias = self.qweight, self.scales, self.bias
        if _check_product(self.in_features, q, scales, bias) != self.out_features:
            raise ValueError(f"W8A8 weight must have {self.out_features} rows, got {tuple(q.shape)}")
        nat.on_device(x, q, scales, bias, residual, *others)
        return q, scales, bias

    def _weight(self) -> torch.Tensor:
        """The weight as the kernels read it: itself, or where its rows do not lie as they need it
        (in_features no multiple of 16, a strided tensor) a copy with padded rows, kept until the
        tensor or its version is another one."""
        q = self.qweight
        return q if _readable(q, True) else self._copied(q)

    def _copied(self, q: torch.Tensor) -> torch.Tensor:
        # Copies of their own: for a graph, which has to follow the weight from replay to replay and
        # would outlive a kept copy, and for inference tensors, which count no versions.
        if q.is_inference() or (q.is_cuda and torch.cuda.is_current_stream_capturing()):
            return _padded(q)
        kept = self._kept_copy
        # the source is held beside its copy, so no other tensor can take its place unseen
        if kept is None or kept[0] is not q or kept[1] != q._version:
            copy = _padded(q)
            self._kept_copy = (q, q._version, copy, nat.made_here(q.device) if q.is_cuda else None)
            return copy
        return nat.use_here(kept[2], kept[3]) if q.is_cuda else kept[2]

    def __getstate__(self) -> dict:
        return {**self.__dict__, "_kept_copy": None}

    def forward(self, x: torch.Tensor, *, residual: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                inplace: bool = False) -> torch.Tensor:
        """linear(x); with `residual`, residual + gate * linear(x), as ConvRotLinear.forward."""
        q, scales, bias = self._checked(x, residual, gate)
        return nat.without_gradient(
            lambda: _linear(x, q if _readable(q, True) else self._copied(q), _scales(scales), _scales(bias), q.shape[1],
                            residual, gate, inplace),
            "Int8Linear", x, scales, bias, residual, gate, target=residual if inplace else None)

    def forward_modulated(self, x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6, *,
                          residual: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                          inplace: bool = False) -> torch.Tensor:
        """self((1 + scale) * layer_norm(x) + shift), the norm and the quantization in one kernel (the
        normalized row goes to codes unrounded); residual, gate and inplace as in forward."""
        _, scales, bias = self._checked(x, residual, gate, shift, scale)
        return nat.without_gradient(lambda: self._modulated(x, shift, scale, eps, residual, gate, inplace), "Int8Linear", x,
                                    shift, scale, scales, bias, residual, gate, target=residual if inplace else None)

    def _modulated(self, x, shift, scale, eps, residual, gate, inplace) -> torch.Tensor:
        k = self.in_features
        x2d = flat_rows(x)
        m = x2d.shape[0]
        gr = _residual(residual, gate, inplace, m, self.out_features, x.dtype)
        gain, sh, each, _ = norm_operands(x2d, None, None, scale, shift, x.shape)
        codes = torch.empty((m, _round16(k)), dtype=torch.int8, device=x.device)
        scales = torch.empty((m,), dtype=torch.float32, device=x.device)
        nat.check(nat.load().convrot_layer_norm_int8(
            x2d.data_ptr(), nat.dtype_code(x.dtype), m, k, x2d.stride(0), gain.data_ptr(), sh.data_ptr(),
            nat.dtype_code(gain.dtype), 1, each, float(eps), codes.data_ptr(), codes.shape[1], scales.data_ptr(),
            nat.stream_handle(x.device)))
        out = _w8a8(codes, self._weight(), scales, _scales(self.scales), _scales(self.bias), k, x.dtype, gr)
        return residual if inplace else out.reshape(*x.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}"
