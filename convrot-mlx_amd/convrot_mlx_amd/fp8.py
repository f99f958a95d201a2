"""Linears in 8-bit floating point: e4m3 codes with a float32 scale for each block of 128.

Activations have a scale for each 128 features of a row, weights one for each 128 x 128, as 8-bit
checkpoints hold them.  The quantizers here take powers of two (scale = the smallest one with
absmax / scale <= 448), so that a value over its scale is exact and the code is its one rounding;
the product takes any scales:

    out[m, n] = sum_b (xs[m, b] ws[n // 128, b]) * (sum of block b's products of codes) + bias[n]

with float32 sums, a gated residual in float32 and one rounding.  (For 16-bit outputs the matrix
units' FP8 form cuts a product 13 bits below the largest of its 16 neighbours, which is 2e-5 of a
sum; float32 outputs are summed at float32 throughout.)  No counterpart in the reference, which
quantizes to 4 bits only.
"""

from __future__ import annotations

import torch
from torch import nn

from . import _native as nat
from .core import _f32, _workspace
from .int8 import _CONTROL_BYTES, _output, _residual, _residual_args
from .norm import flat_rows, hip_layer_norm, rows_of

BLOCK = 128
MAX_FEATURES = 65536
MAX_ROW_STRIDE = 1 << 22
MAX_SCALE_STRIDE = 1 << 21
CODES = torch.float8_e4m3fn


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def quantize_fp8_blockwise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of x [M, K] (any strides) as (float8_e4m3fn codes [M, K], float32 scales [M, ceil(K / 128)]),
    both views of padded memory, laid out as the product reads them.

    The scales are powers of two.  A block that holds a NaN or an infinity gets the scale NaN (its
    products are NaN); one whose largest magnitude is below 2^-100 counts as zero."""
    if x.ndim != 2:
        raise ValueError(f"blockwise fp8 quantization expects 2D input, got {tuple(x.shape)}")
    nat.require_device(x)
    x = rows_of(x)
    m, k = x.shape
    blocks = _blocks(k)
    codes = torch.empty((m, blocks * BLOCK), dtype=torch.uint8, device=x.device)
    scales = torch.empty((blocks, m), dtype=torch.float32, device=x.device)
    with nat.on(x.device):
        nat.check(nat.load().convrot_quantize_fp8(x.data_ptr(), nat.dtype_code(x.dtype), m, k, x.stride(0),
                                                  codes.data_ptr(), max(16, codes.shape[1]), scales.data_ptr(), 1,
                                                  max(1, m), nat.stream_handle(x.device)))
    return codes.view(CODES)[:, :k], scales.t()


def quantize_fp8_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """A dense weight [N, K], or experts' [E, N, K], as (float8_e4m3fn codes of its shape, float32 scales
    [.., ceil(N / 128), ceil(K / 128)]): one scale, a power of two, for each 128 x 128."""
    if weight.ndim not in (2, 3):
        raise ValueError(f"fp8 weights are [N, K] or [E, N, K], got {tuple(weight.shape)}")
    nat.require_device(weight)
    *lead, n, k = weight.shape
    pad = (k + 15) // 16 * 16
    codes = torch.zeros((*lead, n, pad), dtype=torch.uint8, device=weight.device)
    scales = torch.zeros((*lead, _blocks(n), _blocks(k)), dtype=torch.float32, device=weight.device)
    with nat.on(weight.device):
        for e in range(lead[0] if lead else 1):
            w, c, s = (weight, codes, scales) if not lead else (weight[e], codes[e], scales[e])
            w = rows_of(w)
            nat.check(nat.load().convrot_quantize_fp8_weight(w.data_ptr(), nat.dtype_code(w.dtype), n, k, w.stride(0),
                                                             c.data_ptr(), max(16, pad), s.data_ptr(),
                                                             nat.stream_handle(weight.device)))
    return codes.view(CODES)[..., :k].contiguous(), scales


def _row_stride(t: torch.Tensor) -> int:
    """Bytes between an operand's rows (the stride of a single row says nothing)."""
    return t.stride(-2) if t.shape[-2] > 1 else (t.shape[-1] + 15) // 16 * 16


def _operand(t: torch.Tensor) -> torch.Tensor:
    """Codes [.., K] as the product reads them, itself or a copy: adjacent features, rows (and experts)
    16-byte aligned, zeros from K to the next multiple of 16."""
    k = t.shape[-1]
    if k % 16 == 0 and t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        stride = _row_stride(t)
        if (t.stride(-1) == 1 and stride % 16 == 0 and k <= stride <= MAX_ROW_STRIDE
                and (t.ndim == 2 or t.shape[0] == 1 or (t.stride(0) % 16 == 0 and t.stride(0) >= 0))):
            return t
    padded = torch.zeros((*t.shape[:-1], (k + 15) // 16 * 16), dtype=torch.uint8, device=t.device)
    padded[..., :k] = t.view(torch.uint8)
    return padded.view(CODES)


def _check_weight(k: int, weight: torch.Tensor, wscales: torch.Tensor, dims: int) -> int:
    what = "N x K" if dims == 2 else "E x N x K"
    if weight.ndim != dims or weight.dtype != CODES:
        raise ValueError(f"FP8 weight must be {dims}D float8_e4m3fn ({what}), got {tuple(weight.shape)} {weight.dtype}")
    n = weight.shape[-2]
    if weight.shape[-1] != k:
        raise ValueError(f"FP8 weight must be {what} with K={k}, got {tuple(weight.shape)}")
    if not 0 < k <= MAX_FEATURES:
        raise ValueError(f"FP8 product needs 1 to {MAX_FEATURES} features, got {k}")
    want = (*weight.shape[:-2], _blocks(n), _blocks(k))
    if tuple(wscales.shape) != want:
        raise ValueError(f"FP8 weight scales must have shape {want}, got {tuple(wscales.shape)}")
    return n


def _check_bias(bias: torch.Tensor | None, n: int) -> None:
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"FP8 bias must have shape {(n,)}, got {tuple(bias.shape)}")


def _weight_scales(t: torch.Tensor) -> torch.Tensor:
    """float32 scales with adjacent blocks of features and whole rows."""
    if t.dtype == torch.float32 and t.is_contiguous():
        return t
    return t.to(torch.float32).contiguous()


def _vector(t: torch.Tensor | None) -> torch.Tensor | None:
    return t if t is None or (t.dtype == torch.float32 and t.is_contiguous()) else _f32(t).contiguous()


def _product_workspace(device, stream: int, m: int, n: int, k: int) -> torch.Tensor | None:
    """Counters and partial sums of a product whose workgroups share K: the stream's, or, as a graph may be
    replayed beside that stream and beside other graphs, memory of the graph's own."""
    if not torch.cuda.is_current_stream_capturing():
        return _workspace(device, stream)
    need = nat.load().convrot_fp8_workspace_bytes(m, n, k)
    if need == 0:
        return None
    work = torch.empty((need,), dtype=torch.uint8, device=device)
    work[:_CONTROL_BYTES].zero_()
    return work


def _linear(x, weight, wscales, bias, k: int, residual, gate, inplace: bool) -> torch.Tensor:
    """x [..., k] times a weight as the kernel reads it, one library call."""
    n, device = weight.shape[0], x.device
    x2d = flat_rows(x)
    m = x2d.shape[0]
    gr = _residual(residual, gate, inplace, m, n, x.dtype)
    out = _output(gr, m, n, x.dtype, device)
    lib = nat.load()
    with nat.on(device):
        stream = nat.stream_handle(device)
        work = _product_workspace(device, stream, m, n, k)
        need = lib.convrot_fp8_scratch_bytes(m, k)
        scratch = torch.empty((need,), dtype=torch.uint8, device=device)
        nat.check(lib.convrot_fp8_linear(
            x2d.data_ptr(), nat.dtype_code(x.dtype), x2d.stride(0), weight.data_ptr(), _row_stride(weight),
            wscales.data_ptr(), wscales.shape[1], nat.address(bias), m, n, k, *_residual_args(gr), scratch.data_ptr(), need,
            nat.address(work), 0 if work is None else work.numel(), out.data_ptr(), stream))
    if inplace:
        return residual
    return out if x.ndim == 2 else out.reshape(*x.shape[:-1], n)


def hip_fp8_matmul(qact: torch.Tensor, qweight: torch.Tensor, xscales: torch.Tensor, wscales: torch.Tensor,
                   bias: torch.Tensor | None = None, *, output_dtype: torch.dtype, residual=None, gate=None,
                   inplace: bool = False) -> torch.Tensor:
    """float8_e4m3fn activations [M, K] with scales [M, ceil(K / 128)] (any strides) x weight [N, K] with
    scales [ceil(N / 128), ceil(K / 128)] -> output_dtype [M, N]; residual, gate and inplace as in
    hip_w8a8_matmul.  Any float32 scales; K no multiple of 16 copies both operands into padded rows."""
    if qact.ndim != 2 or qact.dtype != CODES:
        raise ValueError(f"FP8 activation must be 2D float8_e4m3fn, got {tuple(qact.shape)} {qact.dtype}")
    m, k = qact.shape
    n = _check_weight(k, qweight, wscales, 2)
    _check_bias(bias, n)
    if tuple(xscales.shape) != (m, _blocks(k)):
        raise ValueError(f"FP8 activation scales must have shape {(m, _blocks(k))}, got {tuple(xscales.shape)}")
    dtype = nat.dtype_code(output_dtype)
    device = nat.on_device(qact, qweight, xscales, wscales, bias, residual, gate)
    gr = _residual(residual, gate, inplace, m, n, output_dtype)

    def run():
        a, w = _operand(qact), _operand(qweight)
        xs, ws, b = xscales.to(torch.float32), _weight_scales(wscales), _vector(bias)
        if min(xs.stride()) < 0 or xs.stride(0) > MAX_SCALE_STRIDE:
            xs = xs.contiguous()
        out = _output(gr, m, n, output_dtype, device)
        with nat.on(device):
            stream = nat.stream_handle(device)
            work = _product_workspace(device, stream, m, n, k)
            nat.check(nat.load().convrot_fp8_gemm(
                a.data_ptr(), _row_stride(a), xs.data_ptr(), xs.stride(0), xs.stride(1), w.data_ptr(), _row_stride(w),
                ws.data_ptr(), ws.shape[1], nat.address(b), m, n, k, *_residual_args(gr), nat.address(work),
                0 if work is None else work.numel(), out.data_ptr(), dtype, stream))
        return residual if inplace else out

    out = nat.without_gradient(run, "hip_fp8_matmul", xscales, wscales, bias, residual, gate,
                               target=residual if inplace else None)
    return out.view(m, n) if inplace else out


def hip_fp8_linear(x: torch.Tensor, qweight: torch.Tensor, wscales: torch.Tensor, bias: torch.Tensor | None = None,
                   *, residual=None, gate=None, inplace: bool = False) -> torch.Tensor:
    """x [..., K] (float32, float16 or bfloat16), quantized in blocks of 128, times the float8_e4m3fn weight
    [N, K] with scales [ceil(N / 128), ceil(K / 128)] -> [..., N] of x's type; residual, gate and inplace as
    in ConvRotLinear.forward, with one rounding at the end."""
    k = x.shape[-1]
    _check_bias(bias, _check_weight(k, qweight, wscales, 2))
    nat.on_device(x, qweight, wscales, bias, residual, gate)
    return nat.without_gradient(
        lambda: _linear(x, _operand(qweight), _weight_scales(wscales), _vector(bias), k, residual, gate, inplace),
        "hip_fp8_linear", x, wscales, bias, residual, gate, target=residual if inplace else None)


class Fp8Buffers(nn.Module):
    """A module whose buffers hold codes and their float32 scales (and bias)."""

    def _apply(self, fn, recurse=True):
        # .half(), .bfloat16() and .to(dtype) cast parameters and buffers of floating types: the codes and
        # their scales stay what they are and only move
        kept = dict(self._buffers)
        super()._apply(fn, recurse)
        for name, t in kept.items():
            if t is not None and self._buffers[name].dtype != t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self


class Fp8Linear(Fp8Buffers):
    """A linear layer stored and executed in 8-bit floating point: `qweight` float8_e4m3fn [N, K], `scales`
    float32 [ceil(N / 128), ceil(K / 128)] (ones), `bias` float32 [N] (zeros); the output type is the input
    type.  It has forward and forward_modulated, each with residual=, gate= and inplace=, and no gradient: a
    backward pass that reaches it raises an error."""

    def __init__(self, in_features: int, out_features: int, *, bias: bool = True, device=None):
        super().__init__()
        if not 0 < in_features <= MAX_FEATURES:
            raise ValueError(f"FP8 product needs 1 to {MAX_FEATURES} features, got {in_features}")
        self.in_features, self.out_features = in_features, out_features
        self.register_buffer("qweight", torch.zeros((out_features, in_features), dtype=torch.uint8,
                                                    device=device).view(CODES))
        self.register_buffer("scales", torch.ones((_blocks(out_features), _blocks(in_features)), dtype=torch.float32,
                                                  device=device))
        self.register_buffer("bias", torch.zeros((out_features,), dtype=torch.float32, device=device))
        self.source_has_bias = bias

    def load_weight(self, weight: torch.Tensor, bias: torch.Tensor | None = None) -> Fp8Linear:
        """Quantize a dense (out, in) weight into this layer."""
        if tuple(weight.shape) != (self.out_features, self.in_features):
            raise ValueError(f"weight must have shape {(self.out_features, self.in_features)}, got "
                             f"{tuple(weight.shape)}")
        _check_bias(bias, self.out_features)
        self.qweight, self.scales = quantize_fp8_weight(weight)
        if bias is not None:
            self.bias = bias.to(weight.device, torch.float32)
        return self

    def forward(self, x: torch.Tensor, *, residual: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                inplace: bool = False) -> torch.Tensor:
        """linear(x); with `residual`, residual + gate * linear(x), as ConvRotLinear.forward."""
        if x.shape[-1] != self.in_features:
            raise ValueError(f"Fp8Linear expected K={self.in_features}, got {x.shape[-1]}")
        if residual is not None and tuple(residual.shape) != (*x.shape[:-1], self.out_features):
            raise ValueError(f"residual {tuple(residual.shape)} must have the output shape "
                             f"{(*x.shape[:-1], self.out_features)}")
        q, scales, bias = self.qweight, self.scales, self.bias
        if _check_weight(self.in_features, q, scales, 2) != self.out_features:
            raise ValueError(f"FP8 weight must have {self.out_features} rows, got {tuple(q.shape)}")
        _check_bias(bias, self.out_features)
        nat.on_device(x, q, scales, bias, residual, gate)
        return nat.without_gradient(
            lambda: _linear(x, _operand(q), _weight_scales(scales), _vector(bias), q.shape[1], residual, gate, inplace),
            "Fp8Linear", x, scales, bias, residual, gate, target=residual if inplace else None)

    def forward_modulated(self, x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6, *,
                          residual: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                          inplace: bool = False) -> torch.Tensor:
        """self((1 + scale) * layer_norm(x) + shift), the norm as hip_layer_norm rounds it; residual, gate and
        inplace as in forward."""
        def normed():
            with nat.on(x.device):  # as the linear itself
                return hip_layer_norm(x, scale=scale, shift=shift, eps=eps)

        return self(nat.without_gradient(normed, "Fp8Linear", x, shift, scale), residual=residual, gate=gate,
                    inplace=inplace)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}"
