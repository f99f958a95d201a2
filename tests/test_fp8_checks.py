"""CPU: what the 8-bit floating point linears refuse before any launch."""

from __future__ import annotations

import pytest
import torch

from convrot_mlx_amd import Fp8Linear, hip_fp8_linear, hip_fp8_matmul, quantize_fp8_blockwise, quantize_fp8_weight

P = 4096  # stands for any 16-byte aligned device address: never read
BF16 = 2
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    from convrot_mlx_amd import _native

    return _native.load()


def refused(lib, status, code, text):
    assert status == code, lib.convrot_last_error()
    assert text in lib.convrot_last_error().decode()


def quantize(lib, **kw):
    a = dict(x=P, dtype=BF16, rows=4, k=64, stride=64, codes=P, cstride=64, scales=P, row=1, block=4) | kw
    return lib.convrot_quantize_fp8(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=9), 1, "dtype code"), (dict(rows=-1), 1, "invalid shape"), (dict(k=65537, cstride=65552), 2, "at most"),
    (dict(x=None), 1, "null"), (dict(x=P + 1), 1, "aligned to its type"), (dict(codes=None), 1, "null"),
    (dict(scales=None), 1, "null"), (dict(codes=P + 8), 1, "16-byte aligned rows"), (dict(cstride=48), 1, "at least 64"),
    (dict(cstride=72), 1, "16-byte aligned rows"), (dict(cstride=1 << 23), 2, "limited"), (dict(row=0), 1, "strides"),
    (dict(block=0), 1, "strides"), (dict(stride=-64), 1, "negative"),
])
def test_quantizer(lib, kw, code, text):
    refused(lib, quantize(lib, **kw), code, text)


def test_weight_quantizer(lib):
    call = lambda *a: lib.convrot_quantize_fp8_weight(*a, None)  # noqa: E731
    refused(lib, call(P, 7, 4, 64, 64, P, 64, P), 1, "dtype code")
    refused(lib, call(P, BF16, 4, 64, 64, P, 60, P), 1, "16-byte aligned rows")
    refused(lib, call(P, BF16, 4, 64, 64, P, 64, None), 1, "null")
    assert call(None, BF16, 0, 64, 64, None, 64, None) == 0


def gemm(lib, **kw):
    a = dict(act=P, lda=64, xs=P, xr=1, xb=4, weight=P, ldw=64, ws=P, wr=1, bias=P, m=4, n=8, k=64, res=None, gate=None,
             gs=0, rpg=1, work=None, wb=0, out=P, dt=BF16) | kw
    return lib.convrot_fp8_gemm(*a.values(), None)


PRODUCT = [
    (dict(dt=7), 1, "dtype code"), (dict(k=0), 1, "invalid GEMM shape"), (dict(m=-1), 1, "invalid GEMM shape"),
    (dict(k=65552, lda=65552, ldw=65552, wr=600), 2, "K up to"), (dict(weight=None), 1, "null"), (dict(ws=None), 1, "null"),
    (dict(out=None), 1, "null"), (dict(ldw=72), 1, "16-byte aligned rows"), (dict(ldw=48), 1, "16-byte aligned rows"),
    (dict(weight=P + 4), 1, "aligned"), (dict(out=P + 8), 1, "aligned"), (dict(ldw=1 << 23), 2, "limited"),
    (dict(wr=0), 1, "weight scales"), (dict(ws=P + 2), 1, "weight scales"), (dict(m=0x7fffffff), 2, "too large"),
]


@pytest.mark.parametrize("kw,code,text", PRODUCT + [
    (dict(act=None), 1, "null"), (dict(xs=None), 1, "null"), (dict(lda=48), 1, "16-byte aligned rows"),
    (dict(act=P + 4), 1, "aligned"), (dict(lda=1 << 23), 2, "limited"), (dict(xr=-1), 2, "strides of activation scales"),
    (dict(xr=1 << 22), 2, "strides of activation scales"), (dict(gate=P), 1, "gate needs a residual"),
    (dict(gate=P, res=P, rpg=0), 1, "rows_per_gate"), (dict(res=P + 2), 1, "aligned"), (dict(gate=P, res=P, rpg=2, gs=4), 1, "overlap"),
    (dict(wb=64), 1, "workspace"), (dict(work=P + 8, wb=64), 1, "256-byte"),
])
def test_product(lib, kw, code, text):
    refused(lib, gemm(lib, **kw), code, text)


def test_linear_scratch(lib):
    assert lib.convrot_fp8_scratch_bytes(5, 100) == 5 * 128 + 8 * 4
    assert lib.convrot_fp8_scratch_bytes(0, 100) == 0

    def call(scratch, nbytes):
        return lib.convrot_fp8_linear(P, BF16, 64, P, 64, P, 1, None, 40, 8, 64, None, None, 0, 1, scratch, nbytes, None, 0,
                                      P, None)

    need = lib.convrot_fp8_scratch_bytes(40, 64)
    for scratch, nbytes in ((None, 0), (P, need - 1), (P + 4, need)):
        refused(lib, call(scratch, nbytes), 1, f"scratch buffer of {need} bytes")


def test_nothing_to_do_is_no_error(lib):
    assert quantize(lib, rows=0, x=None, codes=None) == 0
    assert gemm(lib, m=0, act=None) == 0 and gemm(lib, n=0, weight=None) == 0
    assert lib.convrot_fp8_workspace_bytes(0, 8, 64) == 0


def test_tuning_names(lib):
    assert lib.convrot_set_tuning(b"fp8_tile", b"256x256") == 0 and lib.convrot_set_tuning(b"fp8_tile", None) == 0
    assert lib.convrot_set_tuning(b"fp8_split", b"4") == 0 and lib.convrot_set_tuning(b"fp8_split", None) == 0
    refused(lib, lib.convrot_set_tuning(b"fp8_tile", b"100x100"), 1, "invalid value")
    refused(lib, lib.convrot_set_tuning(b"fp8_split", b"65"), 1, "invalid value")


def f8(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(FP8)


@pytest.mark.parametrize("w,ws,bias,text", [
    (torch.zeros(6, 32), torch.ones(1, 1), None, "float8_e4m3fn"), (f8(6, 48), torch.ones(1, 1), None, "K=32"),
    (f8(6, 32), torch.ones(1), None, "weight scales must have shape"), (f8(6, 32), torch.ones(2, 1), None, "weight scales"),
    (f8(6, 32), torch.ones(1, 1), torch.ones(5), "bias must have shape"), (f8(2, 6, 32), torch.ones(1, 1), None, "2D"),
])
def test_operands(w, ws, bias, text):
    x = torch.zeros(2, 32)
    with pytest.raises(ValueError, match=text):
        hip_fp8_linear(x, w, ws, bias)
    with pytest.raises(ValueError, match=text):
        hip_fp8_matmul(f8(2, 32), w, torch.ones(2, 1), ws, bias, output_dtype=torch.float32)
    layer = Fp8Linear(32, 6)
    layer.qweight, layer.scales = w, ws
    if bias is not None:
        layer.bias = bias
    for call in (lambda: layer(x), lambda: layer(x, residual=torch.zeros(2, 6))):
        with pytest.raises(ValueError, match=text):
            call()


def test_activations():
    w, ws = f8(6, 32), torch.ones(1, 1)
    with pytest.raises(ValueError, match="activation must be 2D float8_e4m3fn"):
        hip_fp8_matmul(torch.zeros(2, 32), w, torch.ones(2, 1), ws, output_dtype=torch.float32)
    with pytest.raises(ValueError, match="activation scales"):
        hip_fp8_matmul(f8(2, 32), w, torch.ones(2), ws, output_dtype=torch.float32)
    with pytest.raises(ValueError, match="unsupported dtype"):
        hip_fp8_matmul(f8(2, 32), w, torch.ones(2, 1), ws, output_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hip_fp8_linear(torch.zeros(2, 32), w, ws)
    for call in (quantize_fp8_blockwise, quantize_fp8_weight):
        with pytest.raises(ValueError):
            call(torch.zeros(4))
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call(torch.zeros(4, 4))
    with pytest.raises(ValueError, match="expected K=32"):
        Fp8Linear(32, 6)(torch.zeros(2, 31))
    with pytest.raises(ValueError, match="output shape"):
        Fp8Linear(32, 6)(torch.zeros(2, 32), residual=torch.zeros(12))
    with pytest.raises(ValueError, match="1 to 65536"):
        Fp8Linear(0, 6)
    with pytest.raises(ValueError, match="weight must have shape"):
        Fp8Linear(32, 6).load_weight(torch.zeros(5, 32))


def test_casts_keep_codes_and_scales():
    layer = Fp8Linear(32, 6)
    layer.qweight.view(torch.uint8).random_(0, 120)
    want = layer.qweight.view(torch.uint8).clone()
    for cast in (layer.half, layer.bfloat16, layer.double, lambda: layer.to(torch.float16)):
        cast()
        assert layer.qweight.dtype == FP8 and torch.equal(layer.qweight.view(torch.uint8), want)
        assert layer.scales.dtype == torch.float32 and layer.bias.dtype == torch.float32
