"""CPU: the entry points of the 8-bit linears, layer norm and rotary positions refuse invalid
arguments with a status and a message before any launch (no GPU is touched by these calls)."""

from __future__ import annotations

import ctypes

import pytest

P = 4096  # stands for any 16-byte aligned device address: never read
BF16, F32 = 2, 0


@pytest.fixture(scope="module")
def lib():
    from convrot_mlx_amd import _native

    return _native.load()


def refused(lib, status, code, text):
    assert status == code, lib.convrot_last_error()
    assert text in lib.convrot_last_error().decode()


def quantize(lib, **kw):
    a = dict(x=P, dtype=BF16, rows=4, k=64, stride=64, codes=P, cstride=64, scales=P) | kw
    return lib.convrot_quantize_int8(a["x"], a["dtype"], a["rows"], a["k"], a["stride"], a["codes"], a["cstride"],
                                     a["scales"], None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=9), 1, "dtype code"), (dict(rows=-1), 1, "invalid shape"), (dict(k=65537, cstride=65552), 2, "at most"),
    (dict(x=None), 1, "null"), (dict(x=P + 1), 1, "aligned to its type"), (dict(codes=None), 1, "null"),
    (dict(codes=P + 8), 1, "16-byte aligned rows"), (dict(cstride=48), 1, "16-byte aligned rows"),
    (dict(cstride=72), 1, "16-byte aligned rows"), (dict(cstride=2048), 2, "too long"), (dict(stride=-64), 1, "negative"),
])
def test_quantizer(lib, kw, code, text):
    refused(lib, quantize(lib, **kw), code, text)


def test_nothing_to_do_is_no_error(lib):
    assert quantize(lib, rows=0, x=None, codes=None) == 0
    assert gemm(lib, m=0, act=None) == 0 and gemm(lib, n=0, weight=None) == 0
    assert norm(lib, rows=0, x=None, out=None, each=1) == 0
    assert rotary(lib, batch=0, q=None) == 0 and rotary(lib, length=0, q=None) == 0
    assert lib.convrot_axes_table(None, 0, 0, 1, (ctypes.c_int * 1)(4), 1e4, None, None) == 0


def gemm(lib, **kw):
    a = dict(act=P, lda=64, xs=P, weight=P, ldw=64, ws=P, bias=P, m=4, n=8, k=64, res=None, gate=None, gs=0, rpg=1,
             work=None, wb=0, out=P, dt=BF16) | kw
    return lib.convrot_w8a8_gemm(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dt=7), 1, "dtype code"), (dict(k=0), 1, "invalid GEMM shape"), (dict(m=-1), 1, "invalid GEMM shape"),
    (dict(k=65552, lda=65552, ldw=65552), 2, "K up to"), (dict(act=None), 1, "null"), (dict(out=None), 1, "null"),
    (dict(lda=48), 1, "16-byte aligned rows"), (dict(ldw=72), 1, "16-byte aligned rows"), (dict(act=P + 4), 1, "aligned"),
    (dict(weight=P + 4), 1, "aligned"), (dict(out=P + 8), 1, "aligned"), (dict(ldw=1 << 23), 2, "limited"),
    (dict(lda=1 << 23), 2, "limited"), (dict(gate=P), 1, "gate needs a residual"),
    (dict(gate=P, res=P, rpg=0), 1, "rows_per_gate"), (dict(res=P + 2), 1, "aligned"),
    (dict(gate=P, res=P, rpg=2, gs=4), 1, "overlap"), (dict(wb=64), 1, "workspace"), (dict(work=P + 8, wb=64), 1, "256-byte"),
    (dict(m=0x7fffffff), 2, "too large"),
])
def test_product(lib, kw, code, text):
    refused(lib, gemm(lib, **kw), code, text)


def test_linear_scratch(lib):
    assert lib.convrot_w8a8_scratch_bytes(5, 100) == 5 * 128 + 20
    assert lib.convrot_w8a8_scratch_bytes(0, 100) == 0
    assert lib.convrot_w8a8_fused(P, BF16, 1, 4096, 4096) == 1
    assert lib.convrot_w8a8_fused(P, BF16, 17, 64, 64) == 0  # more rows than the kernel holds
    assert lib.convrot_w8a8_fused(P + 2, BF16, 1, 64, 64) == 0
    assert lib.convrot_w8a8_fused(P, BF16, 1, 72, 72) == 0
    far = 1 << 30
    args = lambda m, scratch, nbytes, out: (P, BF16, 64, P, 64, P, None, m, 8, 64, None, None, 0, 1, scratch,  # noqa: E731
                                            nbytes, None, 0, out, None)
    refused(lib, lib.convrot_w8a8_linear(*args(40, None, 0, far)), 1, "scratch buffer of 5280 bytes")
    refused(lib, lib.convrot_w8a8_linear(*args(40, P, 5279, far)), 1, "scratch buffer")
    refused(lib, lib.convrot_w8a8_linear(*args(40, P + 4, 6000, far)), 1, "scratch buffer")
    refused(lib, lib.convrot_w8a8_linear(*args(2, None, 0, P)), 1, "scratch buffer")  # out over x: not in one launch


def norm(lib, **kw):
    a = dict(x=P, dtype=BF16, rows=6, k=64, stride=64, gain=P, shift=P, pdt=BF16, one=0, each=3, eps=1e-6, out=P,
             mean=None, rstd=None) | kw
    return lib.convrot_layer_norm(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=5), 1, "dtype code"), (dict(k=65537), 2, "at most"), (dict(x=None), 1, "null"), (dict(out=None), 1, "null"),
    (dict(pdt=1), 1, "norm parameters"), (dict(each=4), 1, "do not split"), (dict(each=0), 1, "do not split"),
    (dict(mean=P), 1, "come together"), (dict(gain=P + 1), 1, "not aligned"), (dict(out=P + 1), 1, "not aligned"),
])
def test_norm(lib, kw, code, text):
    refused(lib, norm(lib, **kw), code, text)


def test_norm_gradient(lib):
    need = lib.convrot_layer_norm_workspace_bytes(6, 64, 3)
    assert need >= 2 * 2 * 64 * 4 and need % (2 * 64 * 4) == 0
    assert lib.convrot_layer_norm_workspace_bytes(6, 64, 4) == 0

    def call(**kw):
        a = dict(dy=P, ds=64, x=P, xs=64, mean=P, rstd=P, dtype=BF16, rows=6, k=64, gain=P, pdt=BF16, one=0, each=3,
                 dx=P, dg=P, db=P, work=P, wb=need) | kw
        return lib.convrot_layer_norm_backward(*a.values(), None)

    refused(lib, call(k=32769), 2, "at most 32768")
    refused(lib, call(wb=need - 1), 1, "workspace")
    refused(lib, call(work=None), 1, "workspace")
    refused(lib, call(work=P + 8), 1, "workspace")
    refused(lib, call(mean=None), 1, "null")
    refused(lib, call(dy=None), 1, "null")
    refused(lib, call(each=0), 1, "rows_per_vector")
    refused(lib, call(each=4), 1, "do not split")


def rotary(lib, **kw):
    a = dict(q=P, k=P, qo=P, ko=P, st=(ctypes.c_int64 * 12)(*[64] * 12), dtype=BF16, batch=1, hq=2, hk=1, length=3, dim=64,
             table=P, pairs=32, ts=0, qw=None, kw=None, wdt=BF16, eps=1e-6, inter=1) | kw
    return lib.convrot_qk_rotary(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=4), 1, "dtype code"), (dict(hq=-1), 1, "invalid rotary shape"), (dict(pairs=33), 1, "do not fit"),
    (dict(dim=516), 2, "up to 512"), (dict(q=None), 1, "null"), (dict(ko=None), 1, "null"), (dict(table=None), 1, "null"),
    (dict(st=None), 1, "null"), (dict(qw=P, wdt=1), 1, "norm weights"), (dict(ts=-1), 1, "rotary table"),
    (dict(batch=1 << 16, length=1 << 16), 2, "at most"),
])
def test_rotary(lib, kw, code, text):
    refused(lib, rotary(lib, **kw), code, text)


def test_rotary_gradient_and_table(lib):
    need = lib.convrot_qk_rotary_workspace_bytes(64)
    assert need > 0 and lib.convrot_qk_rotary_workspace_bytes(513) == 0
    st = (ctypes.c_int64 * 18)(*[64] * 18)

    def call(qw, gqw, work, nbytes):
        return lib.convrot_qk_rotary_backward(P, P, P, P, P, P, gqw, None, st, BF16, 1, 2, 1, 3, 64, P, 32, 0, qw, None,
                                              BF16, 1e-6, 1, work, nbytes, None)

    refused(lib, call(None, P, P, need), 1, "needs the weight")
    refused(lib, call(P, P, None, 0), 1, "workspace")
    refused(lib, call(P, P, P, need - 1), 1, "workspace")
    dims = lambda *d: (ctypes.c_int * len(d))(*d)  # noqa: E731
    refused(lib, lib.convrot_axes_table(P, 9, 3, 1, dims(4), 1e4, P, None), 1, "position type")
    refused(lib, lib.convrot_axes_table(P, 0, 3, 1, dims(5), 1e4, P, None), 1, "even number")
    refused(lib, lib.convrot_axes_table(P, 0, 3, 9, dims(*[2] * 9), 1e4, P, None), 1, "1 to 8 axes")
    refused(lib, lib.convrot_axes_table(P, 0, 3, 1, dims(4), 0.0, P, None), 1, "theta")
    refused(lib, lib.convrot_axes_table(None, 0, 3, 1, dims(4), 1e4, P, None), 1, "null")


def test_tuning_names(lib):
    assert lib.convrot_set_tuning(b"w8a8_tile", b"256x256") == 0 and lib.convrot_set_tuning(b"w8a8_tile", None) == 0
    assert lib.convrot_set_tuning(b"w8a8_split", b"4") == 0 and lib.convrot_set_tuning(b"w8a8_split", None) == 0
    refused(lib, lib.convrot_set_tuning(b"w8a8_tile", b"100x100"), 1, "invalid value")
    refused(lib, lib.convrot_set_tuning(b"w8a8_split", b"65"), 1, "invalid value")
