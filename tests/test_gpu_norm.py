"""GPU: layer norm and its gradient against the formulas in 64 bits, with bounds of float32
evaluation (tests/_plain64.py), at the sizes of every kernel form and at odd, strided and
non-finite inputs."""

from __future__ import annotations

import pytest
import torch

from _plain64 import assert_within, norm, norm_grads

pytestmark = pytest.mark.gpu
EPS = 1e-6
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def inputs(seed, rows, k, dtype, dev, vectors=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, k), generator=g) * 2 + 0.5
    x[:, :: max(1, k // 7)] *= 20.0
    gain, shift = torch.randn((vectors, k), generator=g) * 0.3, torch.randn((vectors, k), generator=g) * 0.3
    dy = torch.randn((rows, k), generator=g)
    return [t.to(dtype).to(dev) for t in (x, gain, shift, dy)]


def wide(t, vectors, rows):
    return t.double().cpu().repeat_interleave(rows // vectors, dim=0)


SIZES = [(1, 1), (1, 7), (5, 16), (3, 100), (4, 512), (3, 520), (2, 1024), (2, 2048), (3, 2050), (2, 3072), (2, 4104),
         (2, 5120), (1, 6152), (2, 8193), (1, 12288), (1, 16384), (1, 20001), (1, 32768)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,k", SIZES)
def test_affine_forward_and_gradient(dev, rows, k, dtype):
    from convrot_mlx_amd import hip_layer_norm, hip_layer_norm_backward

    x, w, b, dy = inputs(k, rows, k, dtype, dev)
    w, b = w[0] + 1, b[0]
    y, mean, rstd = hip_layer_norm(x, w, b, eps=EPS, return_stats=True)
    assert y.dtype == dtype and mean.dtype == rstd.dtype == F32
    x64, w64, b64 = x.double().cpu(), w.double().cpu()[None], b.double().cpu()[None]
    want, _, _, _, _, off = norm(x64, w64, b64, EPS)
    assert_within(y, want, off, "y")
    assert torch.equal(hip_layer_norm(x, w, b, eps=EPS), y)
    dx, dw, db = hip_layer_norm_backward(dy, x, mean, rstd, weight=w)
    wdx, odx, wdw, odw, wdb, odb = norm_grads(x64, w64, dy.double().cpu(), EPS, 1)
    assert dx.dtype == dw.dtype == db.dtype == dtype and dw.shape == db.shape == (k,)
    assert_within(dx, wdx, odx, "dx")
    assert_within(dw, wdw[0], odw[0], "dw")
    assert_within(db, wdb[0], odb[0], "db")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,k,vectors", [(6, 96, 3), (40, 768, 2), (515, 1024, 5), (77, 3072, 1), (9, 130, 9),
                                            (2000, 64, 1), (600, 1536, 2)])
def test_adaptive_forward_and_gradient(dev, rows, k, vectors, dtype):
    from convrot_mlx_amd import hip_layer_norm, hip_layer_norm_backward

    x, scale, shift, dy = inputs(rows, rows, k, dtype, dev, vectors)
    y, mean, rstd = hip_layer_norm(x, scale=scale[:, None], shift=shift, eps=EPS, return_stats=True)
    x64, g64 = x.double().cpu(), 1 + wide(scale, vectors, rows)
    want, _, _, _, _, off = norm(x64, g64, wide(shift, vectors, rows), EPS)
    assert_within(y, want, off, "y")
    dx, ds, dh = hip_layer_norm_backward(dy, x, mean, rstd, scale=scale)
    wdx, odx, wds, ods, wdh, odh = norm_grads(x64, g64, dy.double().cpu(), EPS, vectors)
    assert ds.shape == dh.shape == (vectors, k)
    assert_within(dx, wdx, odx, "dx")
    assert_within(ds, wds, ods, "dscale")
    assert_within(dh, wdh, odh, "dshift")
    again = hip_layer_norm_backward(dy, x, mean, rstd, scale=scale)
    assert all(torch.equal(a, b) for a, b in zip((dx, ds, dh), again))  # no order of addition is left to chance


def test_parameters_in_float32_and_alone(dev):
    from convrot_mlx_amd import hip_layer_norm, hip_layer_norm_backward

    x, w, b, dy = inputs(3, 33, 640, BF16, dev)
    w32, b32 = w[0].float() + 1.001, b[0].float()
    one, zero = torch.ones(1, 640, dtype=torch.float64), torch.zeros(1, 640, dtype=torch.float64)
    x64 = x.double().cpu()
    for kw, g, s in (({}, one, zero), (dict(weight=w32), w32.double().cpu()[None], zero),
                     (dict(bias=b32), one, b32.double().cpu()[None]),
                     (dict(weight=w32, bias=b32.to(BF16)), w32.double().cpu()[None], b32.to(BF16).double().cpu()[None]),
                     (dict(shift=b32[None]), one, b32.double().cpu()[None])):
        want, _, _, _, _, off = norm(x64, g, s, EPS)
        assert_within(hip_layer_norm(x, eps=EPS, **kw), want, off, str(list(kw)))
    _, mean, rstd = hip_layer_norm(x, w32, b32, eps=EPS, return_stats=True)
    dx, dw, db = hip_layer_norm_backward(dy, x, mean, rstd, weight=w32)
    assert dw.dtype == F32
    wdx, odx, wdw, odw, wdb, odb = norm_grads(x64, w32.double().cpu()[None], dy.double().cpu(), EPS, 1)
    assert_within(dx, wdx, odx), assert_within(dw, wdw[0], odw[0]), assert_within(db, wdb[0], odb[0])
    dx2, n1, n2 = hip_layer_norm_backward(dy, x, mean, rstd, weight=w32, param_grads=False)
    assert n1 is None and n2 is None and torch.equal(dx, dx2)


def test_strided_and_unaligned_rows(dev):
    from convrot_mlx_amd import hip_layer_norm, hip_layer_norm_backward

    base, w, b, dbase = inputs(5, 19, 1040, BF16, dev)
    for at, k in ((0, 1024), (1, 1024), (8, 512), (3, 333)):
        x, dy = base[:, at: at + k], dbase[:, at: at + k]
        y, mean, rstd = hip_layer_norm(x, w[0, :k], b[0, :k], eps=EPS, return_stats=True)
        want, _, _, _, _, off = norm(x.double().cpu(), w[:, :k].double().cpu(), b[:, :k].double().cpu(), EPS)
        assert_within(y, want, off, f"{at} {k}")
        dx, dw, _ = hip_layer_norm_backward(dy, x, mean, rstd, weight=w[0, :k])
        wdx, odx, wdw, odw, _, _ = norm_grads(x.double().cpu(), w[:, :k].double().cpu(), dy.double().cpu(), EPS, 1)
        assert_within(dx, wdx, odx), assert_within(dw, wdw[0], odw[0])
    t = base.t()  # features not adjacent: copied
    assert torch.equal(hip_layer_norm(t), hip_layer_norm(t.contiguous()))
    e = base[:1].expand(7, -1)  # rows at stride 0
    assert torch.equal(hip_layer_norm(e), hip_layer_norm(e.contiguous()))


def test_non_finite_constant_and_empty_rows(dev):
    from convrot_mlx_amd import hip_layer_norm, hip_layer_norm_backward

    x, w, b, dy = inputs(7, 6, 512, BF16, dev)
    x[1, 5], x[2, 9], x[3] = float("nan"), float("inf"), 4.0
    clean = hip_layer_norm(x, w[0], b[0], eps=EPS)
    assert torch.isnan(clean[1]).all() and torch.isnan(clean[2]).all()
    assert torch.equal(clean[3], b[0])  # no variance: the bias alone
    keep = torch.tensor([0, 4, 5], device=dev)
    assert torch.equal(clean[keep], hip_layer_norm(x[keep].contiguous(), w[0], b[0], eps=EPS))
    for rows in (0, 1):
        y, mean, rstd = hip_layer_norm(x[:rows], w[0], b[0], return_stats=True)
        assert y.shape == (rows, 512)
        dx, dw, db = hip_layer_norm_backward(dy[:rows], x[:rows], mean, rstd, weight=w[0])
        assert dx.shape == (rows, 512) and dw.shape == (512,)
        if rows == 0:
            assert not dw.any() and not db.any()


def test_no_features_and_one_dimension(dev):
    from convrot_mlx_amd import hip_layer_norm

    assert hip_layer_norm(torch.zeros((3, 0), device=dev)).shape == (3, 0)
    assert hip_layer_norm(torch.zeros((2, 3, 0), device=dev)).shape == (2, 3, 0)
    x = torch.randn(96, generator=torch.Generator().manual_seed(1)).to(dev)
    assert torch.equal(hip_layer_norm(x), hip_layer_norm(x[None])[0])
    with pytest.raises(ValueError, match="at least one dimension"):
        hip_layer_norm(torch.zeros((), device=dev))


@pytest.mark.parametrize("adaptive", [False, True])
def test_autograd_and_differences(dev, adaptive):
    """The operator's gradients in float32 against the formula, and along one direction against
    central differences of the operator in 64 bits."""
    from convrot_mlx_amd import layer_norm

    x, a, b, dy = inputs(11, 12, 96, F32, dev, 2 if adaptive else 1)
    a, b = (a[:, None], b[:, None]) if adaptive else (a[0] + 1, b[0])
    x3 = x.reshape(2, 6, 96)
    leaves = [t.clone().requires_grad_() for t in (x3, a, b)]
    kw = dict(scale=leaves[1], shift=leaves[2]) if adaptive else dict(weight=leaves[1], bias=leaves[2])
    y = layer_norm(leaves[0], eps=EPS, **kw)
    y.backward(dy.reshape_as(y))
    vectors = 2 if adaptive else 1
    g64 = 1 + wide(a.reshape(2, 96), 2, 12) if adaptive else a.double().cpu()[None]
    wdx, odx, wdg, odg, wdb, odb = norm_grads(x.double().cpu(), g64, dy.double().cpu(), EPS, vectors)
    assert_within(leaves[0].grad.reshape(12, 96), wdx, odx, "dx")
    assert_within(leaves[1].grad.reshape(vectors, 96), wdg, odg, "dgain")
    assert_within(leaves[2].grad.reshape(vectors, 96), wdb, odb, "dshift")
    # f(t) = <dy, norm(x + t d)>: central differences in 64 bits, h = 1e-4, are good to h^2 and eps / h
    d = torch.randn(12, 96, generator=torch.Generator().manual_seed(1)).double()
    zero, h = torch.zeros(1, 96, dtype=torch.float64), 1e-4
    f = lambda t: (dy.double().cpu() * norm(x.double().cpu() + t * d, g64, zero, EPS)[0]).sum()  # noqa: E731
    slope = (f(h) - f(-h)) / (2 * h)
    got = (leaves[0].grad.reshape(12, 96).double().cpu() * d).sum()
    assert abs(got - slope) <= 1e-5 * (wdx.abs() * d.abs()).sum()


def test_only_some_gradients_and_expanded_dy(dev):
    from convrot_mlx_amd import layer_norm

    x, w, b, _ = inputs(13, 8, 64, F32, dev)
    wl = (w[0] + 1).requires_grad_()
    y = layer_norm(x, wl, b[0], eps=EPS)
    y.sum().backward()  # dy is one expanded element
    u = norm(x.double().cpu(), torch.ones(1, 64, dtype=torch.float64), torch.zeros(1, 64, dtype=torch.float64), EPS)
    assert_within(wl.grad, u[3].sum(0), 72 * 2.0 ** -24 * u[3].abs().sum(0) + u[4].sum(0))
    assert x.grad is None
    s = torch.zeros(2, 64, device=dev).requires_grad_()
    layer_norm(x, shift=s, eps=EPS).sum().backward()
    assert torch.equal(s.grad, torch.full((2, 64), 4.0, device=dev))


def test_second_gradient_is_refused(dev):
    from convrot_mlx_amd import layer_norm, qk_rotary

    x = torch.randn((4, 64), device=dev, requires_grad=True)
    first = torch.autograd.grad(layer_norm(x).square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.sum().backward()
    q = torch.randn((1, 2, 3, 16), device=dev, requires_grad=True)
    table = torch.randn((3, 8, 2), device=dev)
    first = torch.autograd.grad(qk_rotary(q, q, table)[0].square().sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.sum().backward()


def test_side_stream_and_graph_replays(dev):
    from convrot_mlx_amd import hip_layer_norm, hip_layer_norm_backward

    x, w, b, dy = inputs(17, 300, 1024, BF16, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        y, mean, rstd = hip_layer_norm(x, w[0], b[0], return_stats=True)
        return (y, *hip_layer_norm_backward(dy, x, mean, rstd, weight=w[0]))

    eager = [t.clone() for t in step()]
    with torch.cuda.stream(side):
        other = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            static = step()
    side.synchronize()
    assert all(torch.equal(a, o) for a, o in zip(eager, other))
    for seed in (1, 2, 3):
        x.copy_(inputs(seed, 300, 1024, BF16, dev)[0])
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, o) for a, o in zip(want, static))


def test_refusals(dev):
    from convrot_mlx_amd import hip_layer_norm, hip_layer_norm_backward

    x, w, b, dy = inputs(19, 6, 64, BF16, dev)
    with pytest.raises(ValueError, match="weight and bias, or scale and shift"):
        hip_layer_norm(x, w[0], scale=w)
    with pytest.raises(ValueError, match="must have 64 features"):
        hip_layer_norm(x, w[0, :32])
    with pytest.raises(ValueError, match="do not split evenly"):
        hip_layer_norm(x, scale=w.expand(4, 64))
    with pytest.raises(ValueError, match="unsupported dtype"):
        hip_layer_norm(x.double())
    with pytest.raises(RuntimeError, match="ROCm device"):
        hip_layer_norm(x.cpu())
    with pytest.raises(ValueError, match="at most 65536 features"):
        hip_layer_norm(torch.zeros(1, 65544, dtype=BF16, device=dev))
    _, mean, rstd = hip_layer_norm(x, return_stats=True)
    with pytest.raises(ValueError, match="shape of x"):
        hip_layer_norm_backward(dy[:3], x, mean, rstd)
    with pytest.raises(ValueError, match="differs from x dtype"):
        hip_layer_norm_backward(dy.float(), x, mean, rstd)
    with pytest.raises(ValueError, match="mean must be"):
        hip_layer_norm_backward(dy, x, mean[:3], rstd)
    with pytest.raises(ValueError, match="at most 32768 features"):
        big = torch.zeros(1, 32776, dtype=BF16, device=dev)
        hip_layer_norm_backward(big, big, mean[:1], rstd[:1])
