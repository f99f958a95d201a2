"""GPU: rotary positions of several axes with the head norm, and their gradients, against the
formulas in 64 bits (tests/_plain64.py)."""

from __future__ import annotations

import pytest
import torch

from _plain64 import assert_within, rotary, rotary_grads

pytestmark = pytest.mark.gpu
EPS = 1e-6
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(seed, b, hq, hk, length, d, pairs, dtype, dev, table_batch=None):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn((b, length, (hq + 2 * hk) * d), generator=g) * 1.5).to(dtype).to(dev)
    q = qkv[..., : hq * d].unflatten(-1, (hq, d)).transpose(1, 2)
    k = qkv[..., hq * d: (hq + hk) * d].unflatten(-1, (hk, d)).transpose(1, 2)
    ang = torch.randn((table_batch or b, length, pairs), generator=g).double() * 10
    table = torch.stack([ang.cos(), ang.sin()], -1).float().to(dev)
    qw, kw = ((1 + 0.2 * torch.randn((d,), generator=g)).to(dtype).to(dev) for _ in range(2))
    dq, dk = (torch.randn((b, h, length, d), generator=g).to(dtype).to(dev) for h in (hq, hk))
    return q, k, table, qw, kw, dq, dk


def check(q, k, table, qw, kw, dq, dk, interleaved):
    from convrot_mlx_amd import hip_qk_rotary, hip_qk_rotary_backward

    kwargs = dict(q_weight=qw, k_weight=kw, eps=EPS, interleaved=interleaved)
    t64 = table.double().cpu()
    t64 = t64[None] if t64.ndim == 3 else t64
    outs = hip_qk_rotary(q, k, table, **kwargs)
    grads = hip_qk_rotary_backward(dq, dk, q, k, table, **kwargs)
    for i, (x, w, dy) in enumerate(((q, qw, dq), (k, kw, dk))):
        w64 = None if w is None else w.double().cpu()
        want, off = rotary(x.double().cpu(), w64, t64, EPS, interleaved)
        assert outs[i].dtype == x.dtype and outs[i].is_contiguous()
        assert_within(outs[i], want, off, f"out {i}")
        dx, odx, dw, odw = rotary_grads(x.double().cpu(), w64, t64, dy.double().cpu(), EPS, interleaved)
        assert_within(grads[i], dx, odx, f"grad {i}")
        if w is None:
            assert grads[2 + i] is None
        else:
            assert grads[2 + i].dtype == w.dtype
            assert_within(grads[2 + i], dw, odw, f"weight grad {i}")
    again = hip_qk_rotary_backward(dq, dk, q, k, table, **kwargs)
    assert all(a is b or torch.equal(a, b) for a, b in zip(grads, again))


SHAPES = [
    # b, hq, hk, length, dim, pairs
    (1, 24, 24, 33, 128, 64), (2, 3, 1, 17, 128, 64), (3, 8, 2, 1, 64, 32), (1, 5, 5, 40, 80, 40), (1, 2, 2, 9, 256, 128),
    (1, 1, 1, 65, 16, 8), (2, 7, 3, 5, 32, 16), (1, 3, 2, 11, 512, 256), (1, 4, 4, 13, 128, 32), (1, 3, 3, 12, 96, 40),
    # not in vectors: odd pairs and dims
    (1, 3, 2, 7, 20, 10), (2, 2, 2, 6, 33, 16), (1, 2, 1, 5, 72, 29), (1, 2, 2, 4, 500, 250), (1, 2, 2, 3, 7, 0),
    (1, 1, 2, 8, 64, 0),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradient(dev, shape, interleaved, dtype):
    check(*make(sum(shape), *shape, dtype, dev), interleaved)


@pytest.mark.parametrize("interleaved", [True, False])
def test_without_norm_one_weight_and_float32_weights(dev, interleaved):
    q, k, table, qw, kw, dq, dk = make(5, 2, 6, 2, 19, 64, 24, BF16, dev)
    check(q, k, table, None, None, dq, dk, interleaved)
    check(q, k, table, None, kw, dq, dk, interleaved)
    check(q, k, table, qw.float() + 0.001, kw.float(), dq, dk, interleaved)


def test_many_tokens_and_shared_table(dev):
    check(*make(6, 2, 4, 4, 2500, 64, 32, BF16, dev, table_batch=1), True)
    q, k, table, qw, kw, dq, dk = make(7, 2, 2, 2, 30, 128, 64, BF16, dev, table_batch=1)
    check(q, k, table[0], qw, kw, dq, dk, True)


def test_layouts(dev):
    """Heads in any memory order, unaligned views, outputs in parts of a joint buffer, in place."""
    from convrot_mlx_amd import hip_qk_rotary, hip_qk_rotary_backward

    q, k, table, qw, kw, dq, dk = make(8, 2, 4, 2, 21, 64, 32, BF16, dev)
    kw_ = dict(q_weight=qw, k_weight=kw, eps=EPS)
    want = hip_qk_rotary(q, k, table, **kw_)
    for order in ((0, 1, 2, 3), (2, 0, 1, 3), (1, 2, 0, 3), (0, 1, 3, 2)):
        inverse = [order.index(i) for i in range(4)]
        q2, k2 = (t.permute(order).contiguous().permute(inverse) for t in (q, k))
        got = hip_qk_rotary(q2, k2, table, **kw_)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    check(*(torch.nn.functional.pad(t, (1, 2))[..., 1:-2] for t in (q, k)), table, qw, kw, dq, dk, True)
    # the text stream's part, then the image stream's, of one joint sequence
    joint = [torch.full((2, h, 50, 64), 7.0, dtype=BF16, device=dev) for h in (4, 2)]
    hip_qk_rotary(q, k, table, q_out=joint[0][:, :, 5:26], k_out=joint[1][:, :, 5:26], **kw_)
    for j, w in zip(joint, want):
        assert torch.equal(j[:, :, 5:26], w) and (j[:, :, :5] == 7).all() and (j[:, :, 26:] == 7).all()
    qi, ki = q.contiguous(), k.contiguous()
    hip_qk_rotary(qi, ki, table, q_out=qi, k_out=ki, **kw_)
    assert torch.equal(qi, want[0]) and torch.equal(ki, want[1])
    g = hip_qk_rotary_backward(dq, dk, q, k, table, **kw_)
    assert g[0].transpose(1, 2).is_contiguous() and g[1].transpose(1, 2).is_contiguous()


def test_empty_zero_and_non_finite(dev):
    from convrot_mlx_amd import hip_qk_rotary, hip_qk_rotary_backward

    q, k, table, qw, kw, dq, dk = make(9, 2, 3, 3, 6, 128, 64, BF16, dev)
    for cut in (q[:0], k[:0], table[:0]), (q[:, :, :0], k[:, :, :0], table[:, :0]), (q[:, :0], k, table):
        a, b = hip_qk_rotary(cut[0], cut[1], cut[2], q_weight=qw, k_weight=kw)
        assert a.shape == cut[0].shape and b.shape == cut[1].shape
        g = hip_qk_rotary_backward(torch.zeros_like(a), torch.zeros_like(b), cut[0], cut[1], cut[2], q_weight=qw,
                                   k_weight=kw)
        assert not g[2].any() and (b.numel() == 0 or g[3].isfinite().all())
    q = q.clone()
    q[0, 0, 0] = 0.0
    q[1, 2, 3, 5] = float("nan")
    out, _ = hip_qk_rotary(q, k, table, q_weight=qw, k_weight=kw)
    assert not out[0, 0, 0].any() and out[1, 2, 3].isnan().all()
    assert out[1, 2, 2].isfinite().all() and out[0].isfinite().all() and out[1, :2].isfinite().all()


def test_autograd_and_differences(dev):
    from convrot_mlx_amd import qk_rotary

    q, k, table, qw, kw, dq, dk = make(10, 2, 4, 2, 9, 32, 12, F32, dev)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, qw, kw)]
    a, b = qk_rotary(leaves[0], leaves[1], table, q_weight=leaves[2], k_weight=leaves[3], eps=EPS, interleaved=False)
    torch.autograd.backward([a, b], [dq, dk])
    t64 = table.double().cpu()
    for x, w, dy, i in ((q, qw, dq, 0), (k, kw, dk, 1)):
        dx, odx, dw, odw = rotary_grads(x.double().cpu(), w.double().cpu(), t64, dy.double().cpu(), EPS, False)
        assert_within(leaves[i].grad, dx, odx), assert_within(leaves[2 + i].grad, dw, odw)
        d = torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).double()
        f = lambda t: (dy.double().cpu() * rotary(x.double().cpu() + t * d, w.double().cpu(), t64, EPS,  # noqa: E731
                                                  False)[0]).sum()
        slope = (f(1e-4) - f(-1e-4)) / 2e-4
        assert abs((leaves[i].grad.double().cpu() * d).sum() - slope) <= 1e-5 * (dx.abs() * d.abs()).sum()
    # one output unused: its gradient is zeros
    leaf = q.detach().clone().requires_grad_()
    qk_rotary(leaf, k, table, eps=EPS)[0].sum().backward()
    assert leaf.grad.isfinite().all()


@pytest.mark.parametrize("kind", [F32, torch.float64, torch.int32, torch.int64])
def test_axes_table(dev, kind):
    """Angles in float64: cosines and sines within a float32 rounding of the exact ones, also far
    from the origin (an angle of 1e5 has a float64 error of 1.5e-11 at most)."""
    from convrot_mlx_amd import rotary_axes_table

    axes = (16, 0, 56, 56)
    pos = torch.randint(0, 100000, (2, 37, 4), generator=torch.Generator().manual_seed(1)).to(kind)
    if kind.is_floating_point:
        pos = pos * 0.25
    table = rotary_axes_table(pos.to(dev), axes, 10000.0).double().cpu()
    assert table.shape == (2, 37, 64, 2)
    at = 0
    for a, d in enumerate(axes):
        omega = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        ang = pos[..., a, None].double() * omega
        want = torch.stack([ang.cos(), ang.sin()], -1)
        assert (table[..., at: at + d // 2, :] - want).abs().max().item() <= 2.0 ** -24 if d else True
        at += d // 2
    assert rotary_axes_table(pos[:0].to(dev), axes).shape == (0, 37, 64, 2)


def test_side_stream_and_graph_replays(dev):
    from convrot_mlx_amd import hip_qk_rotary, hip_qk_rotary_backward

    q, k, table, qw, kw, dq, dk = make(12, 1, 8, 8, 200, 128, 64, BF16, dev)
    q, k = q.contiguous(), k.contiguous()
    side = torch.cuda.Stream()

    def step():
        kw_ = dict(q_weight=qw, k_weight=kw, eps=EPS)
        return (*hip_qk_rotary(q, k, table, **kw_), *hip_qk_rotary_backward(dq, dk, q, k, table, **kw_))

    eager = [t.clone() for t in step()]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            static = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    for i in range(3):
        q.mul_(0.5), k.add_(0.25)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, static))


def test_refusals(dev):
    from convrot_mlx_amd import hip_qk_rotary, hip_qk_rotary_backward, rotary_axes_table

    q, k, table, qw, kw, dq, dk = make(13, 1, 4, 2, 5, 64, 32, BF16, dev)
    with pytest.raises(ValueError, match="batch, heads, length, dim"):
        hip_qk_rotary(q[0], k, table)
    with pytest.raises(ValueError, match="must agree"):
        hip_qk_rotary(q, k[:, :, :3], table)
    with pytest.raises(ValueError, match="k dtype"):
        hip_qk_rotary(q, k.float(), table)
    with pytest.raises(ValueError, match="table must be float32"):
        hip_qk_rotary(q, k, table[:, :4])
    with pytest.raises(ValueError, match="table must be float32"):
        hip_qk_rotary(q, k, table.double())
    with pytest.raises(ValueError, match="batch entries"):
        hip_qk_rotary(q, k, table.expand(3, -1, -1, -1))
    with pytest.raises(ValueError, match="pairs do not fit"):
        hip_qk_rotary(q[..., :32], k[..., :32], table)
    with pytest.raises(ValueError, match="q_weight must have"):
        hip_qk_rotary(q, k, table, q_weight=qw[:3])
    with pytest.raises(ValueError, match="up to 512"):
        big = torch.zeros((1, 1, 5, 520), dtype=BF16, device=dev)
        hip_qk_rotary(big, big, table)
    with pytest.raises(ValueError, match="q_out must be"):
        hip_qk_rotary(q, k, table, q_out=torch.empty(4, device=dev))
    with pytest.raises(ValueError, match="expanded"):
        hip_qk_rotary(q, k, table, q_out=torch.empty((1, 1, 5, 64), dtype=BF16, device=dev).expand(1, 4, 5, 64))
    with pytest.raises(ValueError, match="must match q"):
        hip_qk_rotary_backward(dq, dk.float(), q, k, table)
    with pytest.raises(RuntimeError, match="ROCm device"):
        hip_qk_rotary(q.cpu(), k.cpu(), table.cpu())
    with pytest.raises(ValueError, match="axes_dim"):
        rotary_axes_table(torch.zeros((3, 2), device=dev), (4, 5))
    with pytest.raises(ValueError, match="must end in"):
        rotary_axes_table(torch.zeros((3, 2), device=dev), (4, 4, 4))
