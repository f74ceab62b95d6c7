"""Per-head RMSNorm + multi-axis rotation (pf_qk_norm_rope_axes) and its gradient against the definition in 64 bits."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(__file__), "helpers"))
from ranges_ref import U, heads64, within  # noqa: E402

pytestmark = pytest.mark.gpu


def _case(B, L, H, Hkv, D, axes, halves, norm, fused, seed=0, far=0.0):
    from pyflow_hip.plan import RopeAxes
    g = torch.Generator().manual_seed(seed)
    if fused:
        big = (torch.randn(B, L, (H + 2 * Hkv) * D, generator=g) * 2).bfloat16()
        dev = big.cuda()
        cut = lambda t: (t[..., :H * D].unflatten(-1, (H, D)), t[..., H * D:(H + Hkv) * D].unflatten(-1, (Hkv, D)))  # noqa: E731
        (q, k), (qd, kd) = cut(big), cut(dev)
    else:
        q, k = (torch.randn(B, L, n, D, generator=g).mul(2).bfloat16() for n in (H, Hkv))
        qd, kd = q.cuda(), k.cuda()
    pos = torch.rand(B, L, len(axes), generator=g) * 50 - 10
    pos[..., 0] = torch.arange(L) + far
    w = [1 + 0.3 * torch.randn(D, generator=g) for _ in range(2)] if norm else [None, None]
    rope = RopeAxes.build(axes, "cuda", halves=halves)
    return q, k, qd, kd, pos, w, rope, g


CASES = [  # B, L, H, Hkv, D, axes, halves, norm, fused
    (1, 1, 1, 1, 64, [16, 24, 24], False, True, False),
    (2, 77, 3, 3, 64, [16, 24, 24], False, True, True),
    (2, 130, 5, 1, 64, [64], True, True, False),
    (1, 19, 8, 2, 128, [32, 48, 48], False, True, True),
    (3, 33, 12, 4, 128, [32, 32], True, True, False),          # half of the channels only
    (1, 40, 7, 7, 64, [2, 4], False, False, False),            # three pairs: a lane with one rotated and three plain pairs
    (2, 9, 33, 3, 128, [128], True, False, True),
    (1, 2100, 9, 9, 64, [32, 16, 16], True, True, True),       # one wave per token
]


@pytest.mark.parametrize("B,L,H,Hkv,D,axes,halves,norm,fused", CASES)
def test_forward(B, L, H, Hkv, D, axes, halves, norm, fused):
    from pyflow_hip import ops
    q, k, qd, kd, pos, w, rope, _ = _case(B, L, H, Hkv, D, axes, halves, norm, fused, far=1e5)
    qo, ko = torch.empty(B, L, H, D, dtype=torch.bfloat16, device="cuda"), torch.empty(B, L, Hkv, D, dtype=torch.bfloat16, device="cuda")
    dw = [None if x is None else x.cuda() for x in w]
    ops.qk_norm_rope_axes(qd, kd, qo, ko, dw[0], dw[1], rope, pos.cuda(), q_scale=0.18)
    f, a = rope.freq.cpu(), rope.axis.cpu()
    for got, x, wi, s in ((qo, q, w[0], 0.18), (ko, k, w[1], 1.0)):
        want = heads64(x, wi, pos, f, a, halves, scale=s)
        # one rounding; cos / sin, the norm and the products in 32 bits: 2^-18 of the pair's size, at most the row's largest
        bound = U * want.abs() + 2.0 ** -18 * want.abs().amax(-1, keepdim=True) + 1e-30
        assert within(got, want, bound) <= 1
    # in place, through the same views
    ops.qk_norm_rope_axes(qd, kd, qd, kd, dw[0], dw[1], rope, pos.cuda(), q_scale=0.18)
    assert torch.equal(qd, qo) and torch.equal(kd, ko)


@pytest.mark.parametrize("B,L,H,Hkv,D,axes,halves,norm,fused", CASES)
def test_backward(B, L, H, Hkv, D, axes, halves, norm, fused):
    from pyflow_hip import ops
    q, k, qd, kd, pos, w, rope, g = _case(B, L, H, Hkv, D, axes, halves, norm, fused, seed=1, far=3e4)
    dy = [torch.randn(B, L, n, D, generator=g).bfloat16() for n in (H, Hkv)]
    dx = [torch.empty(B, L, n, D, dtype=torch.bfloat16, device="cuda") for n in (H, Hkv)]
    gw = [torch.full((D,), 7.0, device="cuda") if norm else None for _ in range(2)]
    dw = [None if x is None else x.cuda() for x in w]
    args = (rope, pos.cuda())
    ops.qk_norm_rope_axes_backward(dy[0].cuda(), dy[1].cuda(), qd, kd, *dw, *args, *dx, *gw, q_scale=0.18)
    f, a = rope.freq.cpu(), rope.axis.cpu()
    for n, (x, wi, s) in enumerate(((q, w[0], 0.18), (k, w[1], 1.0))):
        x64 = x.double().requires_grad_()
        w64 = None if wi is None else wi.double().requires_grad_()
        y = heads64(x64, w64, pos, f, a, halves, scale=s)
        y.backward(dy[n].double())
        bound = U * x64.grad.abs() + 2.0 ** -17 * x64.grad.abs().amax(-1, keepdim=True) + 1e-30
        assert within(dx[n], x64.grad, bound) <= 1
        if wi is not None:
            # 32-bit sums of |g x r|: partial sums of at most a few hundred terms each, 2^-24 apiece
            mag = (dy[n].double().abs().amax(-1, keepdim=True) * 1.5 * s * (x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-6)).abs())
            assert within(gw[n], w64.grad, 2.0 ** -16 * mag.sum((0, 1, 2)) + 1e-30) <= 1
    # the same bits again, from a caller's workspace, onto the gradients themselves
    again = [t.cuda() for t in dy]
    gw2 = [None if t is None else torch.empty_like(t) for t in gw]
    ws = torch.empty(1 << 20, dtype=torch.float32, device="cuda")
    ops.qk_norm_rope_axes_backward(again[0], again[1], qd, kd, *dw, *args, *again, *gw2, q_scale=0.18, workspace=ws)
    for u, v in zip(again + [t for t in gw2 if t is not None], dx + [t for t in gw if t is not None]):
        assert torch.equal(u, v)


def test_backward_against_differences():
    """directional derivative of the 64-bit forward by central differences, against the kernel's gradients"""
    from pyflow_hip import ops
    q, k, qd, kd, pos, w, rope, g = _case(1, 6, 2, 1, 64, [16, 24, 24], False, True, False, seed=5)
    f, a = rope.freq.cpu(), rope.axis.cpu()
    dy, dyk = torch.randn(1, 6, 2, 64, generator=g).bfloat16(), torch.randn(1, 6, 1, 64, generator=g).bfloat16()
    dq, dk, gq, gk = torch.empty_like(qd), torch.empty_like(kd), torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
    ops.qk_norm_rope_axes_backward(dy.cuda(), dyk.cuda(), qd, kd, w[0].cuda(), w[1].cuda(), rope, pos.cuda(), dq, dk, gq, gk)
    vx, vw = torch.randn(q.shape, generator=g, dtype=torch.float64), torch.randn(64, generator=g, dtype=torch.float64)
    loss = lambda h: (heads64(q.double() + h * vx, w[0].double() + h * vw, pos, f, a, False) * dy.double()).sum()  # noqa: E731
    want = (loss(1e-4) - loss(-1e-4)) / 2e-4
    got = (dq.cpu().double() * vx).sum() + (gq.cpu().double() * vw).sum()
    # each of the 768 gradient entries is off by half a step at most
    assert abs(got - want) <= U * (dq.cpu().double() * vx).abs().sum() + 1e-5 * abs(want)


def test_far_positions_and_plain_channels():
    """positions of 2^24 - 1 keep their angle; channels behind the pairs pass through untouched, infinities among them"""
    from pyflow_hip import ops
    from pyflow_hip.plan import RopeAxes
    for halves in (False, True):
        rope = RopeAxes.build([32], "cuda", halves=halves)
        x = torch.randn(1, 3, 2, 64, generator=torch.Generator().manual_seed(2)).bfloat16()
        x[..., 40] = float("inf")
        x[..., 63] = float("-inf")
        pos = torch.tensor([0.0, 2.0 ** 24 - 1, -12345.5]).view(1, 3, 1)
        y = torch.empty_like(x, device="cuda")
        ops.qk_norm_rope_axes(x.cuda(), None, y, None, None, None, rope, pos.cuda())
        assert torch.equal(y[..., 32:].cpu(), x[..., 32:])
        want = heads64(x[..., :32], None, pos, rope.freq.cpu(), rope.axis.cpu(), halves)
        assert within(y[..., :32], want, U * want.abs() + 2.0 ** -18 * want.abs().amax(-1, keepdim=True)) <= 1
        assert torch.equal(y[0, 0].cpu(), x[0, 0])                       # position 0 turns nothing


def test_shared_positions_one_side_and_no_tokens():
    from pyflow_hip import ops
    q, k, qd, kd, pos, w, rope, g = _case(3, 11, 2, 2, 64, [16, 24, 24], False, True, False, seed=3)
    one = pos[:1].cuda()
    qo, ko = torch.empty_like(qd), torch.empty_like(kd)
    wq, wk = w[0].cuda(), w[1].cuda()
    ops.qk_norm_rope_axes(qd, kd, qo, ko, wq, wk, rope, one)
    ko2 = torch.empty_like(kd)
    ops.qk_norm_rope_axes(None, kd, None, ko2, None, wk, rope, one.expand(3, 11, 3))
    assert torch.equal(ko, ko2)
    # gains for the keys only
    qo3, ko3 = torch.empty_like(qd), torch.empty_like(kd)
    ops.qk_norm_rope_axes(qd, kd, qo3, ko3, None, wk, rope, one)
    want = heads64(q, None, pos[:1], rope.freq.cpu(), rope.axis.cpu(), False)
    assert torch.equal(ko, ko3)
    assert within(qo3, want, U * want.abs() + 2.0 ** -18 * want.abs().amax(-1, keepdim=True) + 1e-30) <= 1
    # no tokens: nothing to write but the gains' gradients, which are zero
    e = qd[:, :0]
    gw = torch.full((64,), 3.0, device="cuda")
    ops.qk_norm_rope_axes(e, None, e, None, wq, None, rope, one[:, :0])
    ops.qk_norm_rope_axes_backward(e, None, e, None, wq, None, rope, one[:, :0], e, None, gw, None)
    assert gw.abs().max() == 0


def test_graph_replays_and_streams():
    """captured forward and backward replay on new data with eager work between; the launch follows torch's current stream"""
    from pyflow_hip import ops
    q, k, qd, kd, pos, w, rope, g = _case(2, 50, 4, 2, 64, [16, 24, 24], False, True, False, seed=4)
    p, wq, wk = pos.cuda(), w[0].cuda(), w[1].cuda()
    bufs = [torch.empty_like(qd), torch.empty_like(kd), torch.empty_like(qd), torch.empty_like(kd), torch.empty(64, device="cuda"), torch.empty(64, device="cuda")]

    def step(o):
        ops.qk_norm_rope_axes(qd, kd, o[0], o[1], wq, wk, rope, p)
        ops.qk_norm_rope_axes_backward(o[0], o[1], qd, kd, wq, wk, rope, p, *o[2:])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(bufs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(bufs)
    for n in range(4):
        qd.copy_(torch.randn(q.shape, generator=g).bfloat16())
        graph.replay()
        eager = [torch.empty_like(t) for t in bufs]
        step(eager)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(bufs, eager)), n
