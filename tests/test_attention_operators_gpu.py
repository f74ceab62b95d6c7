"""Calls of the attention-block operators at the ends of what their documentation allows."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(__file__), "helpers"))
from ranges_ref import U, heads64  # noqa: E402

pytestmark = pytest.mark.gpu


def test_positions_with_too_few_axes_are_refused():
    """a rotation by (t, h, w) at positions of one axis has no answer; more axes than it uses are fine"""
    from pyflow_hip import ops
    from pyflow_hip.plan import RopeAxes
    g = torch.Generator().manual_seed(71)
    q, pos = torch.randn(1, 9, 2, 64, generator=g).bfloat16(), torch.rand(1, 9, 4, generator=g) * 30
    rope, dev, out = RopeAxes.build([16, 24, 24], "cuda"), q.cuda(), torch.empty(1, 9, 2, 64, dtype=torch.bfloat16, device="cuda")
    for n in (1, 2):
        p = pos[..., :n].contiguous().cuda()
        with pytest.raises(ValueError, match="axes"):
            ops.qk_norm_rope_axes(dev, None, out, None, None, None, rope, p)
        with pytest.raises(ValueError, match="axes"):
            ops.qk_norm_rope_axes_backward(dev, None, dev, None, None, None, rope, p, out, None)
    for n in (3, 4):
        ops.qk_norm_rope_axes(dev, None, out, None, None, None, rope, pos[..., :n].contiguous().cuda())
        want = heads64(q, None, pos, rope.freq.cpu(), rope.axis.cpu(), False)
        # one rounding to bf16; 2^-20 of the pair for the 32-bit sine, cosine and sum
        pair = (want[..., 0::2].square() + want[..., 1::2].square()).sqrt().repeat_interleave(2, -1)
        assert ((out.double().cpu() - want).abs() <= U * want.abs() + 2.0 ** -20 * pair + 1e-30).all()


def test_more_tokens_than_one_launch_has_threads_for():
    """2^26 + 5 tokens of one head: a wave each would be more than 2^32 threads; first, last and some of the rows between, in place"""
    from pyflow_hip import ops
    from pyflow_hip.plan import RopeAxes
    L, D = (1 << 26) + 5, 64
    g = torch.Generator(device="cuda").manual_seed(72)
    q = torch.empty(1, L, 1, D, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    pos = torch.empty(1, L, 1, device="cuda").uniform_(0, 1e4, generator=g)
    rows = torch.cat([torch.arange(9), torch.randint(0, L, (200,), generator=torch.Generator().manual_seed(73)), torch.arange(L - 9, L),
                      torch.arange((1 << 26) - 1030, (1 << 26) + 5)]).cuda()
    before, w = q[:, rows].cpu(), torch.full((D,), 1.25)
    rope = RopeAxes.build([D], "cuda")
    ops.qk_norm_rope_axes(q, None, q, None, w.cuda(), None, rope, pos)
    want = heads64(before, w, pos[:, rows].cpu(), rope.freq.cpu(), rope.axis.cpu(), False)
    # one rounding; cos / sin, the norm and the products in 32 bits: 2^-18 of the row's largest
    assert ((q[:, rows].double().cpu() - want).abs() <= U * want.abs() + 2.0 ** -18 * want.abs().amax(-1, keepdim=True)).all()


def test_profiler_sees_the_operators():
    """each call is one record under its operator's name: bytes of the norm and rotation, operations of the pairs that are seen"""
    from pyflow_hip import ops
    from pyflow_hip.plan import KeyRanges, RopeAxes
    B, L, H, Hkv, D = 2, 70, 4, 2, 64
    q, out, dq = (torch.zeros(B, L, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    k, v, dk, dv = (torch.zeros(B, L, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in range(4))
    lse, w = torch.zeros(B, H, L, device="cuda"), torch.ones(D, device="cuda")
    rope, pos, ranges = RopeAxes.build([D], "cuda"), torch.zeros(1, L, 1, device="cuda"), KeyRanges.causal(L, L, "cuda")
    kept, ops.PROFILER.records, ops.PROFILER.enabled = ops.PROFILER.records, {}, True
    try:
        ops.qk_norm_rope_axes(q, k, q, k, w, w, rope, pos)
        ops.attention_ranges(q, k, v, out, lse=lse)
        ops.attention_ranges(q, k, v, out, ranges=ranges, lse=lse)
        ops.attention_ranges_backward(out, q, k, v, out, lse, dq, dk, dv, ranges=ranges)
        ops.qk_norm_rope_axes_backward(dq, dk, q, k, w, None, rope, pos, dq, dk)
        torch.cuda.synchronize()
        seen = {n: (s["launches"], s["work_total"]) for n, s in ops.PROFILER.summary().items()}
    finally:
        ops.PROFILER.records, ops.PROFILER.enabled = kept, False
    causal = B * L * (L + 1) // 2
    assert seen == {"qk_norm_rope_axes": (1, 4.0 * B * L * (H + Hkv) * D), "attention_ranges": (2, 4.0 * D * H * (B * L * L + causal)),
                    "attention_ranges_bwd": (1, 10.0 * D * H * causal), "qk_norm_rope_axes_bwd": (1, 2.0 * B * L * D * (3 * H + 2 * Hkv))}
