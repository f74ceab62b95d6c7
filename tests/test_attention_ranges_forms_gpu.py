"""The many-row forms of pf_attention_ranges_bf16 and of its gradient, each at sizes that reach it, against the definition in 64 bits;
the bounds count roundings (tests/helpers/ranges_ref.py)."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(__file__), "helpers"))
from ranges_ref import attention64, within  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("radius,cap", [(None, 0.0), (4, 0.0), (None, 5000.0), (4, 5000.0)])
@pytest.mark.parametrize("keys", [
    {31: -126.5, 32: 0.0, 64: 1.0},                 # one half's reference lies 126.5 below the other's, its last key above both
    {63: -126.5, 0: 0.0, 96: 1.0},                  # the halves the other way round
    {31: -127.0, 63: -127.0, 64: 0.5, 96: 0.5},     # both sums finite (2^127.5), their sum not
    {31: -127.0, 63: -100.0, 64: 0.5, 96: -0.5},
    {0: 20.0, 32: -100.0, 96: 27.0},                # the larger reference is not the larger half
    {0: 0.0, 64: 100.0},                            # the other half sees nothing that counts
])
def test_halves_with_far_references(keys, radius, cap, D):
    """64-row workgroups whose key halves met different first keys: scores (base 2) as given, all other keys at -250"""
    from pyflow_hip import ops
    Lq, Lk, H = 64, 128, 64
    g = torch.Generator().manual_seed(31)
    q, k = torch.zeros(1, Lq, H, D), torch.zeros(1, Lk, H, D)
    q[..., 0], k[..., 0] = 1.0, -250.0
    for j, s in keys.items():
        k[:, j, :, 0] = s
    v = torch.rand(1, Lk, H, D, generator=g) * 2 - 1
    q, k, v = (t.bfloat16() for t in (q, k, v))
    bias = None if radius is None else torch.zeros(H, 2 * radius + 1)
    out, lse = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device="cuda"), torch.full((1, H, Lq), float("nan"), device="cuda")
    ops.attention_ranges(q.cuda(), k.cuda(), v.cuda(), out, scale=math.log(2.0), cap=cap, lse=lse, bias=None if bias is None else bias.cuda())
    want, want_lse, bound = attention64(q, k, v, scale=math.log(2.0), cap=cap, bias=bias)
    # scores of up to 250 ln 2 carry 2^-23 of themselves into the weights (product, scale, cap: half a step each)
    assert within(out, want, bound + 2.0 ** -23 * 175 * 3) <= 1
    assert within(lse, want_lse, torch.full((), 2.0 ** -23 * 175 * 3).double()) <= 1


@pytest.mark.parametrize("cap,radius", [(0.0, None), (20.0, 6)])
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [
    (3, 1, 777, 8, 2, 64), (2, 1, 5000, 8, 2, 128), (2, 5, 300, 6, 3, 128),        # split keys
    (1, 90, 300, 64, 16, 64), (2, 90, 300, 64, 64, 128),                            # 64 rows
    (8, 150, 300, 64, 8, 64), (4, 150, 300, 64, 8, 128)])                           # 128 rows
def test_slots_that_nobody_sees_cost_nothing(B, Lq, Lk, H, Hkv, D, cap, radius):
    """a cache from torch.empty may hold anything in front of, between and behind the keys that are seen: the same bits as over zeros
    (a result that is computed again from its visible keys alone rounds its weights elsewhere), forward and gradient of the rows"""
    from pyflow_hip import ops
    from pyflow_hip.plan import KeyRanges
    g = torch.Generator().manual_seed(37)
    q, do = (torch.randn(B, Lq, H, D, generator=g).bfloat16().cuda() for _ in range(2))
    k, v = (torch.randn(B, Lk, Hkv, D, generator=g).bfloat16().cuda() for _ in range(2))
    bias = None if radius is None else torch.randn(H, 2 * radius + 1, generator=g).cuda()
    lo, mid, mid2, hi = 9, Lk // 3, Lk // 3 + 30, Lk - 43
    for two in (False, True):
        rows = torch.arange(Lq)[None].expand(B, Lq)
        a_lo, end = torch.full((B, Lq), lo), (hi - Lq + 1 + rows).clamp(min=mid2)         # the last row sees up to `hi`
        args = [a_lo, torch.full_like(a_lo, mid), torch.full_like(a_lo, mid2), end] if two else [a_lo, end]
        ranges = KeyRanges(*[t.int().contiguous().cuda() for t in args])
        how = dict(ranges=ranges, cap=cap, bias=bias)
        unseen = torch.ones(Lk, dtype=torch.bool)
        unseen[lo:hi] = False
        if two:
            unseen[mid:mid2] = True
        got = []
        for bad in (0.0, float("nan"), float("inf")):
            kk, vv = k.clone(), v.clone()
            kk[:, unseen.cuda()], vv[:, unseen.cuda()] = bad, bad
            out, lse = torch.empty_like(q), torch.empty(B, H, Lq, device="cuda")
            ops.attention_ranges(q, kk, vv, out, lse=lse, **how)
            dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
            ops.attention_ranges_backward(do, q, kk, vv, out, lse, dq, dk, dv, **how)
            got.append((out, lse, dq))
            assert not dk[:, unseen.cuda()].any() and not dv[:, unseen.cuda()].any()
        assert torch.isfinite(got[0][0]).all() and torch.isfinite(got[0][2]).all()
        for other in got[1:]:
            for name, x, y in zip(("out", "lse", "dq"), got[0], other):
                assert torch.equal(x, y), (two, name)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B", [1, 8])
def test_slots_that_nobody_sees_in_the_second_pass(B, D):
    """the same where the first pass overflowed and the workgroup ran again with the running maximum"""
    from pyflow_hip import ops
    from pyflow_hip.plan import KeyRanges
    Lq, Lk, H = 70, 400, 64 * (2 if D == 128 else 1) * (1 if B == 1 else 2)
    g = torch.Generator().manual_seed(38)
    q, v = torch.zeros(B, Lq, H, D), torch.randn(B, Lk, 1, D, generator=g)
    q[..., 0] = 1.0
    k = torch.randn(B, Lk, 1, D, generator=g)
    k[..., 0] = torch.linspace(0, 600, Lk)[None, :, None]
    q, k, v = (t.bfloat16().cuda() for t in (q, k, v))
    lo = torch.full((B, Lq), 13, dtype=torch.int32, device="cuda")
    ranges = KeyRanges(lo, torch.full_like(lo, 350))
    got = []
    for bad in (0.0, float("nan")):
        for t in (k, v):
            t[:, :13], t[:, 350:] = bad, bad
        out, lse = torch.empty_like(q), torch.empty(B, H, Lq, device="cuda")
        ops.attention_ranges(q, k.expand(B, Lk, H, D) if B > 1 else k, v.expand(B, Lk, H, D) if B > 1 else v, out, ranges=ranges, scale=1.0, lse=lse)
        got.append((out, lse))
    clean = torch.where(torch.isnan(k), 0, k).cpu(), torch.where(torch.isnan(v), 0, v).cpu()
    want, want_lse, bound = attention64(q.cpu(), *clean, mask=ranges.dense_mask(Lk).cpu(), scale=1.0)
    # scores up to 600 carry 2^-23 of themselves into the weights, three roundings
    assert within(got[0][0], want, bound + 3 * 2.0 ** -23 * 600 * 4) <= 1
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize("radius", [None, 5])
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [
    (1, 320, 140, 8, 2, 64), (1, 300, 140, 8, 2, 128), (2, 301, 77, 4, 4, 64),     # the rows in parts
    (2, 64, 300, 16, 16, 64), (2, 70, 300, 16, 16, 64), (1, 90, 300, 24, 24, 128)])   # all rows in one workgroup
def test_one_infinite_gradient_entry(B, Lq, Lk, H, Hkv, D, radius):
    """nothing is hidden and one entry of dout is infinite: the gradients of its channel say so, those of v's other channels keep their
    bits (keys that are computed again, one by one, would round their weights elsewhere), also where the last row tile is short"""
    from pyflow_hip import ops
    g = torch.Generator().manual_seed(41)
    q, do = (torch.randn(B, Lq, H, D, generator=g).bfloat16().cuda() for _ in range(2))
    k, v = (torch.randn(B, Lk, Hkv, D, generator=g).bfloat16().cuda() for _ in range(2))
    bias = None if radius is None else torch.randn(H, 2 * radius + 1, generator=g).cuda()
    out, lse = torch.empty_like(q), torch.empty(B, H, Lq, device="cuda")
    ops.attention_ranges(q, k, v, out, lse=lse, bias=bias)

    def gradients(do):
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        ops.attention_ranges_backward(do, q, k, v, out, lse, dq, dk, dv, bias=bias)
        return dq, dk, dv
    clean = gradients(do)
    for row in (3, Lq - 1):
        bad = do.clone()
        bad[0, row, 0, 7] = math.inf
        dq, dk, dv = gradients(bad)
        assert (dv[0, :, 0, 7] == math.inf).all() and not torch.isfinite(dk[0, :, 0]).any() and not torch.isfinite(dq[0, row, 0]).any()
        others = torch.ones_like(dv, dtype=torch.bool)
        others[0, :, 0, 7] = False
        if row == 3 or Lq % 64 == 0:              # a short tile repeats the last row, whose infinity then has to be kept away
            assert torch.equal(dv[others], clean[2][others])
        assert torch.equal(dv[:, :, 1:], clean[2][:, :, 1:]) and torch.equal(dk[:, :, 1:], clean[1][:, :, 1:])
        others = torch.ones_like(dq, dtype=torch.bool)
        others[0, row, 0] = False
        assert torch.equal(dq[others], clean[0][others])


def test_outputs_beside_their_inputs_and_over_them():
    """columns of one buffer, head-major halves and the queries themselves take results; anything that overlaps otherwise is refused"""
    from pyflow_hip import ops
    from pyflow_hip.plan import RopeAxes
    B, L, H, D = 2, 90, 4, 64
    g = torch.Generator().manual_seed(43)
    apart = [torch.randn(B, L, H, D, generator=g).bfloat16().cuda() for _ in range(3)]
    want = torch.empty_like(apart[0])
    ops.attention_ranges(*apart, want)
    wide = torch.empty(B, L, 4 * H + 1, D, dtype=torch.bfloat16, device="cuda")
    major = torch.empty(B, 4, H, L, D, dtype=torch.bfloat16, device="cuda")
    mixed = torch.empty(B, L, H, 4, D, dtype=torch.bfloat16, device="cuda")
    for places in ([wide[:, :, n * H:(n + 1) * H] for n in range(4)], [major[:, n].transpose(1, 2) for n in range(4)], [mixed[:, :, :, n] for n in range(4)]):
        for x, t in zip(places, apart):
            x.copy_(t)
        ops.attention_ranges(*places)
        assert torch.equal(places[3], want) and all(torch.equal(x, t) for x, t in zip(places, apart))
        ops.attention_ranges(*places[:3], places[0])
        assert torch.equal(places[0], want)
    shifted = wide[:, :, 1:H + 1]
    for out in (shifted, wide[:, :, H:2 * H], wide[:, :, 2 * H + 1:3 * H + 1]):
        with pytest.raises(RuntimeError, match="overlaps"):
            ops.attention_ranges(wide[:, :, :H], wide[:, :, H:2 * H], wide[:, :, 2 * H:3 * H], out)
    lse = torch.zeros(B, H, L, device="cuda")
    ops.attention_ranges(*apart, want, lse=lse)
    grads = [torch.empty_like(t) for t in apart]
    for n in range(3):
        for taken in (apart[0], apart[2], want, grads[(n + 1) % 3]):
            outs = list(grads)
            outs[n] = taken
            with pytest.raises(RuntimeError, match="overlap"):
                ops.attention_ranges_backward(apart[1], *apart, want, lse, *outs)
    rope = RopeAxes.build([D], "cuda")
    pos = torch.zeros(1, L, 1, device="cuda")
    q, k = wide[:, :, :H], wide[:, :, H:2 * H]
    ops.qk_norm_rope_axes(q, k, q, k, None, None, rope, pos)
    ops.qk_norm_rope_axes(q, k, wide[:, :, 2 * H:3 * H], wide[:, :, 3 * H:4 * H], None, None, rope, pos)
    for qo, ko in ((k, q), (shifted, k), (q, wide[:, :, H + 1:2 * H + 1])):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.qk_norm_rope_axes(q, k, qo, ko, None, None, rope, pos)
