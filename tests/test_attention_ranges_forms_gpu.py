"""The many-row forms of pf_attention_ranges_bf16 and of its gradient, each at sizes that reach it, against the definition in 64 bits;
the bounds count roundings (tests/helpers/ranges_ref.py)."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(__file__), "helpers"))
from ranges_ref import attention64, attention_grad64, within  # noqa: E402
from test_attention_ranges_gpu import _case, _check_backward, _check_forward, _forward  # noqa: E402

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


def _rows(B, Lq, Lk, H, Hkv, D, ranges=True, gradient=False):
    """rows of one head per workgroup (+ 1: sorted), as the library chooses them"""
    import ctypes as C
    from pyflow_hip import lib as L
    from pyflow_hip.lib import AttnRangesDesc, RowsView
    d = AttnRangesDesc()
    d.B, d.H, d.Hkv, d.Lq, d.Lk, d.D, d.scale = B, H, Hkv, Lq, Lk, D, 1.0
    d.Q = d.O = d.K = d.V = d.dO = d.dQ = d.dK = d.dV = RowsView(64, 64, 64, 64)
    d.LSE = 64
    if ranges:
        d.a_lo = d.a_hi = 64
    return L.load().pf_attention_ranges_rows(C.byref(d), int(gradient))


MODES = [(None, 0.0), (None, 20.0), (6, 0.0), (6, 20.0), (None, 300.0), (6, 300.0)]         # bias radius, cap (300: tanh itself)


@pytest.mark.parametrize("radius,cap", MODES)
@pytest.mark.parametrize("form,B,Lq,Lk,H,Hkv,D", [
    (32, 2, 40, 300, 6, 2, 64), (32, 2, 40, 300, 6, 2, 128), (64, 2, 140, 90, 64, 16, 64), (64, 1, 140, 90, 64, 16, 128),
    (128, 8, 127, 90, 128, 16, 64), (128, 4, 129, 90, 64, 16, 128)])
def test_every_forward_form(form, B, Lq, Lk, H, Hkv, D, radius, cap):
    assert _rows(B, Lq, Lk, H, Hkv, D) == form
    host, dev, how, ref, _ = _case(B, Lq, Lk, H, Hkv, D, "random", radius, cap, seed=51, pos=radius is not None)
    _check_forward(host, dev, how, ref)


@pytest.mark.parametrize("form,B,Lq,Lk,H,Hkv,D", [
    (129, 9, 130, 130, 64, 64, 64), (65, 5, 257, 257, 64, 16, 64), (129, 7, 257, 257, 64, 8, 128), (65, 2, 193, 193, 96, 12, 128)])
@pytest.mark.parametrize("kind", ["documents", "documents causal", "random"])
def test_sorted_tiles(form, B, Lq, Lk, H, Hkv, D, kind):
    """row tiles that start in falling order of their keys: ties, rows that see nothing, a last tile of one row; every row is written
    (the outputs start as NaN)"""
    assert _rows(B, Lq, Lk, H, Hkv, D) == form
    host, dev, how, ref, _ = _case(B, Lq, Lk, H, Hkv, D, kind, None, 0.0, seed=52)
    out, lse = _check_forward(host, dev, how, ref)
    again = _forward(dev, how)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("Lq,Lk", [(385, 385), (640, 100)])
def test_sorted_tiles_are_each_taken_once(Lq, Lk):
    """rows that all see the same keys (every count the same) and rows of which only a few see any: values tell the rows apart"""
    from pyflow_hip import ops
    from pyflow_hip.plan import KeyRanges
    B, H, D = 6, 64, 64
    assert _rows(B, Lq, Lk, H, H, D) % 2 == 1
    g = torch.Generator().manual_seed(53)
    q, k, v = (torch.randn(B, n, H, D, generator=g).bfloat16().cuda() for n in (Lq, Lk, Lk))
    whole = torch.empty_like(q)
    ops.attention_ranges(q, k, v, whole)
    hi = torch.full((B, Lq), Lk, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, float("nan"))
    ops.attention_ranges(q, k, v, out, ranges=KeyRanges(torch.zeros_like(hi), hi))
    assert torch.equal(out, whole)
    hi[:, torch.randperm(Lq, generator=g).cuda()[:Lq * 7 // 8]] = 0
    out.fill_(float("nan"))
    ops.attention_ranges(q, k, v, out, ranges=KeyRanges(torch.zeros_like(hi), hi))
    assert torch.equal(out, torch.where(hi[..., None, None] > 0, whole, 0))


@pytest.mark.parametrize("radius,cap,with_dbias", [(r, c, True) for r, c in MODES] + [(r, c, False) for r, c in MODES if r is not None])
@pytest.mark.parametrize("form,B,Lq,Lk,H,Hkv,D", [
    (64, 2, 75, 140, 6, 2, 64), (64, 2, 75, 140, 6, 2, 128), (128, 8, 127, 90, 128, 16, 64), (128, 8, 129, 70, 128, 32, 128)])
def test_every_gradient_form(form, B, Lq, Lk, H, Hkv, D, radius, cap, with_dbias):
    from pyflow_hip import ops
    assert _rows(B, Lq, Lk, H, Hkv, D, gradient=True) == form
    host, dev, how, ref, g = _case(B, Lq, Lk, H, Hkv, D, "random", radius, cap, seed=54, pos=radius is not None)
    if with_dbias:
        _check_backward(host, dev, how, ref, g)
        return
    out, lse = _forward(dev, how)
    do = torch.randn(host[0].shape, generator=g).bfloat16()
    got = [torch.full_like(t, float("nan")) for t in dev]
    ops.attention_ranges_backward(do.cuda(), *dev, out, lse, *got, **how)
    want = attention_grad64(do, *host, out.cpu(), lse.cpu(), **ref)
    for name, x in zip(("dq", "dk", "dv"), got):
        assert within(x, *want[name]) <= 1, name


@pytest.mark.parametrize("radius,cap", [(None, 0.0), (None, 20.0), (6, 0.0)])
def test_gradient_of_many_rows_in_parts(radius, cap):
    """128 rows per workgroup at head_dim 128, and the key gradients' rows in parts"""
    B, Lq, Lk, H, Hkv, D = 1, 2000, 70, 128, 2, 128
    assert _rows(B, Lq, Lk, H, Hkv, D, gradient=True) == 128
    host, dev, how, ref, g = _case(B, Lq, Lk, H, Hkv, D, "random", radius, cap, seed=55)
    _check_backward(host, dev, how, ref, g)


@pytest.mark.parametrize("radius", [None, 6])
def test_hidden_values_in_the_large_gradient(radius):
    """infinities and NaN in keys nobody sees, and in rows that see nothing, at 128 rows per workgroup and head_dim 128"""
    from pyflow_hip import ops
    from pyflow_hip.plan import KeyRanges
    B, Lq, Lk, H, Hkv, D = 8, 129, 100, 128, 32, 128
    assert _rows(B, Lq, Lk, H, Hkv, D, gradient=True) == 128
    host, dev, how, ref, g = _case(B, Lq, Lk, H, Hkv, D, None, radius, 0.0, seed=56)
    lo = torch.randint(10, Lk - 60, (B, Lq), generator=g)
    hi = lo + torch.randint(0, 50, (B, Lq), generator=g)
    hi[:, ::5] = lo[:, ::5]
    empty = hi == lo
    how["ranges"] = KeyRanges(lo.int().cuda(), hi.int().cuda())
    ref["mask"] = how["ranges"].dense_mask(Lk).cpu()
    unseen = ~ref["mask"].any(1)                   # [B, Lk]
    assert unseen.any(1).all() and empty.any()
    do = torch.randn(host[0].shape, generator=g).bfloat16()
    clean_do = torch.where(empty[..., None, None], 0, do)
    for t in dev[1:]:
        t[unseen.cuda()] = float("nan")
    dev[0][empty.cuda()], bad_do = float("inf"), do.cuda()
    bad_do[empty.cuda()] = float("nan")
    out, lse = _forward(dev, how)
    dq, dk, dv = (torch.full_like(t, 7) for t in dev)
    ops.attention_ranges_backward(bad_do, *dev, out, lse, dq, dk, dv, **how)
    host = [torch.where(empty[..., None, None], 0, host[0]), *(torch.where(unseen[..., None, None], 0, t) for t in host[1:])]
    want = attention_grad64(clean_do, *host, out.cpu(), lse.cpu(), **ref)
    for name, x in (("dq", dq), ("dk", dk), ("dv", dv)):
        assert within(x, *want[name]) <= 1, name


def test_forms_of_the_general_cases():
    """which forms the cases of the general tests reach, so that a moved threshold shows"""
    from test_attention_ranges_gpu import CASES, MANY
    assert {_rows(*c[:6], ranges=c[6] is not None) for c in CASES} == {32}
    assert [_rows(*c[:6], ranges=c[6] is not None) for c in MANY] == [64, 64, 32, 64, 64, 64, 128, 128, 128, 64, 64]
    assert [_rows(*c[:6], gradient=True) for c in MANY] == [64] * 6 + [128, 128, 64, 64, 64]


@pytest.mark.parametrize("radius", [None, 3])
@pytest.mark.parametrize("cap", [5.0, 30.0, 64.0])
@pytest.mark.parametrize("form,B,Lq,Lk,H,Hkv,D", [
    (32, 1, 60, 1, 8, 8, 64), (32, 1, 3, 3000, 8, 2, 128), (64, 1, 64, 1, 64, 64, 64), (64, 1, 64, 40, 64, 64, 128), (128, 8, 128, 1, 128, 128, 64)])
def test_precise_log_sum_exp(form, B, Lq, Lk, H, Hkv, D, cap, radius):
    """with `precise` the log-sum-exp of capped scores is right to 32 bits of the scores; one visible key leaves nothing to average"""
    from pyflow_hip import ops
    assert _rows(B, Lq, Lk, H, Hkv, D) == form
    g = torch.Generator().manual_seed(61)
    # products and sums of these are exact in 32 bits, and so is the scale
    q = torch.randint(-3, 4, (B, Lq, H, D), generator=g).bfloat16()
    k, v = ((torch.randint(-4, 5, (B, Lk, Hkv, D), generator=g) / 4).bfloat16() for _ in range(2))
    bias = None if radius is None else torch.randn(H, 2 * radius + 1, generator=g)
    out, lse = torch.empty_like(q).cuda(), torch.empty(B, H, Lq, device="cuda")
    ops.attention_ranges(q.cuda(), k.cuda(), v.cuda(), out, scale=0.125, cap=cap, bias=None if bias is None else bias.cuda(), lse=lse, precise=True)
    want, want_lse, bound = attention64(q, k, v, scale=0.125, cap=cap, bias=bias)
    assert within(out, want, bound) <= 1
    # Half steps, relative to the capped score: 2 for scale / cap and its product, 1 for the series' end (5e-8), 4 for its sums or
    # (beyond |x| = 0.3) the exponential and quotient, 2 for cap log2 e, 1 for the sum with the bias, 2 for the way back; 4 of the bias.
    # The log-sum-exp itself 3; sums over several keys 40 more (their logarithm, at most 24 additions in a row).
    z = torch.matmul(q.double().transpose(1, 2), k.double().repeat_interleave(H // Hkv, 2).permute(0, 2, 3, 1)).mul(0.125)
    t = (cap * torch.tanh(z / cap)).abs().amax(-1)
    steps = 12 * t + 3 * want_lse.abs() + (0 if Lk == 1 else 40) + (0 if bias is None else 4 * bias.abs().max().item())
    error = (lse.double().cpu() - want_lse).abs()
    assert (error <= 2.0 ** -24 * steps).all(), (error / steps).max() * 2.0 ** 24
    loose = torch.empty_like(lse)
    ops.attention_ranges(q.cuda(), k.cuda(), v.cuda(), out, scale=0.125, cap=cap, bias=None if bias is None else bias.cuda(), lse=loose)
    # cap (1 + 2 u), u = -1 / (1 + e), in half steps of the cap (2^-24): e to 2 half steps moves 2 u by at most half of that: 1; 1 + e
    # rounded, and u to a step of its own ([1/2, 1]: 2^-24), each twice: 2 and 2 at the lower end, where e counts for nothing, 1 and 2 in
    # the middle; the product with 2 cap log2 e rounded before the cap is added again, a value of up to the cap (in the middle) or twice
    # that (lower end): 1 or 2.  Together 1 + 1 + 2 + 1 or 0 + 2 + 2 + 2
    assert ((loose.double().cpu() - want_lse).abs() <= 2.0 ** -24 * (steps + 6 * cap)).all()


@pytest.mark.parametrize("radius,cap", [(None, 0.0), (4, 0.0), (None, 5000.0)])
@pytest.mark.parametrize("form,B,Lq,H,D", [(128, 8, 65, 128, 64), (128, 8, 65, 64, 128), (64, 1, 65, 64, 64), (64, 1, 65, 64, 128), (32, 1, 65, 4, 64)])
def test_sums_near_the_end_of_the_range(form, B, Lq, H, D, radius, cap):
    """sums that end just below 2^128 (their reciprocal is subnormal), one that reaches it, and one key after another that outgrows all
    before it by 2^60"""
    from pyflow_hip import ops
    Lk = 400
    g = torch.Generator().manual_seed(91)
    for keys in ({0: -127.0, 64: 0.5, 130: -1.0}, {0: -127.0, 70: 0.5, 140: 0.5, 210: 0.5}, {0: -120.0, 80: -60.0, 160: 0.0, 240: 60.0, 399: 120.0},
                 {0: 60.0, 200: -60.0, 399: -62.0}):
        q, k = torch.zeros(B, Lq, H, D), torch.zeros(B, Lk, 1, D)
        q[..., 0], k[..., 0] = 1.0, -250.0
        for j, s in keys.items():
            k[:, j, :, 0] = s
        v = torch.rand(B, Lk, 1, D, generator=g) * 2 - 1
        q, k, v = (t.bfloat16() for t in (q, k, v))
        bias = None if radius is None else torch.zeros(H, 2 * radius + 1)
        out, lse = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device="cuda"), torch.full((B, H, Lq), float("nan"), device="cuda")
        # one set of keys for all heads, read by each through its own (expanded) key head: what decides the form is H / Hkv = 1
        kk, vv = (t.cuda().expand(B, Lk, H, D) for t in (k, v))
        ops.attention_ranges(q.cuda(), kk, vv, out, scale=math.log(2.0), cap=cap, lse=lse, bias=None if bias is None else bias.cuda())
        assert _rows(B, Lq, Lk, H, H, D, ranges=False) == form
        want, want_lse, bound = attention64(q[:1], k[:1].expand(1, Lk, H, D), v[:1].expand(1, Lk, H, D), scale=math.log(2.0), cap=cap, bias=bias)
        # as for the halves: scores of up to 250 ln 2 carry 2^-23 of themselves, three times
        assert within(out[:1], want, bound + 2.0 ** -23 * 175 * 3) <= 1
        assert within(lse[:1], want_lse, torch.full((), 2.0 ** -23 * 175 * 3).double()) <= 1
        assert torch.isfinite(out).all()
