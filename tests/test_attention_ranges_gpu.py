"""Attention over key ranges (pf_attention_ranges_bf16) and its gradients against the definition in 64 bits; the bounds count
roundings (tests/helpers/ranges_ref.py)."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(__file__), "helpers"))
from ranges_ref import U, attention64, attention_grad64, heads64, within  # noqa: E402

pytestmark = pytest.mark.gpu


def _ranges(kind, B, Lq, Lk, g):
    from pyflow_hip.plan import KeyRanges
    if kind is None:
        return None
    if kind == "causal":
        return KeyRanges.causal(Lq, Lk, "cuda")
    if kind == "padded":
        return KeyRanges.padded([Lk - (b * Lk) // max(1, B) for b in range(B)], Lq, "cuda")
    if kind == "documents":                       # uneven, one empty, padding rows behind the last
        n = [Lq // 5, 0, Lq // 3, 1]
        return KeyRanges.documents(n, Lq, "cuda")
    if kind == "documents causal":
        return KeyRanges.documents([Lq // 2, Lq // 7, Lq // 4], Lq, "cuda", causal=True)
    if kind == "prefix":
        return KeyRanges.prefix([Lq // 3 + b for b in range(B)], Lq, "cuda")
    # "random": two ranges per row and batch entry, overlapping, touching, outside [0, Lk), reversed, empty
    r = [torch.randint(-5, Lk + 6, (B, Lq), generator=g).int() for _ in range(4)]
    r[1][:, ::7] = r[0][:, ::7]
    r[3][:, ::7] = r[2][:, ::7] - 2
    r[1][:, 1::7] = r[2][:, 1::7]
    i = torch.iinfo(torch.int32)
    if Lq > 20:                                   # the ends of the type, alone and against each other
        r[0][:, 5], r[1][:, 5], r[0][:, 6], r[1][:, 6] = i.max, i.min, i.min, i.max
        r[2][:, 12], r[3][:, 12], r[2][:, 13], r[3][:, 13] = i.min, i.max, i.max, i.min
    return KeyRanges(*[t.cuda() for t in r])


def _case(B, Lq, Lk, H, Hkv, D, kind, radius, cap, seed=0, layout="dense", pos=False):
    g = torch.Generator().manual_seed(seed)
    scale_q = 3.0 if cap else 1.0
    n = lambda L, h: torch.randn(B, L, h, D, generator=g)  # noqa: E731
    q, k, v = (n(Lq, H) * scale_q).bfloat16(), n(Lk, Hkv).bfloat16(), n(Lk, Hkv).bfloat16()
    if layout == "dense":
        dev = [t.cuda() for t in (q, k, v)]
    elif layout == "head major":                  # [B, H, L, D] storage
        dev = [t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (q, k, v)]
    else:                                         # columns of one wide buffer, gaps between heads
        dev = []
        for t in (q, k, v):
            wide = torch.full((B, t.shape[1] + 2, t.shape[2], D + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
            w = wide[:, 1:t.shape[1] + 1, :, 8:8 + D]
            w.copy_(t)
            dev.append(w)
    ranges = _ranges(kind, B, Lq, Lk, g)
    bias = torch.randn(H, 2 * radius + 1, generator=g) * 2 if radius is not None else None
    q_pos = torch.randint(-3, Lk + 3, (B, Lq), generator=g).int() if pos else None
    if pos:
        q_pos[:, 3], q_pos[:, 4], q_pos[:, 8] = torch.iinfo(torch.int32).max, torch.iinfo(torch.int32).min, 1 << 30
    how = dict(ranges=ranges, bias=None if bias is None else bias.cuda(), q_pos=None if q_pos is None else q_pos.cuda(), cap=cap)
    ref = dict(mask=None if ranges is None else ranges.dense_mask(Lk).cpu(), bias=bias, pos=q_pos, cap=cap)
    return (q, k, v), dev, how, ref, g


def _forward(dev, how, **more):
    from pyflow_hip import ops
    q = dev[0]
    out = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device="cuda")
    lse = torch.full((q.shape[0], q.shape[2], q.shape[1]), float("nan"), device="cuda")
    ops.attention_ranges(*dev, out, lse=lse, **how, **more)
    return out, lse


def _check_forward(host, dev, how, ref, **more):
    out, lse = _forward(dev, how, **more)
    want, want_lse, bound = attention64(*host, **ref, **more)
    assert within(out, want, bound) <= 1
    # 32-bit scores (64 or 128 products and the cap's tanh), maximum, sum and logarithm
    z = (host[0].double().norm(dim=-1).max() * host[1].double().norm(dim=-1).max() * more.get("scale", host[0].shape[-1] ** -0.5)).item() if host[1].numel() else 0
    assert within(lse, want_lse, torch.full((), 2.0 ** -20 * (1 + min(z, 1e3)) + 0.0).double() + 2.0 ** -21 * want_lse.abs().clamp(max=1e6)) <= 1
    return out, lse


CASES = [  # B, Lq, Lk, H, Hkv, D, kind, radius, cap
    (1, 1, 1, 1, 1, 64, None, None, 0.0),
    (2, 1, 77, 4, 4, 64, None, None, 0.0),
    (1, 5, 33, 8, 2, 128, "causal", None, 0.0),
    (2, 64, 64, 2, 2, 64, "causal", None, 20.0),
    (1, 129, 129, 3, 1, 128, "random", None, 0.0),
    (3, 100, 193, 6, 3, 64, "padded", 7, 0.0),
    (2, 70, 70, 4, 2, 64, "prefix", 0, 0.0),
    (1, 300, 300, 2, 2, 64, "documents", None, 15.0),
    (1, 257, 257, 4, 1, 128, "documents causal", 512, 0.0),
    (2, 31, 1000, 2, 1, 64, "random", 40, 9.0),
    (1, 2, 5000, 4, 2, 128, "padded", None, 30.0),
    (2, 90, 90, 4, 2, 64, "causal", 20, 64.5),
    (1, 3, 700, 4, 2, 128, "random", None, 5000.0),
]
MANY = [  # the many-row forms (and 16 x 1 rows: split keys)
    (4, 70, 70, 64, 64, 64, "causal", None, 0.0),
    (2, 129, 257, 64, 16, 128, "random", None, 0.0),
    (16, 1, 3, 16, 8, 64, None, None, 0.0),
    (3, 200, 200, 48, 12, 64, "documents", 9, 25.0),
    (8, 128, 64, 32, 32, 128, "padded", 64, 0.0),
    (2, 385, 385, 40, 8, 64, "prefix", None, 0.0),
    (8, 130, 130, 64, 64, 64, "random", 33, 0.0),         # 128-row workgroups: this one and the next two, the last of them forward only
    (8, 140, 90, 64, 16, 64, "documents causal", None, 12.0),
    (4, 70, 200, 128, 32, 128, "random", None, 20.0),
    (4, 130, 130, 32, 8, 128, "random", 100, 300.0),
    (4, 150, 150, 32, 32, 64, "causal", 30, 0.0),
]


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D,kind,radius,cap", CASES + MANY)
def test_forward(B, Lq, Lk, H, Hkv, D, kind, radius, cap):
    host, dev, how, ref, _ = _case(B, Lq, Lk, H, Hkv, D, kind, radius, cap)
    out, lse = _check_forward(host, dev, how, ref)
    again = _forward(dev, how)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_forms():
    """which form the sizes choose, and that the listed cases reach both"""
    import ctypes as C
    from pyflow_hip import lib as L
    from pyflow_hip.lib import AttnRangesDesc, RowsView

    def which(B, Lq, Lk, H, Hkv, D, *_):
        d = AttnRangesDesc()
        d.B, d.H, d.Hkv, d.Lq, d.Lk, d.D, d.scale = B, H, Hkv, Lq, Lk, D, 1.0
        d.Q = d.O = d.K = d.V = RowsView(64, 64, 64, 64)
        return L.load().pf_attention_ranges_which(C.byref(d))
    assert {which(*c) for c in CASES} == {2} and 1 in {which(*c) for c in MANY}


@pytest.mark.parametrize("layout", ["head major", "gaps"])
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [(2, 37, 90, 4, 2, 64), (2, 140, 90, 128, 32, 128)])
def test_layouts(B, Lq, Lk, H, Hkv, D, layout):
    host, dev, how, ref, _ = _case(B, Lq, Lk, H, Hkv, D, "random", 5, 0.0, layout=layout, pos=True)
    out, _ = _check_forward(host, dev, how, ref)
    from pyflow_hip import ops
    ops.attention_ranges(*dev, dev[0], **how)                       # onto the queries
    assert torch.equal(dev[0], out)


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [(2, 3, 90, 4, 2, 64), (2, 140, 200, 128, 32, 64)])
def test_shared_keys_and_scale(B, Lq, Lk, H, Hkv, D):
    """one set of keys for the whole batch (an expanded tensor), one set of ranges, another scale"""
    host, dev, how, ref, g = _case(B, Lq, Lk, H, Hkv, D, "causal", None, 0.0)
    host = (host[0], host[1][:1].expand(B, -1, -1, -1), host[2][:1].expand(B, -1, -1, -1))
    dev = [dev[0], dev[1][:1].expand(B, -1, -1, -1), dev[2][:1].expand(B, -1, -1, -1)]
    _check_forward(host, dev, how, ref, scale=0.3)


@pytest.mark.parametrize("H,Lq", [(4, 40), (128, 140)])
def test_no_keys_no_rows(H, Lq):
    from pyflow_hip import ops
    q = torch.randn(2, Lq, H, 64, device="cuda").bfloat16()
    e = q[:, :0]
    out, lse = _forward([q, e, e], {})
    assert out.abs().max() == 0 and (lse == -math.inf).all()
    ops.attention_ranges(e, q, q, e)
    dq, dk, dv = torch.full_like(q, 7), torch.full_like(q, 7), torch.full_like(q, 7)
    none = torch.empty(2, H, 0, device="cuda")
    ops.attention_ranges_backward(q, q, e, e, out, lse, dq, e, e)
    assert dq.abs().max() == 0
    ops.attention_ranges_backward(e, e, q, q, e, none, e, dk, dv)
    assert dk.abs().max() == 0 and dv.abs().max() == 0
    bias = torch.zeros(H, 5, device="cuda")
    db = torch.full_like(bias, 7)
    ops.attention_ranges_backward(e, e, q, q, e, none, e, dk, dv, bias=bias, dbias=db)
    assert db.abs().max() == 0
    z = q[:0]
    db.fill_(7)
    ops.attention_ranges_backward(z, z, z, z, z, torch.empty(0, H, Lq, device="cuda"), z, z, z, bias=bias, dbias=db)
    assert db.abs().max() == 0


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [(1, 66, 130, 2, 1, 64), (1, 1, 130, 4, 2, 128), (2, 130, 130, 128, 64, 64), (2, 3, 2000, 4, 2, 64),
                                             (8, 130, 130, 64, 64, 64), (4, 70, 100, 128, 64, 128)])
def test_hidden_values_do_not_matter(B, Lq, Lk, H, Hkv, D):
    """infinities and NaN in keys that a row does not see change none of its bits' meaning: rows that see them get NaN, others
    their own result"""
    host, dev, how, ref, g = _case(B, Lq, Lk, H, Hkv, D, "random", None, 0.0, seed=3)
    from pyflow_hip.plan import KeyRanges
    lo = torch.randint(0, Lk - 20, (B, Lq), generator=g)
    lo[:, ::2] = (lo[:, ::2] // 64) * 64 + 10
    hi = (lo + 17).clamp(max=Lk)
    ranges = KeyRanges(lo.int().cuda(), hi.int().cuda())
    bad = [5, 9, 70, 73, Lk - 1]
    for n, j in enumerate(bad):
        for t, h in ((dev[1], host[1]), (dev[2], host[2])):
            for x in (t, h):
                x[:, j, :, n] = [float("nan"), float("inf"), float("-inf")][n % 3]
    out, lse = _forward(dev, dict(ranges=ranges))
    mask = ranges.dense_mask(Lk).cpu()
    sees_bad = mask[:, :, bad].any(-1)
    clean = [host[0], torch.nan_to_num(host[1], 0, 0, 0), torch.nan_to_num(host[2], 0, 0, 0)]
    want, want_lse, bound = attention64(*clean, mask=mask)
    ok = ~sees_bad
    assert ok.any() or Lq < 8
    assert torch.isfinite(out.cpu()[ok]).all()
    if ok.any():
        assert ((out.double().cpu() - want).abs() <= bound)[ok].all()
        assert ((lse.double().cpu() - want_lse).abs() <= 1e-4).transpose(1, 2)[ok].all()
    # gradients: finite where the row (key) has nothing to do with a bad key, garbage in rows that see nothing is ignored
    from pyflow_hip import ops
    empty = torch.zeros(B, Lq, dtype=torch.bool)
    empty[:, ::3] = True
    empty |= sees_bad                             # the rest sees clean keys only
    r2 = KeyRanges(ranges.a_lo, torch.where(empty.cuda(), ranges.a_lo, ranges.a_hi))
    out, lse = _forward(dev, dict(ranges=r2))
    do = torch.randn(host[0].shape, generator=g).bfloat16()
    q2, do2 = dev[0].clone(), do.cuda()
    q2[empty] = float("nan")
    do2[empty] = float("inf")
    dq, dk, dv = torch.empty_like(q2), torch.empty_like(dev[1]), torch.empty_like(dev[1])
    ops.attention_ranges_backward(do2, q2, dev[1], dev[2], out, lse, dq, dk, dv, ranges=r2)
    do[empty] = 0
    want = attention_grad64(do, *clean, out.cpu(), lse.cpu(), mask=r2.dense_mask(Lk).cpu())
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv)):
        assert within(got, *want[name]) <= 1, name


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D,radius,cap", [
    (1, 40, 300, 2, 2, 64, None, 0.0), (2, 130, 300, 128, 64, 64, None, 0.0), (8, 130, 300, 64, 64, 64, 5, 0.0),
    (4, 70, 200, 128, 32, 128, None, 0.0), (2, 130, 300, 64, 64, 64, None, 800.0)])
def test_scores_that_outgrow_the_first_tile(B, Lq, Lk, H, Hkv, D, radius, cap):
    """later keys whose weights exceed those of the first keys by 2^200 and more: sums and results stay finite, in every form; also
    for rows that see the first tile only, and with keys in falling order"""
    from pyflow_hip.plan import KeyRanges
    host, dev, how, ref, g = _case(B, Lq, Lk, H, Hkv, D, None, radius, cap, seed=11)
    how["cap"] = ref["cap"] = cap
    rise = torch.linspace(0, 1, Lk)[None, :, None, None] if Lq != 70 else torch.linspace(1, 0, Lk)[None, :, None, None]
    q = torch.sign(host[0].float() + 0.01) * 6
    k = (q[:, :1, ::H // Hkv].expand(B, Lk, Hkv, D) * rise * (8 * 300 / 36 / D) + host[1].float() * 0.1).bfloat16()
    q = (q[:, :1].expand(B, Lq, H, D) + host[0].float() * 0.2).bfloat16()
    hi = torch.full((B, Lq), Lk).int()
    hi[:, ::5] = 20
    ranges = KeyRanges(torch.zeros_like(hi).cuda(), hi.cuda())
    how["ranges"], ref["mask"] = ranges, ranges.dense_mask(Lk).cpu()
    host = (q, k, host[2])
    out, lse = _forward([t.cuda() for t in host], how)
    want, want_lse, bound = attention64(*host, **ref)
    assert (want_lse.max() - want_lse.min()) > 150
    # scores of several hundred carry 2^-24 of themselves into every weight
    assert within(out, want, bound + 2.0 ** -22 * want_lse.abs().max() * host[2].float().abs().max()) <= 1
    assert within(lse, want_lse, torch.full((), 2.0 ** -20).double() * want_lse.abs().max()) <= 1


def test_hidden_distances():
    """bias entries at or below -1e30 (the type's lowest value, -inf) hide their distance; a row may lose all of its keys to them"""
    B, Lq, Lk, H, D = 1, 50, 80, 3, 64
    for fewer in (False, True):
        Hn = 300 if fewer else H
        host, dev, how, ref, g = _case(B, Lq, Lk, Hn, Hn, D, "causal", 6, 0.0, seed=4)
        for t in (how["bias"], ref["bias"]):
            t[0] = -math.inf
            t[1, :8] = torch.finfo(torch.float32).min
            t[2, 3] = -1e30
        out, lse = _check_forward(host, dev, how, ref)
        assert out[:, :, 0].abs().max() == 0 and (lse[:, 0] == -math.inf).all()
        _check_backward(host, dev, how, ref, g)


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [(1, 70, 150, 2, 1, 64), (2, 130, 200, 128, 64, 64), (8, 130, 200, 64, 64, 64), (4, 70, 100, 128, 64, 128),
                                             (1, 1, 150, 2, 1, 128)])
def test_values_behind_hidden_distances_do_not_matter(B, Lq, Lk, H, Hkv, D):
    """infinities and NaN at keys that the bias alone hides, and in the gradients of rows that it hides from a key"""
    from pyflow_hip import ops
    host, dev, how, ref, g = _case(B, Lq, Lk, H, Hkv, D, None, 8, 0.0, seed=13)
    for t in (how["bias"], ref["bias"]):
        t[:, 9:] = -math.inf                      # later keys, from the first on
    last = Lk - 1                                 # seen by the last row alone
    clean = [t.clone() for t in host]
    for n, t in ((1, clean[1]), (2, clean[2])):
        dev[n][:, last] = float("nan") if n == 1 else float("inf")
        t[:, last] = 0
    out, lse = _forward(dev, how)
    want, want_lse, bound = attention64(*clean, **ref)
    if Lq > 1:
        assert within(out[:, :-1], want[:, :-1], bound[:, :-1]) <= 1
    assert torch.isnan(out[:, -1]).all()
    # the last row (the only one that may see the last key) has a gradient that is not finite: keys it does not see do not notice.  It
    # sees all keys but those of a hidden distance, so hide the near ones from it: the keys behind Lk - 6
    if Lq == 1:
        return
    for t in (how["bias"], ref["bias"]):
        t[:, 3:] = -math.inf                      # distances beyond -6 hidden
    dev2 = [t.cuda() for t in host]
    for n in (1, 2):
        dev2[n][:, last] = dev[n][:, last]        # nobody sees it now
    out, lse = _forward(dev2, how)
    do = torch.randn(host[0].shape, generator=g).bfloat16()
    dq, dk, dv, db = torch.empty_like(dev2[0]), torch.empty_like(dev2[1]), torch.empty_like(dev2[1]), torch.empty_like(how["bias"])
    ops.attention_ranges_backward(do.cuda(), *dev2, out, lse, dq, dk, dv, dbias=db, **how)
    grads = attention_grad64(do, *clean, out.cpu(), lse.cpu(), **ref)
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv), ("dbias", db)):
        assert within(got, *grads[name]) <= 1, name
    do2 = do.cuda()
    do2[:, -1] = float("inf")
    ops.attention_ranges_backward(do2, *dev2, out, lse, dq, dk, dv, **how)
    seen = Lk - 6                                 # keys that the last row sees
    for name, got, part in (("dq", dq, slice(0, Lq - 1)), ("dk", dk, slice(seen, Lk)), ("dv", dv, slice(seen, Lk))):
        assert within(got[:, part], *[x[:, part] for x in grads[name]]) <= 1, name
    assert not torch.isfinite(dv[:, :seen]).any()


def _check_backward(host, dev, how, ref, g, **more):
    from pyflow_hip import ops
    q, k, v = host
    out, lse = _forward(dev, how, **more)
    do = torch.randn(q.shape, generator=g).bfloat16()
    bias = how.get("bias")
    grads = lambda: [torch.full(t.shape, float("nan"), dtype=torch.bfloat16, device="cuda") for t in host] + \
        ([] if bias is None else [torch.full_like(bias, float("nan"))])  # noqa: E731
    a, b = grads(), grads()
    for r in (a, b):
        ops.attention_ranges_backward(do.cuda(), *dev, out, lse, *r[:3], dbias=None if bias is None else r[3], **how, **more)
    assert all(torch.equal(x, y) for x, y in zip(a, b))                 # the same bits again
    want = attention_grad64(do, q, k, v, out.cpu(), lse.cpu(), **ref, **more)
    for name, got in zip(("dq", "dk", "dv", "dbias"), a):
        assert within(got, *want[name]) <= 1, name
    return a, out, lse, do


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D,kind,radius,cap", CASES + MANY)
def test_backward(B, Lq, Lk, H, Hkv, D, kind, radius, cap):
    host, dev, how, ref, g = _case(B, Lq, Lk, H, Hkv, D, kind, radius, cap, seed=1)
    _check_backward(host, dev, how, ref, g)


@pytest.mark.parametrize("layout", ["head major", "gaps"])
def test_backward_layouts(layout):
    host, dev, how, ref, g = _case(2, 75, 140, 6, 2, 64, "random", 11, 12.0, seed=2, layout=layout, pos=True)
    _check_backward(host, dev, how, ref, g, scale=0.21)


def test_backward_against_differences():
    """central differences of the 64-bit forward along random directions, against the kernel's gradients"""
    host, dev, how, ref, g = _case(1, 40, 40, 4, 2, 64, "documents causal", 5, 11.0, seed=6)
    (dq, dk, dv, db), out, lse, do = _check_backward(host, dev, how, ref, g)
    x = [t.double() for t in host] + [ref["bias"].double()]
    way = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in x]

    def loss(h):
        y = [a + h * b for a, b in zip(x, way)]
        return (attention64(*y[:3], mask=ref["mask"], bias=y[3], cap=ref["cap"])[0] * do.double()).sum()
    want = (loss(1e-4) - loss(-1e-4)) / 2e-4
    got = sum((a.cpu().double() * b).sum() for a, b in zip((dq, dk, dv, db), way))
    # the rounding of `out` shifts delta_i by up to U sum |dO O| (1 + its own P rounding): every dT of the row moves by P times that;
    # along a direction this is at most sum_i shift_i * sum_j P_ij |direction of the score|, plus half a step per gradient entry
    exact = attention64(*host, **ref)
    shift = (do.double().abs() * exact[2]).sum(-1)                                # [B, Lq, H]
    D = 64
    kk, qq = x[1].repeat_interleave(2, 2), x[0]
    wk = way[1].repeat_interleave(2, 2)
    per_score = (way[0].norm(dim=-1).max() * kk.norm(dim=-1).max() + qq.norm(dim=-1).max() * wk.norm(dim=-1).max()) * D ** -0.5 + way[3].abs().max()
    bound = shift.sum() * per_score + 3 * U * sum((a.cpu().double() * b).abs().sum() for a, b in zip((dq, dk, dv), way)) + 1e-5 * abs(want)
    assert abs(got - want) <= bound
    # and, as the deltas' shifts have random signs, far closer than that worst case
    assert abs(got - want) <= 0.05 * abs(want) + 0.05 * bound


def test_offsets_past_32_bits():
    """keys and queries further than 2^32 bytes apart, in both forms and in the backward pass"""
    from pyflow_hip import ops
    L, H, D = 140, 2, 64
    row = (1 << 24) + 8                                             # 140 rows span 2^31 elements and more
    g = torch.Generator().manual_seed(8)
    buf = torch.zeros(row * (L + 1), dtype=torch.bfloat16, device="cuda")
    far = lambda off: buf.as_strided((1, L, H, D), (buf.numel(), row, D, 1), off)  # noqa: E731
    k, v = far(0), far(512)
    host = [torch.randn(1, L, H, D, generator=g).bfloat16() for _ in range(3)]
    k.copy_(host[1])
    v.copy_(host[2])
    dev = [host[0].cuda(), k, v]
    _check_forward(host, dev, {}, {})
    _check_backward(host, dev, {}, {}, g)
    q = far(1024)
    q.copy_(host[0])
    _check_backward(host, [q, k, v], {}, {}, g)
    many = [torch.randn(1, L, 256, D, generator=g).bfloat16().cuda(), k[:, :, :1].expand(1, L, 256, D), v[:, :, :1].expand(1, L, 256, D)]
    _check_forward([t.cpu() for t in many], many, {}, {})


def test_graphs_streams_and_workspaces():
    """forward (split keys) and backward captured with a caller's workspace each, replayed on new data with eager work between; on a
    side stream"""
    from pyflow_hip import ops
    B, Lq, Lk, H, Hkv, D = 2, 3, 3000, 8, 2, 64
    host, dev, how, ref, g = _case(B, Lq, Lk, H, Hkv, D, "padded", 20, 0.0, seed=9)
    out, lse = torch.empty_like(dev[0]), torch.empty(B, H, Lq, device="cuda")
    do = torch.randn(host[0].shape, generator=g).bfloat16().cuda()
    ws = [torch.empty(1 << 24, dtype=torch.uint8, device="cuda") for _ in range(2)]

    def step(ws_f=None, ws_b=None):
        o, s = torch.empty_like(dev[0]), torch.empty(B, H, Lq, device="cuda")
        gr = [torch.empty_like(t) for t in dev] + [torch.empty_like(how["bias"])]
        ops.attention_ranges(*dev, o, lse=s, workspace=ws_f, **how)
        ops.attention_ranges_backward(do, *dev, o, s, *gr[:3], dbias=gr[3], workspace=ws_b, **how)
        return [o, s] + gr
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(*ws)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for w in (ws, (None, None)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step(*w)))
    assert all(torch.equal(x, y) for x, y in zip(first, step()))
    for n in range(4):
        for t in dev:
            t.copy_(torch.randn(t.shape, generator=g).bfloat16())
        for graph, _ in graphs:
            graph.replay()
        eager = step()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert all(torch.equal(x, y) for x, y in zip(got, eager)), n


@pytest.mark.parametrize("D,cap", [(64, 0.0), (128, 30.0)])
def test_decoding_through_a_graph(D, cap):
    """norm + rotation of one new token per request, its key and value into the cache, attention over the cache: captured once,
    replayed token after token with the lengths and positions advanced on the device; the rest of the cache holds NaN"""
    from pyflow_hip import ops
    from pyflow_hip.plan import KeyRanges, RopeAxes
    B, S, H, Hkv = 3, 2500, 8, 2
    g = torch.Generator().manual_seed(21)
    start = torch.tensor([0, 130, 2400])
    k_cache, v_cache = (torch.full((B, S, Hkv, D), float("nan"), dtype=torch.bfloat16) for _ in range(2))
    for b, n in enumerate(start):
        k_cache[b, :n], v_cache[b, :n] = torch.randn(n, Hkv, D, generator=g).bfloat16(), torch.randn(n, Hkv, D, generator=g).bfloat16()
    k_cache, v_cache = k_cache.cuda(), v_cache.cuda()
    rope = RopeAxes.build([D], "cuda", halves=True)
    wq, wk = torch.full((D,), 1.5, device="cuda"), torch.full((D,), 0.5, device="cuda")
    zeros, lengths = torch.zeros(B, 1, dtype=torch.int32, device="cuda"), start.int()[:, None].cuda()
    pos = lengths[..., None].float()
    q, k, v = (torch.zeros(B, 1, n, D, dtype=torch.bfloat16, device="cuda") for n in (H, Hkv, Hkv))
    out, lse, ranges = torch.empty_like(q), torch.empty(B, H, 1, device="cuda"), KeyRanges(zeros, lengths)
    workspace, rows = torch.empty(1 << 24, dtype=torch.uint8, device="cuda"), torch.arange(B, device="cuda")

    def step():
        ops.qk_norm_rope_axes(q, k, q, k, wq, wk, rope, pos)
        k_cache[rows, lengths[:, 0].long()], v_cache[rows, lengths[:, 0].long()] = k[:, 0], v[:, 0]
        lengths.add_(1)
        pos.add_(1)
        ops.attention_ranges(q, k_cache, v_cache, out, ranges=ranges, cap=cap, lse=lse, workspace=workspace)
    graph = None
    for n in range(5):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g).bfloat16())
        fresh = q.clone()
        if n == 1:                                # the first token ran as it is; capturing runs nothing
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        graph.replay() if graph else step()
        torch.cuda.synchronize()
        assert (lengths[:, 0].cpu() == start + n + 1).all()
        assert not torch.equal(fresh, q) and torch.isfinite(out).all()
        seen = torch.arange(S)[None, None] < (start + n + 1)[:, None, None]
        clean = [torch.where(seen[:, 0, :, None, None], c.cpu(), torch.zeros((), dtype=torch.bfloat16)) for c in (k_cache, v_cache)]
        want, want_lse, bound = attention64(q.cpu(), *clean, mask=seen, cap=cap)
        assert within(out, want, bound) <= 1, n
        assert (lse.double().cpu() - want_lse).abs().max() <= 1e-4, n


def test_wrapper_refusals():
    from pyflow_hip import ops
    from pyflow_hip.plan import KeyRanges
    q = torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16, device="cuda")
    ok = dict(q=q, k=q, v=q, out=torch.empty_like(q))
    ops.attention_ranges(**ok)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    for bad in (dict(q=q.float()), dict(k=q[:1]), dict(v=q[:, :3]), dict(out=q[:, :, :2]), dict(q=q.cpu()), dict(scale=-1.0),
                dict(bias=torch.zeros(4, 4, device="cuda")), dict(bias=torch.zeros(3, 5, device="cuda")), dict(cap=-2.0),
                dict(bias=torch.zeros(4, 1027, device="cuda")), dict(q_pos=i32(2, 4)), dict(q_pos=i32(2, 5).long()),
                dict(ranges=KeyRanges(i32(2, 6), i32(2, 6))), dict(ranges=KeyRanges(i32(3, 5), i32(3, 5))), dict(k=q[:, :, :3], v=q[:, :, :3]),
                dict(lse=torch.zeros(2, 5, 4, device="cuda")), dict(out=q[:1].expand(2, 5, 4, 64))):
        with pytest.raises((ValueError, RuntimeError)):
            ops.attention_ranges(**{**ok, **bad})
    lse = torch.zeros(2, 4, 5, device="cuda")
    g = [torch.empty_like(q) for _ in range(3)]
    with pytest.raises(ValueError):
        ops.attention_ranges_backward(q, q, q, q, q, lse, *g, dbias=torch.zeros(4, 5, device="cuda"))
    with pytest.raises(ValueError):
        ops.attention_ranges_backward(q, q, q, q, q, lse, *g, workspace=torch.zeros(8, device="cuda"))
    with pytest.raises(ValueError):
        ops.attention_ranges_backward(q, q, q, q, q, lse.double(), *g)


def test_block_of_operators():
    """norm + rotation, attention, and both gradients as one transformer block would run them, against autograd in 64 bits"""
    from pyflow_hip import ops
    from pyflow_hip.plan import KeyRanges, RopeAxes
    B, L, H, Hkv, D = 2, 150, 6, 2, 64
    g = torch.Generator().manual_seed(12)
    x = torch.randn(B, L, (H + 2 * Hkv) * D, generator=g).bfloat16()
    wq, wk = 1 + 0.2 * torch.randn(D, generator=g), 1 + 0.2 * torch.randn(D, generator=g)
    pos = torch.rand(B, L, 3, generator=g) * 30
    do = torch.randn(B, L, H, D, generator=g).bfloat16()
    rope = RopeAxes.build([16, 24, 24], "cuda")
    ranges = KeyRanges.documents([70, 50], L, "cuda", causal=True)
    cut = lambda t: [c.unflatten(-1, (-1, D)) for c in t.split([H * D, Hkv * D, Hkv * D], dim=-1)]  # noqa: E731
    dev = x.cuda()
    q, k, v = cut(dev)
    w = wq.cuda(), wk.cuda()
    qn, kn = torch.empty(q.shape, dtype=q.dtype, device="cuda"), torch.empty(k.shape, dtype=k.dtype, device="cuda")
    out, lse = torch.empty_like(qn), torch.empty(B, H, L, device="cuda")
    ops.qk_norm_rope_axes(q, k, qn, kn, *w, rope, pos.cuda())
    ops.attention_ranges(qn, kn, v, out, ranges=ranges, cap=40.0, lse=lse)
    grad = torch.empty_like(dev)
    gq, gk, gv = cut(grad)                                           # the gradient of the projection, written in place by column
    dqn, dkn, dwq, dwk = torch.empty_like(qn), torch.empty_like(kn), torch.empty_like(w[0]), torch.empty_like(w[1])
    ops.attention_ranges_backward(do.cuda(), qn, kn, v, out, lse, dqn, dkn, gv, ranges=ranges, cap=40.0)
    ops.qk_norm_rope_axes_backward(dqn, dkn, q, k, *w, rope, pos.cuda(), gq, gk, dwq, dwk)
    x64, wq64, wk64 = x.double().requires_grad_(), wq.double().requires_grad_(), wk.double().requires_grad_()
    f, a = rope.freq.cpu(), rope.axis.cpu()
    q64, k64, v64 = cut(x64)
    o64 = attention64(heads64(q64, wq64, pos, f, a, False), heads64(k64, wk64, pos, f, a, False), v64,
                      mask=ranges.dense_mask(L).cpu(), cap=40.0)[0]
    o64.backward(do.double())
    rel = lambda u, v: ((u.double().cpu() - v).norm() / v.norm()).item()  # noqa: E731
    # bf16 values on the way: q, k, P, O forward; dO's partners P, dZ, dq, dk backward.  Six roundings of at most U each, in 2-norm
    assert rel(out, o64.detach()) <= 4 * U
    assert rel(grad, x64.grad) <= 6 * U
    assert rel(dwq, wq64.grad) <= 6 * U and rel(dwk, wk64.grad) <= 6 * U
