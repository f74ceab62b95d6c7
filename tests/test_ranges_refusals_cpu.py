"""Refusals of the attention-block operators: every check is on the host, before any launch."""
import ctypes as C

import pytest
import torch


def _view(L, H, D, p=1 << 20):
    from pyflow_hip.lib import RowsView
    return RowsView(p, L * H * D, H * D, D)


def _attn(**kw):
    from pyflow_hip.lib import AttnRangesDesc
    d = AttnRangesDesc()
    d.B, d.H, d.Hkv, d.Lq, d.Lk, d.D, d.scale, d.cap = 2, 4, 2, 5, 9, 64, 0.125, 0.0
    for n in ("Q", "O", "dO", "dQ"):
        setattr(d, n, _view(5, 4, 64))
    for n in ("K", "V", "dK", "dV"):
        setattr(d, n, _view(9, 2, 64))
    d.LSE = 1 << 20
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BAD = [
    (dict(D=96), b"head_dim"), (dict(D=0), b"head_dim"), (dict(H=3), b"multiple of the key heads"), (dict(Hkv=0), b"key heads"),
    (dict(B=-1), b"negative"), (dict(Lk=-1), b"negative"), (dict(Lq=(1 << 30) + 1), b"2^30"), (dict(scale=0.0), b"scale"),
    (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"), (dict(scale=-1.0), b"scale"),
    (dict(cap=-1.0), b"cap"), (dict(cap=float("nan")), b"cap"), (dict(cap=float("inf")), b"cap"), (dict(cap=1e-38), b"cap too small"),
    (dict(a_lo=64), b"range"), (dict(b_lo=64, b_hi=64), b"range"), (dict(range_batch=-1), b"stride"),
    (dict(bias=64, bias_radius=513), b"radius"), (dict(bias=64, bias_radius=-1), b"radius"), (dict(dbias=64), b"without a bias"),
]


@pytest.mark.parametrize("change,word", BAD)
def test_attention_descriptor_refusals(change, word):
    from pyflow_hip import lib as L
    lib = L.load()
    d = _attn(**change)
    assert lib.pf_attention_ranges_bf16(C.byref(d), None) == -1 and word in lib.pf_last_error()
    assert lib.pf_attention_ranges_bwd(C.byref(d), None) == -1 and word in lib.pf_last_error()
    assert lib.pf_attention_ranges_workspace_bytes(C.byref(d)) == -1
    assert lib.pf_attention_ranges_bwd_workspace_bytes(C.byref(d)) == -1
    assert lib.pf_attention_ranges_which(C.byref(d)) == -1


def test_attention_views_and_workspace():
    from pyflow_hip import lib as L
    from pyflow_hip.lib import RowsView
    lib = L.load()
    for name in ("Q", "K", "V", "O"):
        for bad in (RowsView(0, 64, 64, 64), RowsView(8, 64, 64, 64), RowsView(64, 64, 60, 64), RowsView(64, 64, -64, 64), RowsView(64, 4, 64, 64)):
            assert lib.pf_attention_ranges_bf16(C.byref(_attn(**{name: bad})), None) == -1 and b"aligned" in lib.pf_last_error()
    for name in ("dO", "dQ", "dK", "dV"):
        assert lib.pf_attention_ranges_bwd(C.byref(_attn(**{name: RowsView(0, 0, 0, 0)})), None) == -1
    assert lib.pf_attention_ranges_bwd(C.byref(_attn(LSE=0)), None) == -1 and b"LSE" in lib.pf_last_error()
    need = lib.pf_attention_ranges_bwd_workspace_bytes(C.byref(_attn()))
    assert need >= 2 * 4 * 5 * 4
    for ws, n in ((0, 1 << 30), (64 + 8, 1 << 30), (64, need - 1)):
        assert lib.pf_attention_ranges_bwd(C.byref(_attn(workspace=ws, workspace_bytes=n)), None) == -1 and b"workspace" in lib.pf_last_error()
    long = _attn(Lk=1 << 20, Lq=1)
    need = lib.pf_attention_ranges_workspace_bytes(C.byref(long))
    assert need > 0 and lib.pf_attention_ranges_which(C.byref(long)) == 2
    assert lib.pf_attention_ranges_bf16(C.byref(long), None) == -1 and b"workspace" in lib.pf_last_error()
    assert lib.pf_attention_ranges_which(C.byref(_attn(Lq=4096, Lk=4096, H=32, Hkv=8))) == 1
    assert lib.pf_attention_ranges_bf16(None, None) == -1


def _heads(**kw):
    from pyflow_hip.lib import HeadsDesc
    d = HeadsDesc()
    d.B, d.L, d.H, d.Hkv, d.D, d.n_axes, d.n_pairs = 2, 3, 4, 2, 64, 3, 32
    for n in ("Q", "Qo", "dQ"):
        setattr(d, n, _view(3, 4, 64))
    for n in ("K", "Ko", "dK"):
        setattr(d, n, _view(3, 2, 64))
    d.pos = d.freq = d.axis = 1 << 20
    d.pos_batch, d.pos_row = 9, 3
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("change,word", [
    (dict(D=80), b"head_dim"), (dict(B=-1), b"negative"), (dict(n_pairs=33), b"rotated"), (dict(n_pairs=-1), b"rotated"),
    (dict(halves=1, n_pairs=12), b"multiple of 8"), (dict(pos=0), b"null"), (dict(freq=0), b"null"), (dict(axis=0), b"null"),
    (dict(n_axes=0), b"axis"), (dict(pos_row=-3), b"stride"), (dict(H=70000), b"heads"), (dict(B=1 << 20, L=1 << 20), b"tokens")])
def test_heads_descriptor_refusals(change, word):
    from pyflow_hip import lib as L
    lib = L.load()
    d = _heads(**change)
    assert lib.pf_qk_norm_rope_axes(C.byref(d), None) == -1 and word in lib.pf_last_error()
    assert lib.pf_qk_norm_rope_axes_bwd(C.byref(d), None, None, None, C.c_longlong(0), None) == -1 and word in lib.pf_last_error()
    assert lib.pf_qk_norm_rope_axes_bwd_workspace_bytes(C.byref(d)) == -1


def test_heads_gain_gradient_refusals():
    from pyflow_hip import lib as L
    lib = L.load()
    some = C.c_void_p(1 << 20)
    assert lib.pf_qk_norm_rope_axes_bwd(C.byref(_heads()), some, None, some, C.c_longlong(1 << 30), None) == -1 and b"without its gains" in lib.pf_last_error()
    d = _heads(wq=1 << 20)
    need = lib.pf_qk_norm_rope_axes_bwd_workspace_bytes(C.byref(d))
    assert need > 0
    assert lib.pf_qk_norm_rope_axes_bwd(C.byref(d), some, None, some, C.c_longlong(need - 1), None) == -1 and b"workspace" in lib.pf_last_error()
    assert lib.pf_qk_norm_rope_axes_bwd(C.byref(d), some, None, None, C.c_longlong(need), None) == -1 and b"workspace" in lib.pf_last_error()


def test_wrapper_views():
    from pyflow_hip import ops
    from pyflow_hip.lib import RowsView
    x = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    ops._rows(RowsView(), x, x.shape, "x", out=True)
    for bad in (x.float(), x[:, :, :3], torch.zeros(2, 3, 64, 4, dtype=torch.bfloat16).transpose(2, 3),
                torch.zeros(2, 3, 4, 65, dtype=torch.bfloat16)[..., 1:], torch.zeros(2, 3, 4, 65, dtype=torch.bfloat16)[..., :64]):
        with pytest.raises(ValueError):
            ops._rows(RowsView(), bad, x.shape, "x")
    wide = torch.zeros(1, 3, 4, 64, dtype=torch.bfloat16).expand(2, 3, 4, 64)
    ops._rows(RowsView(), wide, x.shape, "x")                          # an expanded input is read once per batch entry
    with pytest.raises(ValueError, match="expanded"):
        ops._rows(RowsView(), wide, x.shape, "x", out=True)


def test_recording_refuses():
    from pyflow_hip import ops
    ops.RECORDER = object()
    try:
        with pytest.raises(RuntimeError, match="recorded"):
            ops._one_device("attention_ranges")
    finally:
        ops.RECORDER = None


def test_plan_objects():
    import numpy as np
    from pyflow_hip.plan import KeyRanges, RopeAxes, SequencePlan, rope_cos_sin
    cpu = "cpu"
    i = torch.arange(7)
    assert torch.equal(KeyRanges.causal(5, 7, cpu).dense_mask(7)[0], torch.arange(7) <= (torch.arange(5) + 2)[:, None])
    assert torch.equal(KeyRanges.padded([3, 7], 2, cpu).dense_mask(7), (i < torch.tensor([[3], [7]]))[:, None].expand(2, 2, 7))
    d = KeyRanges.documents([2, 0, 3], 7, cpu, causal=True).dense_mask(7)[0]
    doc = torch.tensor([0, 0, 1, 1, 1, -1, -1])
    assert torch.equal(d, (doc[:, None] == doc) & (doc[:, None] >= 0) & (i[None] <= i[:, None]))
    assert torch.equal(KeyRanges.documents([2, 3], 7, cpu).dense_mask(7)[0], (doc[:, None] == doc) & (doc[:, None] >= 0))
    assert torch.equal(KeyRanges.prefix([3, 9], 7, cpu).dense_mask(7), (i < torch.tensor([3, 9])[:, None, None]) | (i[None] <= i[:, None])[None])
    m = torch.tensor([[1, 1, 0, 0, 1, 1, 1], [0, 0, 0, 0, 0, 0, 0], [0, 1, 1, 1, 1, 0, 0]])
    assert torch.equal(KeyRanges.from_key_mask(m, 3, cpu).dense_mask(7), (m != 0)[:, None].expand(3, 3, 7))
    with pytest.raises(NotImplementedError):
        KeyRanges.from_key_mask(torch.tensor([[1, 0, 1, 0, 1]]), 2, cpu)
    with pytest.raises(ValueError):
        KeyRanges.documents([4, 4], 7, cpu)
    with pytest.raises(ValueError):
        KeyRanges(torch.zeros(1, 3), torch.zeros(1, 3))
    with pytest.raises(ValueError):
        KeyRanges(torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int32))
    mask = torch.zeros(2, 16, dtype=torch.long)
    mask[0, :5] = 1
    mask[1, :12] = 1
    plan = SequencePlan([(2, 4, 8), (1, 8, 16)], mask, [16, 24, 24], cpu)
    assert np.array_equal(KeyRanges.from_plan(plan).dense_mask(plan.L).numpy(), plan.dense_mask())
    rope = RopeAxes.build([16, 24, 24], cpu)
    pos = torch.tensor([[3.0, 1.5, 7.25]])
    ang = pos.double()[:, rope.axis.long()] * rope.freq
    assert torch.equal(torch.stack([ang.cos(), ang.sin()], -1).float(), rope_cos_sin(pos, [16, 24, 24]))
    with pytest.raises(ValueError):
        RopeAxes(rope.freq.float(), rope.axis)
    with pytest.raises(ValueError):
        RopeAxes.build([3], cpu)
