"""Views that share memory: the host's test against a count of every element, and what the attention-block operators refuse.  Every
refusal is on the host, before any launch."""
import ctypes as C
import random

import pytest


def _elements(p, strides, sizes, D):
    out = set()
    for b in range(sizes[0]):
        for r in range(sizes[1]):
            for h in range(sizes[2]):
                at = p + b * strides[0] + r * strides[1] + h * strides[2]
                out.update(range(at, at + D))
    return out


def _share(a, b, D):
    from pyflow_hip import lib as L
    from pyflow_hip.lib import RowsView
    (pa, sa, na), (pb, sb, nb) = a, b
    x, y = RowsView(2 * pa, *sa), RowsView(2 * pb, *sb)
    return bool(L.load().pf_rows_views_share(C.byref(x), *na, C.byref(y), *nb, D))


def _nested(rng, sizes, D, orders):
    """strides of a layout of the sizes in some order, with gaps"""
    strides, step = [0, 0, 0], D
    for i in rng.choice(orders):
        strides[i] = step + 8 * rng.choice([0, 0, 1, 5, 16])
        step = strides[i] * sizes[i]
    return strides


@pytest.mark.parametrize("seed", range(40))
def test_sharing_against_every_element(seed):
    rng = random.Random(seed)
    orders = [(2, 1, 0), (1, 2, 0), (2, 0, 1), (0, 1, 2)]
    for _ in range(25):
        D = 64
        na, nb = ([rng.choice([0, 1, 1, 2, 3, 4]) if rng.random() < 0.1 else rng.randint(1, 4) for _ in range(3)] for _ in range(2))
        sa = _nested(rng, [max(1, n) for n in na], D, orders)
        sb = list(sa) if rng.random() < 0.6 else _nested(rng, [max(1, n) for n in nb], D, orders)
        if rng.random() < 0.3:                     # an expanded input
            sb[rng.randrange(3)] = 0
        pa = 4096
        pb = pa + 8 * rng.randint(-80, 80)
        a, b = (pa, sa, na), (pb, sb, nb)
        assert _share(a, b, D) == bool(_elements(*a, D) & _elements(*b, D)), (a, b)
        assert _share(b, a, D) == _share(a, b, D)


def test_columns_of_one_buffer():
    B, L, D = 2, 700, 64
    row = (30 + 2 * 10) * D
    q, k, v = (0, [L * row, row, D], [B, L, 30]), (30 * D, [L * row, row, D], [B, L, 10]), (40 * D, [L * row, row, D], [B, L, 10])
    assert not _share(q, k, D) and not _share(k, v, D) and not _share(q, v, D)
    assert _share(q, (30 * D - 8, *k[1:]), D) and _share(k, (30 * D + 8, *k[1:]), D)
    head_major = lambda n: (n * 5 * L * D, [3 * 5 * L * D, D, L * D], [B, L, 5])  # noqa: E731  [B, 3, H, L, D]
    assert not _share(head_major(0), head_major(1), D) and not _share(head_major(0), head_major(2), D) and _share(head_major(0), q, D)
    mixed = lambda n: (n * D, [L * 5 * 3 * D, 5 * 3 * D, 3 * D], [B, L, 5])  # noqa: E731       [B, L, H, 3, D]
    assert not _share(mixed(0), mixed(1), D) and not _share(mixed(1), mixed(2), D) and _share(mixed(1), (D + 8, *mixed(1)[1:]), D)


def _view(p, L, H, D=64):
    from pyflow_hip.lib import RowsView
    return RowsView(p, L * H * D, H * D, D)


def _attn(**kw):
    """a descriptor whose tensors lie a MiB apart, and a workspace"""
    from pyflow_hip.lib import AttnRangesDesc
    d = AttnRangesDesc()
    d.B, d.H, d.Hkv, d.Lq, d.Lk, d.D, d.scale = 2, 4, 2, 5, 9, 64, 0.125
    for n, name in enumerate(("Q", "O", "dO", "dQ")):
        setattr(d, name, _view((n + 1) << 20, 5, 4))
    for n, name in enumerate(("K", "V", "dK", "dV")):
        setattr(d, name, _view((n + 9) << 20, 9, 2))
    d.LSE, d.workspace, d.workspace_bytes = 1 << 28, 1 << 29, 1 << 28
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("out,other", [("O", "K"), ("O", "V"), ("O", "Q")])
def test_attention_output_overlaps(out, other):
    from pyflow_hip import lib as L
    from pyflow_hip.lib import RowsView
    lib = L.load()
    d = _attn()
    at = getattr(d, other).p
    setattr(d, out, _view(at + 64 * 2, 5, 4))      # half inside
    assert lib.pf_attention_ranges_bf16(C.byref(d), None) == -1 and b"overlaps" in lib.pf_last_error()
    d = _attn(O=RowsView(1 << 24, 0, 4 * 64, 64))
    assert lib.pf_attention_ranges_bf16(C.byref(d), None) == -1 and b"overlaps itself" in lib.pf_last_error()
    d = _attn(O=RowsView(1 << 24, 5 * 4 * 64, 2 * 64, 64))
    assert lib.pf_attention_ranges_bf16(C.byref(d), None) == -1 and b"overlaps itself" in lib.pf_last_error()


@pytest.mark.parametrize("out", ["dQ", "dK", "dV"])
@pytest.mark.parametrize("other", ["Q", "K", "V", "O", "dO", "dQ", "dK", "dV"])
def test_attention_gradient_overlaps(out, other):
    from pyflow_hip import lib as L
    lib = L.load()
    d = _attn()
    if out == other:
        getattr(d, out).row = 64                   # its own heads on its own rows
    else:
        getattr(d, out).p = getattr(d, other).p
    assert lib.pf_attention_ranges_bwd(C.byref(d), None) == -1 and b"overlap" in lib.pf_last_error()


def _heads(**kw):
    from pyflow_hip.lib import HeadsDesc
    d = HeadsDesc()
    d.B, d.L, d.H, d.Hkv, d.D = 2, 3, 4, 2, 64
    for n, name in enumerate(("Q", "Qo", "dQ")):
        setattr(d, name, _view((n + 1) << 20, 3, 4))
    for n, name in enumerate(("K", "Ko", "dK")):
        setattr(d, name, _view((n + 9) << 20, 3, 2))
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("out,other,shift", [("Qo", "Q", 128), ("Qo", "K", 0), ("Ko", "K", 128), ("Ko", "Q", 0), ("Qo", "Ko", 0)])
def test_heads_output_overlaps(out, other, shift):
    from pyflow_hip import lib as L
    lib = L.load()
    d = _heads()
    getattr(d, out).p = getattr(d, other).p + shift
    assert lib.pf_qk_norm_rope_axes(C.byref(d), None) == -1 and b"overlap" in lib.pf_last_error()
    assert lib.pf_qk_norm_rope_axes_bwd(C.byref(d), None, None, None, C.c_longlong(0), None) == -1 and b"overlap" in lib.pf_last_error()


@pytest.mark.parametrize("out,other,shift", [("Qo", "dQ", 128), ("Qo", "dK", 0), ("Ko", "dK", 128), ("Ko", "dQ", 0)])
def test_heads_gradient_overlaps(out, other, shift):
    from pyflow_hip import lib as L
    lib = L.load()
    d = _heads()
    getattr(d, out).p = getattr(d, other).p + shift
    assert lib.pf_qk_norm_rope_axes_bwd(C.byref(d), None, None, None, C.c_longlong(0), None) == -1 and b"overlap" in lib.pf_last_error()
