"""Sizes that a launch cannot hold: refused on the host, before any launch."""
import ctypes as C

import pytest


def _desc(B, H, Lq, Lk, D=64):
    from pyflow_hip.lib import AttnRangesDesc, RowsView
    d = AttnRangesDesc()
    d.B, d.H, d.Hkv, d.Lq, d.Lk, d.D, d.scale = B, H, H, Lq, Lk, D, 0.125
    far = 1 << 44                                  # apart by more than any of the tensors is long
    for n, name in enumerate(("Q", "O", "dO", "dQ")):
        setattr(d, name, RowsView((n + 1) * far, Lq * H * D, H * D, D))
    for n, name in enumerate(("K", "V", "dK", "dV")):
        setattr(d, name, RowsView((n + 5) * far, Lk * H * D, H * D, D))
    d.LSE, d.workspace, d.workspace_bytes = 9 * far, 10 * far, 1 << 43
    return d


@pytest.mark.parametrize("B,H,Lq,Lk", [
    (1 << 20, 16, 1, 1),                # one workgroup per row: 2^32 threads, which a launch takes for none
    ((1 << 20) + 1, 16, 1, 1),
    (1 << 18, 64, 33, 4),
    (1 << 14, 512, 129, 1)])
def test_launches_of_2_to_the_32_threads_are_refused(B, H, Lq, Lk):
    from pyflow_hip import lib as L
    lib = L.load()
    d = _desc(B, H, Lq, Lk)
    assert lib.pf_attention_ranges_bf16(C.byref(d), None) == -1 and b"workgroups" in lib.pf_last_error()


@pytest.mark.parametrize("B,H,Lq,Lk", [(1 << 14, 1 << 10, 1, 1), (1 << 15, 256, 1, 200), (1 << 14, 512, 65, 1)])
def test_gradient_launches_of_2_to_the_32_threads_are_refused(B, H, Lq, Lk):
    from pyflow_hip import lib as L
    lib = L.load()
    d = _desc(B, H, Lq, Lk)
    assert lib.pf_attention_ranges_bwd(C.byref(d), None) == -1 and b"workgroups" in lib.pf_last_error()
