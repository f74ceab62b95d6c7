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
