"""KeyRanges.pairs against the dense mask."""
import pytest
import torch


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("two", [False, True])
def test_pairs_are_those_of_the_dense_mask(two, shared):
    from pyflow_hip.plan import KeyRanges
    g = torch.Generator().manual_seed(81)
    B, Lq, Lk = 3, 40, 23
    i = torch.iinfo(torch.int32)
    r = [torch.randint(-5, Lk + 6, (1 if shared else B, Lq), generator=g).int() for _ in range(4 if two else 2)]
    r[0][:, 3], r[1][:, 3], r[0][:, 4], r[1][:, 4] = i.min, i.max, i.max, i.min
    ranges = KeyRanges(*r)
    assert ranges.pairs(B, Lk) == int(ranges.dense_mask(Lk).expand(B, Lq, Lk).sum())


def test_pairs_of_the_named_masks():
    from pyflow_hip.plan import KeyRanges
    assert KeyRanges.causal(5, 7, "cpu").pairs(2, 7) == 2 * (3 + 4 + 5 + 6 + 7)
    assert KeyRanges.documents([2, 0, 3], 7, "cpu").pairs(1, 7) == 4 + 9
    assert KeyRanges.padded([3, 9], 4, "cpu").pairs(2, 7) == 4 * (3 + 7)
