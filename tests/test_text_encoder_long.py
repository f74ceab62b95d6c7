"""T5EncoderHIP beyond 256 tokens: the bias by distance, and the encoder against transformers."""
import os
import sys

import pytest
import torch

from util import rel_l2

sys.path.insert(0, os.path.join(os.path.dirname(__file__), "helpers"))


@pytest.mark.parametrize("nb,md", [(32, 128), (16, 64), (32, 20)])
def test_bias_by_distance_is_the_position_bias(nb, md):
    from pyflow_hip.text_encoder import t5_bias_by_distance, t5_relative_position_buckets
    w = torch.randn(nb, 3, generator=torch.Generator().manual_seed(nb + md))
    table = t5_bias_by_distance(w, nb, md)
    assert table.shape == (3, 2 * md + 1)
    L = 3 * md + 7
    j = torch.arange(L)
    clamped = (j[None] - j[:, None]).clamp(-md, md) + md
    assert torch.equal(table[:, clamped], w[t5_relative_position_buckets(L, nb, md)].permute(2, 0, 1))


def test_wide_distances_are_refused_beyond_256():
    from pyflow_hip.text_encoder import T5EncoderHIP
    e = T5EncoderHIP.__new__(T5EncoderHIP)
    e.max_distance = 1024
    with pytest.raises(ValueError, match="max_distance"):
        e.forward(torch.zeros(1, 257, dtype=torch.long))


@pytest.mark.gpu
@pytest.mark.parametrize("L,valid", [(257, [257, 30]), (512, [500, 1]), (700, [700])])
def test_long_prompts_vs_transformers(L, valid):
    """the bar of the encoder tests: rel-L2 <= 2e-2 per output"""
    from hf_text import tiny_t5
    from pyflow_hip.text_encoder import T5EncoderHIP
    model, cfg = tiny_t5(seed=4)
    g = torch.Generator().manual_seed(L)
    ids = torch.randint(3, cfg.vocab_size - 1, (len(valid), L), generator=g)
    mask = torch.zeros(len(valid), L, dtype=torch.long)
    for b, n in enumerate(valid):
        mask[b, :n] = 1
    if L == 512:
        mask[0, 100:180] = 0                       # a hole: two runs
    with torch.no_grad():
        ref = model(ids, attention_mask=mask)[0]
    eng = T5EncoderHIP(model.state_dict(), cfg, "cuda")
    out = eng(ids, attention_mask=mask.cuda()).float().cpu()
    for b, n in enumerate(valid):
        assert rel_l2(out[b, :n], ref[b, :n]) < 2e-2
    assert rel_l2(out, ref) < 2e-2
    with torch.no_grad():
        ref = model(ids)[0]
    assert rel_l2(eng(ids).float().cpu(), ref) < 2e-2
    # the short form of the same weights is what it was: 256 tokens of the scalar kernel against the first 256 of a padded long call
    short = eng(ids[:, :256]).float().cpu()
    m = torch.zeros(len(valid), L, dtype=torch.long)
    m[:, :256] = 1
    assert rel_l2(eng(ids, attention_mask=m)[:, :256].float().cpu(), short) < 2e-2
    m[:, 10] = m[:, 20] = 0                        # three runs
    with pytest.raises(NotImplementedError):
        eng(ids, attention_mask=m)
