"""Rotary frequencies from a model's configuration, whose original context may stand beside its rope_scaling dict."""
import pytest
import torch

import fftsparse_b200 as F

SCALINGS = [
    {"type": "dynamic", "factor": 2.0},
    {"rope_type": "yarn", "factor": 4.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0},
]


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("missing", [{}, {"original_max_position_embeddings": None}])
def test_the_context_may_come_from_the_configuration(scaling, missing):
    inside = dict(scaling, original_max_position_embeddings=4096)
    want, attn = F.rotary_inv_freq(64, 10000.0, inside, 16384)
    got, factor = F.rotary_inv_freq(64, 10000.0, dict(scaling, **missing), 16384, max_position_embeddings=4096)
    assert torch.equal(got, want) and factor == attn
    # the dict's own number comes first
    got, _ = F.rotary_inv_freq(64, 10000.0, inside, 16384, max_position_embeddings=32768)
    assert torch.equal(got, want)
    other, _ = F.rotary_inv_freq(64, 10000.0, scaling, 16384, max_position_embeddings=1024)
    assert not torch.equal(other, want)


@pytest.mark.parametrize("scaling", SCALINGS + [{"rope_type": "yarn", "factor": None, "original_max_position_embeddings": 4096}])
def test_what_is_missing_is_named(scaling):
    with pytest.raises(ValueError, match="factor" if "original_max_position_embeddings" in scaling else "original_max"):
        F.rotary_inv_freq(64, 10000.0, scaling, 16384)
