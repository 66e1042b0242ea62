"""Sampling at the ends of what it takes: the largest vocabulary, whose sum of weights is the largest."""
from __future__ import annotations

import pytest
import torch

from thintensor_b200.kernels import api

DEV = "cuda"


def test_a_vocabulary_whose_weights_could_come_to_64_bits_is_refused():
    assert api.SAMPLE_FILTERED_VOCAB << 45 < 1 << 64
    logits = torch.zeros(1, api.SAMPLE_FILTERED_VOCAB + 1)
    with pytest.raises(api.KernelError, match="vocabularies"):
        api.sample_filtered(logits, 1.0, 0, 1.0, 0.0, torch.zeros(1, dtype=torch.int32), uniform=torch.zeros(1))


@pytest.mark.gpu
@pytest.mark.parametrize("spread,temperature", [(0.0, 1.0), (5.0, 1e30)])
@pytest.mark.parametrize("settings", [dict(), dict(top_p=0.75), dict(top_k=1 << 19), dict(min_p=0.5)])
def test_equal_weights_over_the_largest_vocabulary(spread, temperature, settings):
    """All weights are equal, so the token is the number of whole ones in u times the vocabulary (both sides exact in float64), of which a nucleus leaves all
    where the logits are equal.  Where they are not and a nucleus is asked for, the tokens with the larger logits stay, in order of their id."""
    vocab = 8 * 65536 - 1
    g = torch.Generator().manual_seed(1)
    x = spread * torch.randn(1, vocab, generator=g) + 2.0
    u = torch.tensor([0.0, 2.0 ** -24, 0.25, 0.5, 0.7310585975646973, 1.0 - 2.0 ** -24])
    kept = torch.arange(vocab)
    if spread and "top_p" in settings:
        order = x[0].double().sort(descending=True).values
        above = torch.searchsorted(-order, -x[0].double())            # tokens with a larger logit, whose weights are one each
        kept = kept[above <= 0.75 * vocab]
    out = torch.full((len(u),), -1, dtype=torch.int32, device=DEV)
    api.sample_filtered(x.to(DEV).expand(len(u), vocab), temperature, settings.get("top_k", 0), settings.get("top_p", 1.0), settings.get("min_p", 0.0), out, uniform=u.to(DEV))
    assert out.tolist() == [int(kept[int(v * len(kept))]) for v in u.double().tolist()]
