"""The operators of text generation at the sizes that they take at most."""
import pytest
import torch

import decoding_cases as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"


def test_select_at_the_most_ranges():
    from pam_b200 import decoding
    g = torch.Generator().manual_seed(1)
    logits, scores = torch.randn(1, 64, 261889, generator=g), -torch.rand(1, 64, generator=g)
    with pytest.raises(ValueError, match="ranges"):
        decoding.beam_select(logits.to(DEV), scores.to(DEV), 3)
    logits = logits[:, :, :-1]
    best, beams, tokens = decoding.beam_select(logits.to(DEV), scores.to(DEV), 3)
    want = oracle.select(logits, scores, 3)
    assert torch.equal(beams.cpu(), want[1]) and torch.equal(tokens.cpu(), want[2])
    assert bool(((best.double().cpu() - want[0]).abs() <= oracle.select_bound(want[0])).all())
