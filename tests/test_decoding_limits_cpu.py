"""The sizes that the operators of text generation take at most, by name; no GPU needed."""
import ctypes

import pytest
import torch

from pam_b200 import _lib, decoding


@pytest.mark.parametrize("beams,vocab,fits", [(64, 261888, True), (64, 261889, False), (1, 4096 * 4092, True), (1, 4096 * 4092 + 1, False), (33, 510000, False)])
def test_ranges_of_a_group(beams, vocab, fits):
    logits, scores = torch.zeros(1, 1, 1).expand(1, beams, vocab), torch.zeros(1, beams)
    # (what fits is refused for being on the CPU)
    with pytest.raises(RuntimeError if fits else ValueError, match="CUDA" if fits else "ranges"):
        decoding.beam_select(logits, scores, 2)
    h, one = _lib.lib(), ctypes.addressof(ctypes.c_float(1.0))
    status = h.pamk_beam_select(one, one, None, one, one, one, 1, beams, vocab, 2, 1, 1, 0, 0, None, 0, None)
    assert status == (-4 if fits else -2)                  # no workspace; a size
