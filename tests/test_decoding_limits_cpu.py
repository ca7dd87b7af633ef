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


@pytest.mark.parametrize("groups,rows,heads,shared,own,fits", [
    (1, 1 << 20, 1, 3, 0, True), (1, (1 << 20) + 1, 1, 3, 0, False), (1, 1 << 19, 3, 3, 0, False), (1, 1, 1, 1 << 30, 0, True), (1, 1, 1, (1 << 30) + 1, 0, False),
    (1, 1, 1, 1 << 29, (1 << 29) + 1, False), (1 << 20, 1, 1, 2046 * 64, 0, False), (1 << 20, 1, 1, 2045 * 64, 0, True),
])
def test_rows_and_positions(groups, rows, heads, shared, own, fits):
    z = torch.zeros(1)
    q, kv = z.expand(groups, rows, heads, 1), {}
    if shared:
        kv.update(shared_k=z.expand(groups, shared, 1, 1), shared_v=z.expand(groups, shared, 1, 1))
    if own:
        kv.update(own_k=z.expand(groups, rows, own, 1, 1), own_v=z.expand(groups, rows, own, 1, 1))
    with pytest.raises(RuntimeError if fits else ValueError, match="CUDA" if fits else "too many"):
        decoding.cached_attention(q, **kv)
    h, one = _lib.lib(), ctypes.addressof(ctypes.c_float(1.0))
    needed = h.pamk_cached_attention_workspace_bytes(groups, rows, heads, 1, 1, shared, own)
    if needed or not fits:                                 # (the workspace is missing; a call that needs none would run)
        status = h.pamk_cached_attention(one, one, one, one, None, one, one, None, groups, rows, heads, 1, 1, shared, own, (ctypes.c_int64 * 17)(), None, 0, None)
        assert status == (-4 if fits else -2)
