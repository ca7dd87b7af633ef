"""Beam search of a batch: each sentence gets what it gets alone."""
import pytest
import torch

import generation_cases as cases


def _alone(net, src, lengths, **kw):
    """Each sentence by itself: [(scores [beam], [tokens without padding])]."""
    out = []
    for g in range(src.shape[0]):
        tokens, scores = net.generate(src[g:g + 1, :src.shape[1] if lengths is None else int(lengths[g])], **kw)
        out.append((scores[0], [t[t != net.cfg.pad].tolist() for t in tokens[0]]))
    return out


@pytest.mark.parametrize("seed", range(4))
def test_a_batch_is_its_sentences(seed):
    net = cases.model({}, "cpu", seed)
    src = torch.randint(4, net.cfg.vocab, (4, 7), generator=torch.Generator().manual_seed(seed))
    tokens, scores = net.generate(src, 3, 12)
    for g, (want, words) in enumerate(_alone(net, src, None, beam=3, max_len=12)):
        # (sums of some ten fp32 log-probabilities of 40 classes, near -10 at most)
        assert bool(((scores[g] - want).abs() <= 1e-4).all())
        assert [t[t != net.cfg.pad].tolist() for t in tokens[g]] == words


def test_a_padded_batch_is_its_sentences():
    net = cases.model({}, "cpu", 2)
    src = torch.randint(4, net.cfg.vocab, (5, 9), generator=torch.Generator().manual_seed(7))
    lengths = torch.tensor([9, 2, 7, 4, 1])
    kw = dict(beam=4, max_len=10, min_len=2, length_penalty=0.7)
    tokens, scores = net.generate(src, src_lengths=lengths, **kw)
    for g, (want, words) in enumerate(_alone(net, src, lengths, **kw)):
        assert bool(((scores[g] - want).abs() <= 1e-4).all())
        assert [t[t != net.cfg.pad].tolist() for t in tokens[g]] == words
