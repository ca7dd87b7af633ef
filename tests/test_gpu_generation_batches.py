"""Beam search of a batch in PAM arithmetic: each sentence gets what it gets alone."""
import pytest
import torch

from test_gpu_generation import TOLERANCE, _net

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(4))
def test_a_batch_is_its_sentences(seed):
    net = _net(seed)
    src = torch.randint(4, net.cfg.vocab, (4, 7), generator=torch.Generator().manual_seed(seed)).cuda()
    tokens, scores = net.generate(src, 3, 12)
    for g in range(4):
        _, want = net.generate(src[g:g + 1], 3, 12)
        assert bool(((scores[g] - want[0]).abs() <= TOLERANCE).all())


def test_a_padded_batch_is_its_sentences():
    net = _net(2)
    src = torch.randint(4, net.cfg.vocab, (5, 9), generator=torch.Generator().manual_seed(7)).cuda()
    lengths = torch.tensor([9, 2, 7, 4, 1], device="cuda")
    kw = dict(beam=4, max_len=10, min_len=2, length_penalty=0.7)
    _, scores = net.generate(src, src_lengths=lengths, **kw)
    for g in range(5):
        _, want = net.generate(src[g:g + 1, :int(lengths[g])], **kw)
        assert bool(((scores[g] - want[0]).abs() <= TOLERANCE).all())
