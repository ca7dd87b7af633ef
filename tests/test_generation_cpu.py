"""Beam search of the translation model with the ordinary operators, against a search without caches."""
import pytest
import torch

import generation_cases as cases


@pytest.mark.parametrize("beam,max_len,min_len,penalty", [(1, 6, 1, 1.0), (3, 8, 1, 1.0), (4, 7, 4, 0.6), (2, 1, 1, 1.0)])
def test_against_search_without_caches(beam, max_len, min_len, penalty):
    net = cases.model({}, "cpu")
    src = torch.randint(4, net.cfg.vocab, (3, 7), generator=torch.Generator().manual_seed(beam))
    # (scores near -10, sums of some ten fp32 log-probabilities of 40 classes)
    for g in range(3):
        cases.check(net, src[g:g + 1], None, beam, max_len, min_len, penalty, lambda x: torch.log_softmax(x, -1), 1e-4)
    cases.check(net, src, None, beam, max_len, min_len, penalty, lambda x: torch.log_softmax(x, -1), 1e-4)


def test_padded_batch():
    net = cases.model({}, "cpu", 1)
    src = torch.randint(4, net.cfg.vocab, (3, 9), generator=torch.Generator().manual_seed(3))
    lengths = torch.tensor([9, 4, 6])
    cases.check(net, src, lengths, 3, 8, 1, 1.0, lambda x: torch.log_softmax(x, -1), 1e-4)
    other = src.clone()
    other[1, 4:], other[2, 6:] = 1, 5                        # what the padding holds does not matter
    for a, b in zip(net.generate(src, 3, 8, src_lengths=lengths), net.generate(other, 3, 8, src_lengths=lengths)):
        assert torch.equal(a, b)


def test_refusals():
    net = cases.model({}, "cpu")
    src = torch.full((1, 3), 4)
    for kw in (dict(beam=0), dict(beam=33), dict(max_len=0), dict(min_len=5, max_len=4), dict(eos=1), dict(eos=40)):
        with pytest.raises(ValueError):
            net.generate(src, **kw)


@pytest.mark.parametrize("lengths", [[0, 3], [4, 1], [-1, 2]])
def test_refuses_lengths_outside_the_sentences(lengths):
    with pytest.raises(ValueError, match="lengths"):
        cases.model({}, "cpu").generate(torch.full((2, 3), 4), src_lengths=torch.tensor(lengths))


def test_double_precision():
    net = cases.model({}, "cpu", 2)
    src = torch.randint(4, net.cfg.vocab, (2, 5), generator=torch.Generator().manual_seed(8))
    want = net.generate(src, 3, 6)
    got = net.double().generate(src, 3, 6)
    assert torch.equal(got[0], want[0]) and bool(((got[1] - want[1]).abs() < 1e-4).all())
