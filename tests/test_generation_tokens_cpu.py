"""Generation refuses source tokens outside the vocabulary, on the CPU."""
import pytest
import torch

import generation_cases as cases


@pytest.mark.parametrize("token", [-1, -100, 40, 2 ** 40])
@pytest.mark.parametrize("what", ["generate", "sample"])
def test_source_tokens_outside_the_vocabulary(what, token):
    net = cases.model({}, "cpu")
    src = torch.full((2, 5), 7)
    src[1, 3] = token
    with pytest.raises(ValueError, match="vocabulary"):
        getattr(net, what)(src, 2, 4)
    with pytest.raises(ValueError, match="vocabulary"):
        getattr(net, what)(src, 2, 4, src_lengths=torch.tensor([5, 3]))


@pytest.mark.parametrize("what", ["generate", "sample"])
def test_its_ends(what):
    net = cases.model({}, "cpu")
    tokens, _ = getattr(net, what)(torch.tensor([[0, 39, 1]], dtype=torch.int32), 2, 4)
    assert tokens.shape[0] == 1
