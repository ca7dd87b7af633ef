"""Generation refuses source tokens outside the vocabulary, on the GPU, where the lookup gives NaN for them."""
import pytest
import torch

from test_gpu_generation import _net

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["generate", "sample"])
def test_source_tokens_outside_the_vocabulary(what):
    net = _net()
    src = torch.full((2, 5), 7, device="cuda")
    getattr(net, what)(src, 2, 4)
    for token in (-1, net.cfg.vocab):
        src[1, 3] = token
        with pytest.raises(ValueError, match="vocabulary"):
            getattr(net, what)(src, 2, 4)
        with torch.no_grad():
            x = net.encoder.embed(src)                        # (rows without gradients: this one is NaN, the others not)
        at = torch.zeros(2, 5, dtype=torch.bool, device="cuda")
        at[1, 3] = True
        assert torch.equal(x.isnan(), at.unsqueeze(-1).expand_as(x))
