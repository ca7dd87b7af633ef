"""The gradient of tokens that occur very often: its error does not grow with their number."""
import pytest
import torch

from vocabulary_cases import U

pytestmark = pytest.mark.gpu


def gradient(tokens, g, vocab):
    import pam_b200 as pam
    w = torch.zeros(vocab, g.shape[1], device="cuda", requires_grad=True)
    return torch.autograd.grad(pam.embedding(tokens.cuda(), w), w, g.cuda())[0].double().cpu()


# Up to 32 terms that follow one another in the order are added in fp32: 31 roundings of at most u = 2^-24 of the sum of their magnitudes.  Up to 16 of these
# sums are added pair by pair, four roundings more for each, and what comes of it in 64 bits, rounded once: 36 u together, to first order; 37 u covers the
# second and 2^16 roundings of 2^-53.
BOUND = 37 * U


@pytest.mark.parametrize("dim", [4, 5])
@pytest.mark.parametrize("n", [300, 20000, (1 << 20) + 7, 1 << 22])
def test_equal_terms(n, dim):
    """Terms of one sign and size, whose roundings do not average out."""
    tokens = torch.full((n,), 2)
    tokens[::100] = 0
    g = torch.full((n, dim), 1.1e-3)
    count = torch.bincount(tokens, minlength=4).double()[:, None]
    want = count * float(g[0, 0])
    d = gradient(tokens, g, 4)
    assert bool(((d - want).abs() <= BOUND * want).all()), ((d - want).abs() / want.clamp(min=1e-30)).max()


@pytest.mark.parametrize("runs", [(32 * 13 - 1, 32 * 12, 32 * 11 + 3, 40000), (700000, 5, 300000)])
def test_terms_of_one_sign(runs):
    order = torch.randperm(sum(runs), generator=torch.Generator().manual_seed(1))
    tokens = torch.arange(len(runs)).repeat_interleave(torch.tensor(runs))[order]
    g = torch.rand(len(tokens), 6, generator=torch.Generator().manual_seed(2)) + 0.5
    want = torch.zeros(len(runs), 6, dtype=torch.float64).index_add_(0, tokens, g.double())
    d = gradient(tokens, g, len(runs))
    assert bool(((d - want).abs() <= BOUND * want).all()), ((d - want).abs() / want.clamp(min=1e-30)).max()
