"""cached_attention where queries, keys and values lie far from one (beyond what goes without the range rule), with scores as they mostly are: powers of two
that cancel change nothing, to the bit."""
import pytest
import torch

import decoding_cases as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
FAR = 2.0 ** 84                                            # 1.9e25


def _inputs(groups, rows, heads, kv_heads, dim, shared, own):
    g = torch.Generator().manual_seed(60 + dim + shared)
    randn = lambda *shape: torch.randn(*shape, generator=g).to(DEV)
    case = dict(q=randn(groups, rows, heads, dim) * dim ** -0.5)
    if shared:
        case.update(shared_k=randn(groups, shared, kv_heads, dim), shared_v=randn(groups, shared, kv_heads, dim))
    if own:
        case.update(own_k=randn(groups, rows, own, kv_heads, dim), own_v=randn(groups, rows, own, kv_heads, dim))
    return case


@pytest.mark.parametrize("size", [(2, 3, 2, 2, 64, 40, 10), (1, 8, 2, 1, 128, 300, 0), (300, 1, 4, 4, 67, 0, 50), (2, 5, 2, 2, 256, 33, 0), (1, 2, 1, 1, 20, 700, 9)])
@pytest.mark.parametrize("where", ["queries", "keys", "values up", "values down"])
@pytest.mark.parametrize("columns", [slice(None), slice(3, None, 17)])
def test_powers_of_two_cancel(size, where, columns):
    from pam_b200 import decoding
    case = _inputs(*size)
    want = decoding.cached_attention(**case)
    exact, bound = oracle.attention(*(case[k].cpu() if k in case else None for k in ("q", "own_k", "own_v", "own_lengths", "shared_k", "shared_v", "shared_lengths")))
    assert float(bound.max()) < 0.01 * float(exact.abs().max())                 # (what is compared says something)
    assert bool(((want.double().cpu() - exact).abs() <= bound).all())
    by = torch.ones(size[4], device=DEV)
    by[columns] = {"queries": FAR, "keys": 1 / FAR, "values up": FAR, "values down": 1 / FAR}[where]
    for name in case:
        case[name] = case[name] * (by if name == "q" and where in ("queries", "keys") else 1 / by if name.endswith("_k") and where in ("queries", "keys") else
                                   by if name.endswith("_v") and where.startswith("values") else 1.0)
    got = decoding.cached_attention(**case)
    assert torch.equal(got, want * by if where.startswith("values") else want)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("side", ["q", "k"])
def test_one_score_of_many(sign, side):
    """Scores of 2^24 and of -2^24 from numbers of 2^84 beside ones near zero: one position has all of the weight, or none."""
    from pam_b200 import decoding
    case = _inputs(2, 3, 2, 2, 64, 40, 0)
    q, k, v = case["q"], case["shared_k"], case["shared_v"]
    q[..., 0], k[..., 0] = (FAR, 0.0) if side == "q" else (2.0 ** 24 / FAR, 0.0)
    k[:, 7, :, 0] = sign * (2.0 ** 24 / FAR if side == "q" else FAR)
    got = decoding.cached_attention(q, shared_k=k, shared_v=v)
    if sign > 0:
        assert torch.equal(got, v[:, 7].unsqueeze(1).expand_as(got))
    else:
        rest = torch.arange(40, device=DEV) != 7
        want, bound = oracle.attention(q.cpu(), None, None, None, k[:, rest].cpu(), v[:, rest].cpu(), None)
        assert float(bound.max()) < 0.01 and bool(((got.double().cpu() - want).abs() <= bound).all())
