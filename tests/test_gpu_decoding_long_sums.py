"""cached_attention: what the order of its sums costs on long rows."""
import pytest
import torch

import decoding_cases as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
POSITIONS, UNITS = 1 << 16, 2400                 # rows enough for every CTA to have one to itself, were its positions not limited


@pytest.mark.parametrize("own", [False, True])
def test_long_rows_are_summed_in_blocks(own):
    """Every position has the same weight 2^-16 and the same value c: the result is c, up to the rounding of sums.  What c has beyond 1 is a little below half a
    step of a sum from 2^13 on, where each addition would drop it: a sum of 2^14 terms in a row would be 2.4e-4 off.  Sums of at most 1024
    positions by a CTA, over at most 8 warps and 32 lanes, and of 64 CTAs add at most 1024 + 8 + 5 + 64 roundings of u."""
    from pam_b200 import decoding
    c = 1.0 + 0.4999 * 2.0 ** -10
    q = torch.ones(UNITS, 1, 1, 128, device=DEV)
    k, v = torch.zeros(POSITIONS, 1, 128, device=DEV), torch.full((POSITIONS, 1, 128), c, device=DEV)
    c = float(v[0, 0, 0])
    if own:
        out = decoding.cached_attention(q, k.expand(UNITS, 1, -1, -1, -1), v.expand(UNITS, 1, -1, -1, -1))
    else:
        out = decoding.cached_attention(q, shared_k=k.expand(UNITS, -1, -1, -1), shared_v=v.expand(UNITS, -1, -1, -1))
    assert bool(((out.double() - c).abs() <= (1024 + 8 + 5 + 64) * oracle.U * c).all())
