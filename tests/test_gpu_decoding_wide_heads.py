"""cached_attention: what the order of its sums costs on wide heads."""
import pytest
import torch

import decoding_cases as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("groups,rows,positions", [(700, 1, 2), (700, 8, 2), (700, 1, 300), (64, 8, 600), (1, 5, 2), (2, 3, 5000)])
@pytest.mark.parametrize("dim,zero", [(256, False), (256, True), (250, False), (224, False)])
def test_wide_heads_are_summed_in_blocks(groups, rows, positions, dim, zero):
    """Keys of 2^18, -2^18 and then many numbers, each a little less than what a sum of 2^18 can hold: one behind another they would all be lost, and every position would
    count the same.  Slices of 32 floats are two sums of 16 each, which two sums over the slices take up; behind 2^18 each addition loses 2^-6 at most, so what is lost
    is at most 2 (16 + dim / 32) 2^-6 of a score (all of it: dim 2^-7)."""
    from pam_b200 import decoding
    small = 0.4999 * 2.0 ** -6
    q = torch.ones(groups, rows, 1, dim, device=DEV)
    k, v = torch.full((1, positions, 1, dim), small), torch.ones(1, positions, 1, dim)
    k[0, 1::2] = small * (1 - 2 * (torch.arange(dim) // 2 % 2))                  # every other position: alternating signs
    v[0, 1::2] = 0.0625
    k[..., 0], k[..., 1] = 2.0 ** 18, -2.0 ** 18
    if zero:                                                                     # (a value for the range rule)
        q[..., 5] = 0.0
    s = (k[0, :, 0].double() * q[0, 0, 0].cpu().double()).sum(-1)
    lost = 2 * (16 + dim / 32) * 2.0 ** -6
    assert lost < 0.75 * float(s[0])
    weight = lambda x: oracle.exp2(oracle.pam(x, oracle.LOG2E))                  # (shifts scale all of a row's weights by a power of two)
    live = torch.full((positions // 2,), 1.0, dtype=torch.float64)

    def result(off):
        high, low = weight(s[0] + off) * live, weight(s[1] - off) * live
        total = high.sum() + low.sum()
        return float(oracle.pad(high, total).sum() + oracle.pam(oracle.pad(low, total), 0.0625).sum())

    out = decoding.cached_attention(q, shared_k=k.to(DEV).expand(groups, -1, -1, -1), shared_v=v.to(DEV).expand(groups, -1, -1, -1))
    assert out.amin() >= result(-lost) * (1 - 1e-4) and out.amax() <= result(lost) * (1 + 1e-4)
