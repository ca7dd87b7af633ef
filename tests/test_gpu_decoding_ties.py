"""beam_select where thousands of logits are equal."""
import pytest
import torch

import decoding_cases as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _milliseconds(call):
    for _ in range(3):
        call()
    times = []
    for _ in range(7):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call()
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end))
    return sorted(times)[3]


@pytest.mark.parametrize("banned", [False, True])
def test_many_equal_logits_cost_as_much_for_more_beams(banned):
    """With k = 33 as with k = 32: the candidates are narrowed down to a multiple of k, not ranked among all 4092 of a range (which took six times as long)."""
    from pam_b200 import decoding
    logits, scores = torch.zeros(8, 4, 20000, device=DEV), torch.zeros(8, 4, device=DEV)
    flags = torch.ones(20000, dtype=torch.bool, device=DEV)
    flags[::1000] = False
    few, many = (_milliseconds(lambda: decoding.beam_select(logits, scores, k, flags if banned else None)) for k in (32, 33))
    assert many <= 2 * few


@pytest.mark.parametrize("k", [1, 8, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("vocab", [513, 600, 4092, 9001])
def test_equal_logits(k, vocab):
    """The lowest beams and tokens; with a few larger and banned ones among them, those in their order."""
    from pam_b200 import decoding
    logits, scores = torch.zeros(2, 3, vocab), torch.zeros(2, 3)
    logits[1, 1, vocab - 3:] = 0.5
    logits[1, 2, ::7] = 1.0
    banned = torch.zeros(vocab, dtype=torch.bool)
    banned[5:200] = True
    for ban in (None, banned):
        got = decoding.beam_select(logits.to(DEV), scores.to(DEV), k, None if ban is None else ban.to(DEV))
        want = oracle.select(logits, scores, k, ban)
        assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
